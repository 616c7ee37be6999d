"""Decoding over 8-bit caches and with log probabilities.

* With ``kv_block=1`` a cache does not depend on how its tokens were split into calls, so
  speculative decoding emits what plain decoding over the same kind of cache emits; the output
  head is scaled up so that argmax margins are far above rounding.
* The log probabilities, entropies and alternatives of the emitted tokens are those of the
  model's logits at their positions.
"""

import pytest
import torch

from tests.conftest import tiny_model_config

CASES = [{"mtp.depth": 2}, {"mtp.depth": 1, "layer_pattern": "GL"}, {"mtp.depth": 2, "layer_pattern": "GLXX"},
         {"mtp.depth": 2, "layer_pattern": "GD"}]


def _model(ov, device, gain):
    from myk_llm_b200.models import MykLLM

    torch.manual_seed(0)
    model = MykLLM(tiny_model_config(**ov)).to(device).eval()
    with torch.no_grad():
        model.lm_head.weight.mul_(gain)
    return model


def _spec_equals_plain(ov, device, dtype):
    from myk_llm_b200.infer import StaticDecoder

    model = _model(ov, device, 40.0)
    prompts = torch.randint(0, 512, (3, 12), device=device)
    outs = []
    for depth in (0, None):
        dec = StaticDecoder(model, batch_size=3, max_len=64, draft_depth=depth, kv_dtype=dtype, kv_block=1)
        outs.append(dec.generate(prompts, 24, check_every=2)[0])
    assert torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("ov", CASES)
def test_8bit_spec_decode_equals_plain_cpu(ov, dtype):
    _spec_equals_plain(ov, "cpu", dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("ov", CASES)
def test_8bit_spec_decode_equals_plain_gpu(ov, dtype):
    from myk_llm_b200.ops import ext

    _spec_equals_plain(ov, "cuda", dtype)
    assert ext().take_status() == 0


def _logprobs(device, kv_dtype, tol):
    from myk_llm_b200.infer import StaticDecoder

    model = _model({"mtp.depth": 2}, device, 4.0)
    prompts = torch.randint(0, 512, (3, 12), device=device)
    dec = StaticDecoder(model, batch_size=3, max_len=64, kv_dtype=kv_dtype, logprobs=5)
    toks, st = dec.generate(prompts, 20, check_every=2)
    lp = st.logprobs
    assert lp.logprobs.shape == lp.entropy.shape == (3, 20) and lp.top_tokens.shape == lp.top_logprobs.shape == (3, 20, 5)
    # greedy: the emitted token is the first alternative
    assert torch.equal(lp.top_tokens[..., 0], toks[:, 12:])
    torch.testing.assert_close(lp.top_logprobs[..., 0], lp.logprobs, rtol=0, atol=1e-5)
    with torch.no_grad():
        out = model(toks[:, :-1])
        want = torch.log_softmax(model.logits(out.hidden[:, 11:]).double(), -1)
    got = want.gather(-1, toks[:, 12:, None])[..., 0]
    assert (lp.logprobs.double() - got).abs().max() <= tol
    assert (lp.entropy.double() + (want.exp() * want).sum(-1)).abs().max() <= tol
    # without the option, the same tokens
    plain, st = StaticDecoder(model, batch_size=3, max_len=64, kv_dtype=kv_dtype).generate(prompts, 20, check_every=2)
    assert torch.equal(plain, toks) and st.logprobs is None


# fp32 throughout on the CPU; on the GPU bf16 activations (2^-8) through a few layers move logits of size ~4 by a
# few hundredths, and an 8-bit cache (e4m3: 2^-4 per key and value, averaged over the keys) about as much again
def test_decoder_logprobs_cpu():
    _logprobs("cpu", None, 1e-4)


def test_decoder_logprobs_8bit_cpu():
    _logprobs("cpu", torch.int8, 0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("kv_dtype", [None, torch.float8_e4m3fn, torch.int8])
def test_decoder_logprobs_gpu(kv_dtype):
    from myk_llm_b200.ops import ext

    _logprobs("cuda", kv_dtype, 0.3)
    assert ext().take_status() == 0
