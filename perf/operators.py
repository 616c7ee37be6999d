"""Cases of three operators of the decoder and their plain forms in elementary torch operations.

* ``cache``: keys and values written into an 8-bit cache (one power-of-two scale for each
  block of tokens of each sequence and head), then read back;
* ``attend``: attention over that cache, alone (a layer that reads another layer's cache)
  or as a whole step (the new tokens are written first);
* ``logprobs``: log probabilities of given tokens with entropy and top alternatives, and
  (``grad``) the gradient with respect to the logits.

The cache is (batch, kv_heads, capacity, head_dim) in e4m3 or int8 with scale bytes
(batch, kv_heads, blocks) that hold ``log2(scale) + 127``; 255 marks a block that was given
a NaN or an infinity.  Sizes are those of the repository's configurations (16/4 heads of 64,
16/4 and 8/2 heads of 128, a 512-token window, 8192-token sequences, 65536 and 32768
vocabularies) and of its decoding benchmark (2048-token prompts, batches of 1 to 64, two
drafted tokens).
"""

import math

import torch

own = False

QMAX = {"e4m3": 448.0, "int8": 127.0}
DTYPE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


# ------------------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step's new token for each of 8 sequences, mid-block, and a short cache read back
        dict(name="cache-step", op="cache", batch=8, new=1, ctx=509, kv_heads=4, dim=64, kind="e4m3", block=16),
        # a prompt of the decoding benchmark written into empty caches and read back
        dict(name="cache-prompt", op="cache", batch=8, new=2048, ctx=0, kv_heads=4, dim=128, kind="e4m3", block=16),
        # prompt chunks that continue sequences of unequal length, odd sizes, wide blocks
        dict(name="cache-ragged", op="cache", batch=13, new=1000, ctx=3001, kv_heads=2, dim=128, kind="int8", block=64),
        # one query token of one sequence at the benchmark's context: latency
        dict(name="attend-one", op="attend", batch=1, new=1, step=False, ctx=2048, heads=16, kv_heads=4, dim=64,
             kind="e4m3", block=16, window=0, ragged=False),
        # a speculative verify step (bonus + two drafts) of 64 sequences of unequal length
        dict(name="attend-verify", op="attend", batch=64, new=3, step=True, ctx=2048, heads=16, kv_heads=4, dim=64,
             kind="e4m3", block=16, window=0, ragged=True),
        # the 200M model's sliding-window layer: long ragged sequences of which 512 tokens are seen
        dict(name="attend-window", op="attend", batch=48, new=1, step=False, ctx=8191, heads=8, kv_heads=2, dim=128,
             kind="int8", block=64, window=512, ragged=True),
        # two very long sequences: the key axis is all there is to split
        dict(name="attend-long", op="attend", batch=2, new=1, step=False, ctx=131071, heads=16, kv_heads=4, dim=128,
             kind="int8", block=32, window=0, ragged=False),
        # a full batch at the models' longest sequence: bandwidth
        dict(name="attend-full", op="attend", batch=64, new=1, step=False, ctx=8192, heads=16, kv_heads=4, dim=128,
             kind="e4m3", block=16, window=0, ragged=False),
        # a chunk of a prompt written behind what the cache holds, attending to all of it
        dict(name="attend-chunk", op="attend", batch=4, new=509, step=True, ctx=4096, heads=16, kv_heads=4, dim=128,
             kind="e4m3", block=16, window=0, ragged=True),
        # the logits of one decode step of 8 sequences, with 20 alternatives a token
        dict(name="logprobs-step", op="logprobs", rows=8, vocab=65536, top=20, kind="bf16", grad=False, masked=False),
        # scoring a batch of continuations
        dict(name="logprobs-score", op="logprobs", rows=4096, vocab=65536, top=5, kind="bf16", grad=False, masked=False),
        # a policy-gradient step with an entropy bonus: values and the logits' gradient
        dict(name="logprobs-train", op="logprobs", rows=4095, vocab=32768, top=0, kind="bf16", grad=True, masked=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["cache", "attend", "attend", "logprobs"])
    if op == "logprobs":
        grad = rng.random() < 0.5
        kind = rng.choice(["bf16", "bf16", "fp32"])
        vocab = _log(rng, 300, 131072)
        most = 2 ** 28 // (2 if grad else 1) // (2 if kind == "fp32" else 1)
        return dict(op=op, rows=_log(rng, 1, min(8192, most // vocab)), vocab=vocab,
                    top=rng.choice([0, 1, 5, 20, 32]), kind=kind, grad=grad, masked=rng.random() < 0.3)
    kind, block = rng.choice(["e4m3", "int8"]), rng.choice([1, 8, 16, 16, 32, 64, 128])
    group, kv_heads, dim = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 128])
    batch = _log(rng, 1, 64)
    if op == "cache":
        ctx = _log(rng, 1, 8192) - 1
        new = _log(rng, 1, 4096)
        while batch * (new + ctx) * kv_heads * dim > 2 ** 25:
            batch, new, ctx = max(1, batch // 2), max(1, new * 2 // 3), ctx * 2 // 3
        return dict(op=op, batch=batch, new=new, ctx=ctx, kv_heads=kv_heads, dim=dim, kind=kind, block=block)
    new = 1 if rng.random() < 0.5 else _log(rng, 2, 512)
    ctx = _log(rng, 1, 131072)
    while batch * (ctx + new) * kv_heads * dim > 2 ** 27 or batch * (ctx + new) * kv_heads * group * new > 2 ** 27:
        batch, ctx = max(1, batch * 2 // 3), max(1, ctx * 3 // 4)
    return dict(op=op, batch=batch, new=new, step=rng.random() < 0.5, ctx=ctx, heads=group * kv_heads,
                kv_heads=kv_heads, dim=dim, kind=kind, block=block,
                window=rng.choice([0, 0, 0, _log(rng, 16, 1024)]), ragged=rng.random() < 0.6)


def _capacity(case):
    return case["ctx"] + case["new"] + 2 * case["block"] + 3


def _lengths(case, seed):
    """Tokens each sequence holds before the call, as a list."""
    g = torch.Generator().manual_seed(seed * 7 + 3)
    ctx, n = case["ctx"], case["batch"]
    if case["op"] == "cache":
        lo = 0 if ctx == 0 else max(0, ctx - 4 * case["block"])
        return torch.randint(lo, ctx + 1, (n,), generator=g).tolist()
    if not case["ragged"]:
        return [ctx] * n
    return (torch.rand(n, generator=g) * ctx).long().add(1).clamp(max=ctx).tolist()


def work(case):
    if case["op"] == "logprobs":
        size = 2 if case["kind"] == "bf16" else 4
        n = case["rows"] * case["vocab"]
        out = case["rows"] * (8 + 8 + 12 * case["top"])
        passes = 2 if case["grad"] else 1  # logits read, gradient written
        return {"bytes": passes * n * size + out, "flops": n * (12 if case["grad"] else 5)}
    row = case["kv_heads"] * case["dim"] * 2  # elements of a token's key and value
    written = case["batch"] * case["new"] * row * 3  # 2-byte input, 1-byte cache
    if case["op"] == "cache":
        read = case["batch"] * (case["ctx"] + case["new"]) * row * 3
        return {"bytes": written + read, "flops": case["batch"] * (2 * case["new"] + case["ctx"]) * row}
    lens = _lengths(case, 0)
    new = case["new"]
    seen = [n + (new if case["step"] else 0) for n in lens]
    if case["window"]:
        keys = sum(min(n, case["window"] + new - 1) for n in seen)
        pairs = sum(min(n, case["window"]) * new for n in seen)
    else:
        keys = sum(seen)
        pairs = sum(n * new - new * (new - 1) // 2 if n >= new else n * (n + 1) // 2 for n in seen)
    io = case["batch"] * new * case["heads"] * case["dim"] * 4
    held = case["batch"] * new * row * 3 if case["step"] else 0  # the new tokens read back
    return {"bytes": keys * row + io + (written + held if case["step"] else 0),
            "flops": 4 * pairs * case["heads"] * case["dim"]}


# ------------------------------------------------------------------------------- plain cache
def _exponent(amax, kind):
    """log2 of the smallest power of two s with amax <= QMAX * s, at least -100; 128 where amax is not finite."""
    m, e = torch.frexp(amax)
    top, bits = (0.875, 9) if kind == "e4m3" else (0.9921875, 7)
    e = (e - bits + (m > top)).clamp(min=-100)
    return torch.where(torch.isfinite(amax), e, torch.full_like(e, 128))


def _power(e):
    """2**e as fp32, NaN for the exponent that marks a block without a scale."""
    return torch.where(e == 128, math.nan, torch.ldexp(torch.ones_like(e, dtype=torch.float32), e.clamp(max=127)))


def _round(x, kind):
    """To the 8-bit type's values (in fp32), ties to even."""
    if kind == "int8":
        return x.round().clamp(-127, 127).nan_to_num(0.0)
    return x.clamp(-448, 448).nan_to_num(0.0).to(torch.float8_e4m3fn).float()


def _quantise(x, kind, block):
    """x (batch, heads, tokens, dim) -> 8-bit values and scale bytes of whole blocks."""
    b, h, n, d = x.shape
    blocks = -(-n // block)
    pad = torch.nn.functional.pad(x.float(), (0, 0, 0, blocks * block - n)).view(b, h, blocks, block, d)
    e = _exponent(pad.abs().amax((-1, -2)), kind)
    q = _round(pad / _power(e)[..., None, None], kind).view(b, h, -1, d)[:, :, :n]
    return q.to(DTYPE[kind]).contiguous(), (e + 127).to(torch.uint8)


def _plain_append(data, scales, x, lens, kind, block):
    """x (batch, new, heads, dim) into data / scales at positions lens[b]: over the blocks that the new tokens touch."""
    b, new, h, d = x.shape
    span = (-(-new // block) + 1) * block
    first = (lens // block) * block
    pos = first[:, None] + torch.arange(span, device=x.device)  # (batch, span)
    is_old = pos < lens[:, None]
    is_new = (pos >= lens[:, None]) & (pos < lens[:, None] + new) & (pos < data.shape[2])
    at = pos.clamp(max=data.shape[2] - 1)[:, None, :, None].expand(-1, h, -1, d)
    held = data.gather(2, at) if kind == "int8" else data.view(torch.uint8).gather(2, at).view(torch.float8_e4m3fn)
    src = (pos - lens[:, None]).clamp(0, new - 1)
    fresh = x.float().gather(1, src[:, :, None, None].expand(-1, -1, h, d)).transpose(1, 2)  # (batch, heads, span, dim)
    fresh = torch.where(is_new[:, None, :, None], fresh, 0.0)
    blk = (pos[:, ::block] // block).clamp(max=scales.shape[2] - 1)[:, None].expand(-1, h, -1)
    e_old = scales.gather(2, blk).int() - 127
    need = _exponent(fresh.abs().view(b, h, -1, block, d).amax((-1, -2)), kind)
    has_old = is_old.view(b, -1, block).any(-1)[:, None]
    has_new = is_new.view(b, -1, block).any(-1)[:, None]
    e_new = torch.where(has_old, torch.maximum(need, e_old), need)
    e_new = torch.where(has_new, e_new, e_old)
    per = lambda e: _power(e).repeat_interleave(block, 2)[..., None]  # noqa: E731
    moved = _round(held.float() * (per(e_old) / per(e_new)), kind)
    keep = (e_new == e_old).repeat_interleave(block, 2)[..., None]
    old = torch.where(keep | ~is_old[:, None, :, None] | (e_new == 128).repeat_interleave(block, 2)[..., None], held.float(), moved)
    out = torch.where(is_new[:, None, :, None], _round(fresh / per(e_new), kind), old).to(DTYPE[kind])
    if kind == "int8":
        data.scatter_(2, at, out)
    else:
        data.view(torch.uint8).scatter_(2, at, out.view(torch.uint8))
    scales.scatter_(2, blk, (e_new + 127).to(torch.uint8))


def _values(data, scales, block):
    e = scales.int() - 127
    return data.float() * _power(e).repeat_interleave(block, 2)[:, :, :data.shape[2], None]


def _plain_read(data, scales, block, lens, start, length):
    """Tokens start[b] .. start[b] + length as (batch, length, heads, dim) bf16, 0 from lens[b] on."""
    b, h, cap, d = data.shape
    pos = start[:, None] + torch.arange(length, device=data.device)
    at = pos.clamp(max=cap - 1)[:, None].expand(-1, h, -1)
    raw = data.view(torch.uint8).gather(2, at[..., None].expand(-1, -1, -1, d)).view(data.dtype)
    x = raw.float() * _power(scales.gather(2, at // block).int() - 127)[..., None]
    return torch.where((pos < lens[:, None])[:, None, :, None], x, 0.0).transpose(1, 2).to(torch.bfloat16).contiguous()


def _plain_attend(s):
    case, lens, q = s["case"], s["lens"], s["q"]
    b, new, heads, d = q.shape
    hk = case["kv_heads"]
    if case["step"]:
        _plain_append(s["k8"], s["ks"], s["k"], lens, case["kind"], case["block"])
        _plain_append(s["v8"], s["vs"], s["v"], lens, case["kind"], case["block"])
    total = lens + (new if case["step"] else 0)
    keys, values = _values(s["k8"], s["ks"], case["block"]), _values(s["v8"], s["vs"], case["block"])
    rows = q.float().view(b, new, hk, heads // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    score = rows @ keys.transpose(-1, -2) / math.sqrt(d)  # (batch, kv_heads, group * new, capacity)
    at = total[:, None] - new + torch.arange(new, device=q.device)  # position of each query
    j = torch.arange(keys.shape[2], device=q.device)
    seen = (j <= at[..., None]) & (j < total[:, None, None])
    if case["window"]:
        seen &= j > at[..., None] - case["window"]
    seen = seen[:, None, None].expand(-1, hk, heads // hk, -1, -1).reshape(score.shape)
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    w = torch.where(seen, torch.exp(score - torch.where(top == -math.inf, 0.0, top)), 0.0)
    total_w = w.sum(-1, keepdim=True)
    held = torch.where((j < total[:, None])[:, None, :, None], values, 0.0)
    o = (w @ held) / torch.where(total_w == 0, 1.0, total_w)
    out = o.view(b, hk, heads // hk, new, d).permute(0, 3, 1, 2, 4).reshape(b, new, heads, d).to(torch.bfloat16)
    if not case["step"]:
        return out
    return [out, _plain_read(s["k8"], s["ks"], case["block"], total, lens, new),
            _plain_read(s["v8"], s["vs"], case["block"], total, lens, new)]


# ------------------------------------------------------------------------------- plain log probabilities
def _plain_logprobs(s):
    case, tokens = s["case"], s["tokens"]
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    ex = torch.exp(x - top)
    lse = top + torch.log(ex.sum(-1, keepdim=True))
    logp = x - lse
    p = torch.exp(logp)
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    out = [logp.gather(1, tokens[:, None])[:, 0], entropy]
    if case["top"]:
        values, index = torch.sort(x, dim=-1, descending=True, stable=True)
        out += [values[:, :case["top"]] - lse, index[:, :case["top"]].contiguous()]
    if case["grad"]:
        g = -p * s["g_logprob"][:, None]
        g -= torch.where(p > 0, p * (logp + entropy[:, None]), 0.0) * s["g_entropy"][:, None]
        if case["top"]:
            g -= p * s["g_top"].sum(-1, keepdim=True)
            g.scatter_add_(1, out[3], s["g_top"])
        g.scatter_add_(1, tokens[:, None], s["g_logprob"][:, None])
        out.append(g.to(s["logits"].dtype))
    return out


# ------------------------------------------------------------------------------- states and passes
def _tokens_data(g, shape):
    """Keys or values: normal, with a few channels of each head several times larger, rounded to bf16."""
    x = torch.randn(*shape, device="cuda", generator=g)
    wide = torch.rand(shape[-2:], device="cuda", generator=g) < 0.04
    return (x * torch.where(wide, 6.0, 1.0)).to(torch.bfloat16)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        x = torch.randn(rows, vocab, device="cuda", generator=g) * 2.0
        x += 6.0 * torch.rand(rows, vocab, device="cuda", generator=g).pow_(40)  # a few likely tokens a row
        tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
        if case["masked"]:  # a constrained vocabulary: most entries are excluded, the given token is not
            allowed = torch.rand(rows, vocab, device="cuda", generator=g) < 0.01
            allowed.scatter_(1, tokens[:, None], True)
            x = torch.where(allowed, x, -math.inf)
        s = {"case": case, "logits": x.to(torch.bfloat16 if case["kind"] == "bf16" else torch.float32), "tokens": tokens}
        if case["grad"]:
            s["g_logprob"] = torch.randn(rows, device="cuda", generator=g) / rows
            s["g_entropy"] = torch.full((rows,), -0.01 / rows, device="cuda")
            s["g_top"] = torch.randn(rows, case["top"], device="cuda", generator=g) / rows
        return s
    b, new, hk, d, kind, block = (case[k] for k in ("batch", "new", "kv_heads", "dim", "kind", "block"))
    cap = _capacity(case)
    s = {"case": case, "lens": torch.tensor(_lengths(case, seed), dtype=torch.int32, device="cuda")}
    for name in ("k", "v"):
        held = [_quantise(_tokens_data(g, (min(8, b - i), cap, hk, d)).transpose(1, 2), kind, block) for i in range(0, b, 8)]
        s[name + "8"] = torch.cat([h[0].view(torch.uint8) for h in held]).view(DTYPE[kind])
        s[name + "s"] = torch.cat([h[1] for h in held])
        del held
        s[name] = _tokens_data(g, (b, new, hk, d))
    if case["op"] == "attend":
        s["q"] = torch.randn(b, new, case["heads"], d, device="cuda", generator=g).to(torch.bfloat16)
        if not case["step"]:
            del s["k"], s["v"]
    return s


def _own_cache(s):
    from myk_llm_b200 import ops

    return ops, ops.KVCache8(s["k8"], s["v8"], s["ks"], s["vs"], s["case"]["block"])


def run(s):
    case = s["case"]
    if case["op"] == "logprobs":
        if not own:
            return _plain_logprobs(s)
        from myk_llm_b200 import ops

        if not case["grad"]:
            r = ops.token_logprobs(s["logits"], s["tokens"], top=case["top"])
            return [r.logprobs, r.entropy] + ([r.top_logprobs, r.top_tokens] if case["top"] else [])
        x = s["logits"].detach().requires_grad_()
        r = ops.token_logprobs(x, s["tokens"], top=case["top"])
        given, grads = [r.logprobs, r.entropy], [s["g_logprob"], s["g_entropy"]]
        if case["top"]:
            given, grads = given + [r.top_logprobs], grads + [s["g_top"]]
        gx, = torch.autograd.grad(given, x, grads)
        return [v.detach() for v in given] + ([r.top_tokens] if case["top"] else []) + [gx]
    if case["op"] == "cache":
        total, length = s["lens"] + case["new"], case["ctx"] + case["new"]
        if own:
            ops, cache = _own_cache(s)
            ops.kv8_append(cache, s["k"], s["v"], cache_seqlens=s["lens"])
            return list(ops.kv8_read(cache, cache_seqlens=total, length=length))
        _plain_append(s["k8"], s["ks"], s["k"], s["lens"], case["kind"], case["block"])
        _plain_append(s["v8"], s["vs"], s["v"], s["lens"], case["kind"], case["block"])
        start = torch.zeros_like(s["lens"])
        return [_plain_read(s["k8"], s["ks"], case["block"], total, start, length),
                _plain_read(s["v8"], s["vs"], case["block"], total, start, length)]
    if not own:
        return _plain_attend(s)
    ops, cache = _own_cache(s)
    window = (case["window"] - 1, 0) if case["window"] else (-1, -1)
    out = ops.flash_attn_with_kvcache8(s["q"], cache, s.get("k"), s.get("v"), cache_seqlens=s["lens"], causal=True,
                                       window_size=window)
    if not case["step"]:
        return out
    return [out, *ops.kv8_read(cache, cache_seqlens=s["lens"] + case["new"], start=s["lens"], length=case["new"])]


# ------------------------------------------------------------------------------- definitions in 64 bits
def _exact_store(x, old, old_exp, at, n_new, case):
    """One sequence and tensor in place: x (new, heads, dim) fp64 written at position `at` of old (heads, cap, dim), the
    fp64 8-bit values, with the blocks' exponents old_exp (heads, blocks)."""
    block, kind = case["block"], case["kind"]
    qmax = QMAX[kind]
    for blk in range(at // block, (at + n_new - 1) // block + 1):
        lo, hi = max(at, blk * block), min(at + n_new, (blk + 1) * block)
        rows = x[lo - at:hi - at].transpose(0, 1)  # (heads, rows, dim)
        amax = rows.abs().amax((1, 2))
        e = torch.log2(amax.clamp(min=2.0 ** -120) / qmax).ceil()
        e = torch.where(amax > qmax * torch.exp2(e), e + 1, torch.where(amax <= qmax * torch.exp2(e - 1), e - 1, e)).clamp(min=-100)
        if lo > blk * block:
            e = torch.maximum(e, old_exp[:, blk])
            shift = torch.exp2(old_exp[:, blk] - e)[:, None, None]
            old[:, blk * block:lo] = _exact_round(old[:, blk * block:lo] * shift, kind)
        old_exp[:, blk] = e
        old[:, lo:hi] = _exact_round(rows / torch.exp2(e)[:, None, None], kind)


def _exact_round(x, kind):
    if kind == "int8":
        return x.round()
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)  # spacing of e4m3 at |x|
    return (x / step).round() * step


def _exact_cache(s):
    """fp64 keys and values (batch of (heads, cap, dim)) after the new tokens, and the lengths."""
    case, lens = s["case"], s["lens"].tolist()
    both, stored = [], case["op"] == "cache" or case["step"]
    for name in ("k", "v"):
        got = []
        for i, n in enumerate(lens):
            q = s[name + "8"][i].to(torch.float32).double()
            e = s[name + "s"][i].double() - 127
            if stored:
                _exact_store(s[name][i].double(), q, e, n, case["new"], case)
            got.append(q * torch.exp2(e).repeat_interleave(case["block"], 1)[:, :q.shape[1], None])
        both.append(got)
    return both[0], both[1], [n + (case["new"] if stored else 0) for n in lens]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        rows = []
        for lo in range(0, case["rows"], 512):
            x, t = s["logits"][lo:lo + 512].double(), s["tokens"][lo:lo + 512]
            logp = torch.log_softmax(x, -1)
            plogp = torch.special.xlogy(logp.exp(), logp.exp())
            entropy = -plogp.sum(-1)
            one = [logp[torch.arange(len(t)), t], entropy]
            if case["top"]:
                order = torch.argsort(x, dim=-1, descending=True, stable=True)[:, :case["top"]]
                one += [logp.gather(1, order), order]
            if case["grad"]:
                p, gl = logp.exp(), s["g_logprob"][lo:lo + 512].double()
                extra = torch.zeros_like(p)
                extra[torch.arange(len(t)), t] = gl
                if case["top"]:
                    gt = s["g_top"][lo:lo + 512].double()
                    extra.scatter_add_(1, order, gt)
                    gl = gl + gt.sum(-1)
                one.append(extra - p * gl[:, None] - s["g_entropy"][lo:lo + 512].double()[:, None] * (plogp + p * entropy[:, None]))
            rows.append(one)
        return [torch.cat(part) for part in zip(*rows)]
    keys, values, total = _exact_cache(s)
    b, new = case["batch"], case["new"]
    if case["op"] == "cache":
        out = []
        for held in (keys, values):
            x = torch.zeros(b, case["ctx"] + new, case["kv_heads"], case["dim"], dtype=torch.float64, device="cuda")
            for i, n in enumerate(total):
                x[i, :n] = held[i][:, :n].transpose(0, 1)
            out.append(x)
        return out
    out = torch.zeros(b, new, case["heads"], case["dim"], dtype=torch.float64, device="cuda")
    group = case["heads"] // case["kv_heads"]
    for i, n in enumerate(total):
        at = torch.arange(n - new, n, device="cuda")
        first = max(0, n - new - case["window"] + 1) if case["window"] else 0
        j = torch.arange(first, n, device="cuda")
        hidden = j[None] > at[:, None]
        if case["window"]:
            hidden |= j[None] <= at[:, None] - case["window"]
        live = ~hidden.all(-1)
        for h in range(case["heads"]):
            k, v = keys[i][h // group, first:n], values[i][h // group, first:n]
            score = (s["q"][i, :, h].double() @ k.T / math.sqrt(case["dim"])).masked_fill(hidden, -math.inf)
            out[i, live, h] = torch.softmax(score[live], -1) @ v
    if not case["step"]:
        return out
    back = [torch.stack([held[i][:, n - new:n].transpose(0, 1) for i, n in enumerate(total)]) for held in (keys, values)]
    return [out, *back]
