"""8-bit key/value cache and the attention over it, against fp64 statements written here.

The cache must be exact: block scales are powers of two, so quantising is one rounding of an
exactly scaled value and reading back is exact; both are compared for equality.  Attention:
weights are rounded to f16 (unit roundoff 2^-11, their sum is not) and the output to bf16
(2^-8), the rest is fp32, so each output may be off by 2^-8 |o| + 2^-10 sum p |v|; where the
cache is read back for the prefill kernel the weights are bf16 and the second term is
2^-7 sum p |v|.
"""

import math

import pytest
import torch

E4M3, INT8 = torch.float8_e4m3fn, torch.int8


# ------------------------------------------------------------------------- fp64 statements
def _round64(x, dtype):
    if dtype == INT8:
        return x.round()
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (x / step).round() * step


class Plain:
    """One tensor of a cache: fp64 8-bit values (B, H, cap, D), fp64 exponents (B, H, blocks)."""

    def __init__(self, b, h, cap, d, dtype, block, device):
        self.q = torch.zeros(b, h, cap, d, dtype=torch.float64, device=device)
        self.e = torch.full((b, h, -(-cap // block)), -127.0, dtype=torch.float64, device=device)
        self.dtype, self.block, self.qmax = dtype, block, 127.0 if dtype == INT8 else 448.0

    def append(self, x, lens):
        for b, n in enumerate(lens):
            for h in range(x.shape[2]):
                t = 0
                while t < x.shape[1] and n + t < self.q.shape[2]:
                    blk = (n + t) // self.block
                    m = min(x.shape[1], (blk + 1) * self.block - n, self.q.shape[2] - n)
                    rows = x[b, t:m, h].double()
                    a = rows.abs().max().item()
                    if not math.isfinite(a):
                        e = math.inf
                    else:
                        e = -100.0
                        while a > self.qmax * 2.0 ** e:
                            e += 1
                    first = blk * self.block
                    if n + t > first:
                        old = self.e[b, h, blk].item()
                        e = max(e, old)
                        if e > old and e != math.inf:
                            self.q[b, h, first:n + t] = _round64(self.q[b, h, first:n + t] * 2.0 ** (old - e), self.dtype)
                    self.e[b, h, blk] = e
                    self.q[b, h, n + t:n + m] = 0 if e == math.inf else _round64(rows * 2.0 ** -e, self.dtype)
                    t = m

    def values(self):
        s = torch.where(self.e == math.inf, math.nan, torch.exp2(self.e)).repeat_interleave(self.block, 2)
        return self.q * s[:, :, :self.q.shape[2], None]


def _read(plain, lens, start, length):
    v = plain.values()
    out = torch.zeros(v.shape[0], length, v.shape[1], v.shape[3], dtype=torch.float64, device=v.device)
    for b, n in enumerate(lens):
        lo, hi = start[b], min(start[b] + length, n, v.shape[2])
        if lo < hi:
            out[b, :hi - lo] = v[b, :, lo:hi].transpose(0, 1)
    return out


def _attend(q, keys, values, lens, left, right, scale):
    """fp64 output and sum p |v| of q (B, L, H, D) over (B, Hkv, cap, D)."""
    b, new, heads, d = q.shape
    group = heads // keys.shape[1]
    out = torch.zeros(b, new, heads, d, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    for i, n in enumerate(lens):
        at = torch.arange(n - new, n, device=q.device)[:, None]
        j = torch.arange(n, device=q.device)[None]
        seen = torch.ones(new, n, dtype=torch.bool, device=q.device)
        if right >= 0:
            seen &= j <= at + right
        if left >= 0:
            seen &= j >= at - left
        live = seen.any(-1)
        if not bool(live.any()):
            continue
        for h in range(heads):
            k, v = keys[i, h // group, :n], values[i, h // group, :n]
            s = (q[i, :, h].double() @ k.T * scale).masked_fill(~seen, -math.inf)[live]
            p = torch.softmax(s, -1)
            p = torch.where(seen[live], p, 0.0)
            held = torch.where(seen.any(0)[:, None], v, 0.0)
            out[i, live, h], mag[i, live, h] = p @ held, p @ held.abs()
    return out, mag


def _data(shape, seed, device, spread=True):
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(*shape, generator=g, device=device)
    if spread:  # magnitudes that rise and fall along the sequence, so blocks are moved to new scales
        x = x * torch.exp2(torch.randint(-3, 4, (*shape[:2], 1, 1), generator=g, device=device).float())
    return x.to(torch.bfloat16)


def _cache(b, cap, h, d, dtype, block, device):
    from myk_llm_b200 import ops

    return ops.kv8_cache(b, cap, h, d, dtype=dtype, block=block, device=device), \
        [Plain(b, h, cap, d, dtype, block, device) for _ in range(2)]


def _steps(device, dtype, block, d, h, steps, lens, cap):
    from myk_llm_b200 import ops

    cache, plain = _cache(len(lens), cap, h, d, dtype, block, device)
    lens = list(lens)
    for i, new in enumerate(steps):
        k, v = _data((len(lens), new, h, d), 10 + i, device), _data((len(lens), new, h, d), 50 + i, device)
        ops.kv8_append(cache, k, v, cache_seqlens=torch.tensor(lens, dtype=torch.int32, device=device))
        plain[0].append(k, lens)
        plain[1].append(v, lens)
        lens = [n + new for n in lens]
    t = torch.tensor(lens, dtype=torch.int32, device=device)
    for start, length in ((0, None), (0, 0), (3, min(17, cap - 3))):
        got = ops.kv8_read(cache, cache_seqlens=t, start=start, length=length)
        for g, p in zip(got, plain):
            want = _read(p, lens, [start] * len(lens), cap - start if length is None else length)
            assert g.dtype == torch.bfloat16 and torch.equal(g.double(), want)
    each = torch.tensor([max(0, n - 5) for n in lens], dtype=torch.int32, device=device)
    for g, p in zip(ops.kv8_read(cache, cache_seqlens=t, start=each, length=9), plain):
        assert torch.equal(g.double(), _read(p, lens, each.tolist(), 9))


APPEND = [
    # (block, head_dim, kv_heads, tokens of each call, lengths before, capacity)
    (16, 64, 4, (1, 1, 3, 40), (0, 5, 15, 16), 77),
    (16, 128, 1, (33, 1, 2), (0, 31), 64),
    (1, 128, 2, (1, 7, 100), (0, 1, 2), 128),
    (8, 64, 3, (20, 5, 1, 1), (3,), 40),
    (64, 128, 2, (100, 1, 1, 60), (0, 63, 64), 301),
    (128, 64, 1, (1, 300, 2), (127, 1), 500),
    (1024, 64, 2, (5, 700), (0, 1000), 2000),
    (32, 128, 2, (50, 50), (0, 30), 64),  # the second call passes the capacity
]


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("case", APPEND)
def test_append_and_read_cpu(case, dtype):
    block, d, h, steps, lens, cap = case
    _steps("cpu", dtype, block, d, h, steps, lens, cap)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("case", APPEND)
def test_append_and_read_gpu(case, dtype):
    block, d, h, steps, lens, cap = case
    _steps("cuda", dtype, block, d, h, steps, lens, cap)


def _special(device, dtype):
    """Zeros, the type's extremes, infinities and NaN."""
    from myk_llm_b200 import ops

    cache, plain = _cache(1, 48, 1, 64, dtype, 16, device)
    k = _data((1, 40, 1, 64), 1, device)
    v = _data((1, 40, 1, 64), 2, device)
    k[0, :16] = 0
    k[0, 16, 0, :4] = torch.tensor([2.0 ** 120, -2.0 ** 120, 1e-38, 448.0])
    v[0, 5, 0, 3] = math.nan
    v[0, 20, 0, 9] = -math.inf
    v[0, 32:, 0] = torch.finfo(torch.bfloat16).tiny  # far below the smallest scale
    lens = torch.zeros(1, dtype=torch.int32, device=device)
    ops.kv8_append(cache, k, v, cache_seqlens=lens)
    plain[0].append(k, [0])
    plain[1].append(v, [0])
    got = ops.kv8_read(cache, cache_seqlens=lens + 40, length=40)
    for g, p in zip(got, plain):
        assert torch.equal(torch.nan_to_num(g.double(), nan=-7.0), torch.nan_to_num(_read(p, [40], [0], 40), nan=-7.0))
    assert got[1][0, :32].isnan().all() and not got[1][0, 32:].isnan().any()
    # written again from a block's first token, the block is sound again
    ops.kv8_append(cache, k[:, :16], k[:, :16], cache_seqlens=lens)
    assert torch.equal(ops.kv8_read(cache, cache_seqlens=lens + 40, length=16)[1], torch.zeros_like(k[:, :16]))


@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_append_special_values_cpu(dtype):
    _special("cpu", dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_append_special_values_gpu(dtype):
    _special("cuda", dtype)


def _full(device, dtype):
    """Tokens at and past the capacity are dropped, also where the last block is a partial one; the rest is untouched."""
    from myk_llm_b200 import ops

    for cap, block in ((40, 16), (8, 16), (33, 32), (20, 1), (64, 16)):
        b, h, d = 5, 2, 64
        lens = [cap, cap + 1, cap + 100, cap - 2, 0]
        cache, plain = _cache(b, cap, h, d, dtype, block, device)
        first = [_data((b, cap, h, d), s, device) for s in (1, 2)]
        more = [_data((b, 7, h, d), s, device) * 64 for s in (3, 4)]  # would raise every scale
        zero = torch.zeros(b, dtype=torch.int32, device=device)
        ops.kv8_append(cache, *first, cache_seqlens=zero)
        ops.kv8_append(cache, *more, cache_seqlens=torch.tensor(lens, dtype=torch.int32, device=device))
        for got, p, x, y in zip(ops.kv8_read(cache, cache_seqlens=zero + cap), plain, first, more):
            p.append(x, [0] * b)
            p.append(y, lens)
            assert torch.equal(got.double(), _read(p, [cap] * b, [0] * b, cap))


@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_append_past_the_capacity_cpu(dtype):
    _full("cpu", dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_append_past_the_capacity_gpu(dtype):
    _full("cuda", dtype)


@pytest.mark.gpu
def test_append_strided_and_split_calls():
    """New tokens as slices of a fused projection (rows apart, some not 16-byte aligned) and,
    with block 1, the same cache whatever the calls."""
    from myk_llm_b200 import ops

    b, n, h, d = 2, 37, 2, 64
    qkv = _data((b, n, 6, d), 3, "cuda").view(b, n, 6 * d)
    k, v = qkv[..., 2 * d:4 * d].view(b, n, h, d), qkv[..., 4 * d:].view(b, n, h, d)
    wide = _data((b, n, 1, h * d + 3), 4, "cuda")[:, :, 0]
    odd = torch.as_strided(wide, (b, n, h, d), (n * (h * d + 3), h * d + 3, d, 1), 1)
    zero = torch.zeros(b, dtype=torch.int32, device="cuda")
    for kk, vv in ((k, v), (odd, v), (k.transpose(2, 3).contiguous().transpose(2, 3), odd)):
        whole, parts = (ops.kv8_cache(b, 64, h, d, block=1, device="cuda") for _ in range(2))
        ops.kv8_append(whole, kk, vv, cache_seqlens=zero)
        for lo, hi in ((0, 1), (1, 20), (20, 37)):
            ops.kv8_append(parts, kk[:, lo:hi], vv[:, lo:hi], cache_seqlens=zero.long() + lo)
        plain = Plain(b, h, 64, d, E4M3, 1, "cuda")
        plain.append(kk, [0, 0])
        assert torch.equal(whole.keys.view(torch.uint8), parts.keys.view(torch.uint8))
        assert torch.equal(whole.values.view(torch.uint8), parts.values.view(torch.uint8))
        assert torch.equal(whole.key_scales, parts.key_scales) and torch.equal(whole.value_scales, parts.value_scales)
        assert torch.equal(ops.kv8_read(whole, cache_seqlens=zero + n, length=n)[0].double(), _read(plain, [n, n], [0, 0], n))


# ------------------------------------------------------------------------- attention
ATTEND = [
    # (lengths before, new, appended, heads, kv_heads, d, block, causal, window)
    ((1,), 1, False, 1, 1, 64, 16, True, (-1, -1)),
    ((0, 1, 2, 31, 32, 33), 1, False, 4, 2, 64, 16, True, (-1, -1)),
    ((0, 7, 300), 1, True, 4, 1, 128, 16, True, (-1, -1)),
    ((2048,), 1, False, 16, 4, 64, 16, True, (-1, -1)),
    ((1500, 3, 0, 700), 3, True, 16, 4, 64, 16, True, (-1, -1)),
    ((513, 100, 2), 1, False, 8, 2, 128, 64, True, (511, 0)),
    ((90, 1000), 5, True, 6, 2, 64, 1, True, (40, 0)),
    ((77, 4), 9, True, 8, 1, 128, 8, True, (-1, -1)),          # 72 rows: five row tiles
    ((77, 4), 6, True, 8, 1, 128, 8, True, (-1, -1)),          # 48 rows: three row tiles
    ((3, 10), 8, False, 2, 2, 64, 32, True, (-1, -1)),         # more queries than keys: empty rows
    ((200, 50), 4, False, 4, 4, 128, 16, False, (-1, -1)),     # bidirectional
    ((200, 50), 4, False, 4, 4, 64, 4, False, (20, 2)),
    ((5000,), 1, False, 3, 1, 128, 128, True, (-1, -1)),
    ((300, 0), 130, True, 4, 2, 64, 16, True, (100, 0)),
    ((40, 41), 1, False, 64, 2, 64, 2, True, (-1, -1)),        # 32 heads a KV head
]


def _attend_case(device, case, dtype, seed=0):
    from myk_llm_b200 import ops

    lens, new, step, heads, hk, d, block, causal, window = case
    b, cap = len(lens), max(lens) + new + 5
    cache, plain = _cache(b, cap, hk, d, dtype, block, device)
    # fill past the lengths: what lies there must not be seen
    for name, p, s in (("keys", plain[0], 1), ("values", plain[1], 2)):
        p.append(_data((b, cap, hk, d), seed + s, device, spread=False), [0] * b)
    ops.kv8_append(cache, _data((b, cap, hk, d), seed + 1, device, spread=False),
                   _data((b, cap, hk, d), seed + 2, device, spread=False),
                   cache_seqlens=torch.zeros(b, dtype=torch.int32, device=device))
    q = _data((b, new, heads, d), seed + 3, device) * 0.5
    k, v = _data((b, new, hk, d), seed + 4, device, spread=False), _data((b, new, hk, d), seed + 5, device, spread=False)
    t = torch.tensor(lens, dtype=torch.int32, device=device)
    out = ops.flash_attn_with_kvcache8(q, cache, *((k, v) if step else ()), cache_seqlens=t, causal=causal,
                                       window_size=window)
    total = list(lens)
    if step:
        plain[0].append(k, lens)
        plain[1].append(v, lens)
        total = [n + new for n in lens]
    left, right = window[0], 0 if causal else window[1]
    want, mag = _attend(q, plain[0].values(), plain[1].values(), total, left, right, 1 / math.sqrt(d))
    assert out.dtype == q.dtype and out.shape == q.shape
    weight = 2.0 ** -7 if heads // hk * new > 64 else 2.0 ** -10
    off = (out.double() - want).abs()
    assert bool((off <= 2.0 ** -8 * want.abs() + weight * mag).all()), (off - 2.0 ** -8 * want.abs() - weight * mag).max()
    for i, n in enumerate(total):  # queries before the first token
        if causal and n < new:
            assert not out[i, :new - n].any()


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("case", ATTEND)
def test_attend_cpu(case, dtype):
    _attend_case("cpu", case, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("case", ATTEND)
def test_attend_gpu(case, dtype):
    from myk_llm_b200 import ops

    _attend_case("cuda", case, dtype)
    assert ops.ext().take_status() == 0


PREFILL = [  # wide enough that the cache is read back for the prefill kernel
    ((100, 0, 3000), 600, True, 16, 4, 128, 16, True, (-1, -1)),
    ((700, 31), 601, False, 16, 4, 64, 8, True, (-1, -1)),
    ((100,), 1030, True, 8, 2, 128, 64, True, (200, 0)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("case", PREFILL)
def test_attend_prefill_gpu(case, dtype):
    from myk_llm_b200 import ops

    _attend_case("cuda", case, dtype)
    assert ops.ext().take_status() == 0


@pytest.mark.gpu
def test_prefill_nan_only_where_seen():
    """As test_attend_nan_only_where_seen, through the prefill kernel: earlier queries of the same
    tile and queries whose window has passed the block stay finite, for a bad key or value."""
    from myk_llm_b200 import ops

    b, n, new, hk, d = 2, 900, 700, 2, 64
    q = _data((b, new, 8, d), 3, "cuda")
    zero = torch.zeros(b, dtype=torch.int32, device="cuda")
    at = torch.arange(n - new, n, device="cuda")
    for bad in (0, 1):
        kv = [_data((b, n, hk, d), 1, "cuda"), _data((b, n, hk, d), 2, "cuda")]
        kv[bad][0, 300, 1, 5] = math.nan  # tokens 288 .. 303 of sequence 0, head 1
        cache = ops.kv8_cache(b, 960, hk, d, block=16, device="cuda")
        ops.kv8_append(cache, *kv, cache_seqlens=zero)
        for left in (-1, 99):
            out = ops.flash_attn_with_kvcache8(q, cache, cache_seqlens=zero + n, causal=True, window_size=(left, 0))
            sees = (at >= 288) & ((at - left <= 303) if left >= 0 else (at >= 0))
            assert out[0, sees, 4:].isnan().all() and not out[0, ~sees, 4:].isnan().any()
            assert not out[0, :, :4].isnan().any() and not out[1].isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_attend_many_sequences(d):
    """More sequences than threads of a CTA, most of them short or empty."""
    lens = [(7 * i * i + i) % 97 if i % 3 else 0 for i in range(300)]
    lens[150] = 1900
    _attend_case("cuda", (tuple(lens), 1, False, 4, 2, d, 16, True, (-1, -1)), E4M3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_attend_scales_far_apart(dtype):
    """Blocks whose keys and values differ by 2^40, weights concentrated on a small-valued block,
    large and tiny queries, a negative softmax scale."""
    from myk_llm_b200 import ops

    b, n, hk, d = 1, 96, 1, 64
    k, v = _data((b, n, hk, d), 1, "cuda", spread=False), _data((b, n, hk, d), 2, "cuda", spread=False)
    v[:, 16:32] *= 2.0 ** 20
    v[:, 32:48] *= 2.0 ** -20
    k[:, 48:64] *= 2.0 ** -30
    v[:, 64:80] = 0
    cache, plain = _cache(b, n, hk, d, dtype, 16, "cuda")
    zero = torch.zeros(b, dtype=torch.int32, device="cuda")
    ops.kv8_append(cache, k, v, cache_seqlens=zero)
    plain[0].append(k, [0])
    plain[1].append(v, [0])
    q = torch.cat([_data((b, 1, 1, d), 3, "cuda", spread=False) * s for s in (1.0, 2.0 ** 4, 2.0 ** -60, 0.0)], 2)
    q = torch.cat([q, 4 * k[:, 40:41].expand(-1, -1, 4, -1)], 2)  # looks at a token with small values
    for scale in (0.125, -0.125, 0.0):
        out = ops.flash_attn_with_kvcache8(q, cache, cache_seqlens=zero + n, causal=True, softmax_scale=scale)
        want, mag = _attend(q, plain[0].values(), plain[1].values(), [n], -1, 0, scale)
        assert bool(((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * mag).all())


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 20])
def test_attend_nan_only_where_seen(new):
    """A block holding a NaN reaches the queries that see it and no others; NaN bytes past the
    length are never read."""
    from myk_llm_b200 import ops

    b, n, hk, d = 2, 200, 2, 64
    cache = ops.kv8_cache(b, 256, hk, d, block=16, device="cuda")
    cache.keys.view(torch.uint8).fill_(0x7F)
    cache.values.view(torch.uint8).fill_(0x7F)
    cache.key_scales.fill_(255)
    cache.value_scales.fill_(255)
    k, v = _data((b, n, hk, d), 1, "cuda"), _data((b, n, hk, d), 2, "cuda")
    v[0, 3, 1, 5] = math.nan  # sequence 0, head 1, block 0
    zero = torch.zeros(b, dtype=torch.int32, device="cuda")
    ops.kv8_append(cache, k, v, cache_seqlens=zero)
    q = _data((b, new, 8, d), 3, "cuda")
    out = ops.flash_attn_with_kvcache8(q, cache, cache_seqlens=zero + n, causal=True)
    assert out[0, :, 4:].isnan().all() and not out[0, :, :4].isnan().any() and not out[1].isnan().any()
    out = ops.flash_attn_with_kvcache8(q, cache, cache_seqlens=zero + n, causal=True, window_size=(99, 0))
    assert not out.isnan().any()


@pytest.mark.gpu
def test_attend_strided_queries_streams_and_repeats():
    """Queries as a slice of a fused projection; a call on another stream; the same bits again."""
    from myk_llm_b200 import ops

    b, n, hk, d = 3, 700, 2, 128
    cache = ops.kv8_cache(b, 800, hk, d, dtype=INT8, block=32, device="cuda")
    zero = torch.zeros(b, dtype=torch.int32, device="cuda")
    ops.kv8_append(cache, _data((b, n, hk, d), 1, "cuda"), _data((b, n, hk, d), 2, "cuda"), cache_seqlens=zero)
    fused = _data((b, 2, 12, d), 3, "cuda")
    q = fused[:, :, 2:10]
    kw = dict(cache_seqlens=zero + n, causal=True)
    out = ops.flash_attn_with_kvcache8(q.contiguous(), cache, **kw)
    assert torch.equal(out, ops.flash_attn_with_kvcache8(q, cache, **kw))
    odd = torch.as_strided(_data((1, 1, 1, b * 2 * 8 * d + 8), 4, "cuda").flatten(), q.shape,
                           (2 * 8 * d, 8 * d, d, 1), 1)
    odd.copy_(q)
    assert torch.equal(out, ops.flash_attn_with_kvcache8(odd, cache, **kw))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        again = [ops.flash_attn_with_kvcache8(q, cache, **kw) for _ in range(3)]
    s.synchronize()
    assert all(torch.equal(out, a) for a in again)


@pytest.mark.gpu
def test_attend_in_a_cuda_graph():
    """Append + attend captured once and replayed while the lengths advance."""
    from myk_llm_b200 import ops

    b, hk, d, heads, cap = 2, 2, 64, 8, 400
    x = [_data((b, 300, hk, d), s, "cuda") for s in (1, 2)]
    qs = _data((b, 300, heads, d), 3, "cuda")
    caches = [ops.kv8_cache(b, cap, hk, d, device="cuda") for _ in range(2)]
    lens = [torch.tensor([0, 90], dtype=torch.int32, device="cuda") for _ in range(2)]
    for c in caches:
        ops.kv8_append(c, x[0][:, :90], x[1][:, :90], cache_seqlens=torch.zeros_like(lens[0]))
    q, k, v = qs[:, :1].clone(), x[0][:, :1].clone(), x[1][:, :1].clone()

    def step(i):
        out = ops.flash_attn_with_kvcache8(q, caches[i], k, v, cache_seqlens=lens[i], causal=True)
        lens[i] += 1
        return out

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(0)
    torch.cuda.current_stream().wait_stream(s)
    step(1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(0)
    for t in range(1, 60):
        q.copy_(qs[:, t:t + 1])
        k.copy_(x[0][:, t:t + 1])
        v.copy_(x[1][:, t:t + 1])
        graph.replay()
        assert torch.equal(out, step(1))
    assert torch.equal(lens[0], lens[1])


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A cache of more than 2^32 elements: the last sequence's tokens."""
    from myk_llm_b200 import ops

    b, cap, hk, d = 9, 1 << 20, 4, 128  # 4.8e9 elements each for keys and values
    cache = ops.kv8_cache(b, cap, hk, d, block=64, device="cuda")
    n = 3000
    lens = torch.zeros(b, dtype=torch.int32, device="cuda")
    lens[-1] = cap - n
    k, v = _data((b, n, hk, d), 1, "cuda", spread=False), _data((b, n, hk, d), 2, "cuda", spread=False)
    ops.kv8_append(cache, k, v, cache_seqlens=lens)
    plain = [Plain(1, hk, n + 24, d, E4M3, 64, "cuda") for _ in range(2)]  # (cap - n) % 64 == 8
    first = (cap - n) % 64
    for p, x in zip(plain, (k, v)):
        p.append(x[-1:], [first])
    got = ops.kv8_read(cache, cache_seqlens=lens + n, start=lens, length=n)
    for g, p in zip(got, plain):
        assert torch.equal(g[-1].double(), p.values()[0, :, first:first + n].transpose(0, 1))
    q = _data((b, 1, 16, d), 3, "cuda")
    out = ops.flash_attn_with_kvcache8(q, cache, cache_seqlens=lens + n, causal=True, window_size=(n - 1, 0))
    want, mag = _attend(q[-1:], plain[0].values()[:, :, first:], plain[1].values()[:, :, first:], [n], n - 1, 0,
                        1 / math.sqrt(d))
    assert bool(((out[-1:].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * mag).all())


SCALES = [  # (lengths before, new, appended, heads, kv_heads, d, block, window): wide enough for the prefill kernel
    ((100, 0, 700), 600, True, 8, 2, 64, 16, (-1, -1)),
    ((300, 41), 515, False, 8, 2, 128, 8, (99, 0)),
    ((900,), 1100, True, 12, 4, 64, 64, (1200, 0)),  # an odd number of query heads a KV head
]


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [-0.125, 0.0])
@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("case", SCALES)
def test_attend_prefill_scale_not_positive(case, dtype, scale):
    """Negative and zero softmax scales in calls as wide as a prompt, under causal and window masks."""
    from myk_llm_b200 import ops

    lens, new, step, heads, hk, d, block, window = case
    b, cap = len(lens), max(lens) + new + 5
    cache, plain = _cache(b, cap, hk, d, dtype, block, "cuda")
    held = [_data((b, cap, hk, d), s, "cuda", spread=False) for s in (1, 2)]
    zero = torch.zeros(b, dtype=torch.int32, device="cuda")
    ops.kv8_append(cache, *held, cache_seqlens=zero)
    for p, x in zip(plain, held):
        p.append(x, [0] * b)
    q = _data((b, new, heads, d), 3, "cuda") * 0.5
    kv = [_data((b, new, hk, d), s, "cuda", spread=False) for s in (4, 5)] if step else []
    out = ops.flash_attn_with_kvcache8(q, cache, *kv, cache_seqlens=zero + torch.tensor(lens, device="cuda"), causal=True,
                                       window_size=window, softmax_scale=scale)
    for p, x in zip(plain, kv):
        p.append(x, lens)
    total = [n + new if step else n for n in lens]
    want, mag = _attend(q, plain[0].values(), plain[1].values(), total, window[0], 0, scale)
    assert bool(((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -7 * mag).all())
    assert ops.ext().take_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("new", [4, 600])
def test_attend_query_layouts(new):
    """Queries laid out head by head, as a chunk of a longer batch of tokens, as heads of a fused projection and
    shared by the batch, for few and for many rows: the same bits as contiguous ones, and the new tokens in the cache."""
    from myk_llm_b200 import ops

    b, n, hk, heads, d = 2, 300, 2, 8, 64
    k, v = (_data((b, n + new, hk, d), s, "cuda") for s in (1, 2))
    zero = torch.zeros(b, dtype=torch.int32, device="cuda")
    q = _data((b, new, heads, d), 3, "cuda")

    def call(x, window):
        cache = ops.kv8_cache(b, n + new, hk, d, device="cuda")
        ops.kv8_append(cache, k[:, :n], v[:, :n], cache_seqlens=zero)
        out = ops.flash_attn_with_kvcache8(x, cache, k[:, n:], v[:, n:], cache_seqlens=zero + n, causal=True,
                                           window_size=window)
        return out, *ops.kv8_read(cache, cache_seqlens=zero + n + new)

    wide = torch.zeros(b, new + 70, heads, d, dtype=torch.bfloat16, device="cuda")
    wide[:, 33:33 + new] = q
    fused = torch.zeros(b, new, heads + 2 * hk, d, dtype=torch.bfloat16, device="cuda")
    fused[:, :, :heads] = q
    gaps = torch.zeros(b, new, heads, 2 * d, dtype=torch.bfloat16, device="cuda")
    gaps[..., :d] = q
    layouts = [q.transpose(1, 2).contiguous().transpose(1, 2), wide[:, 33:33 + new], fused[:, :, :heads], gaps[..., :d],
               q.transpose(0, 1).contiguous().transpose(0, 1), q.transpose(2, 3).contiguous().transpose(2, 3)]
    for window in ((-1, -1), (99, 0)):
        want = call(q, window)
        for x in layouts:
            assert not x.is_contiguous() and torch.equal(x, q)
            assert all(torch.equal(a, c) for a, c in zip(call(x, window), want))
        want = call(q[:1].repeat(b, 1, 1, 1), window)
        assert all(torch.equal(a, c) for a, c in zip(call(q[:1].expand(b, -1, -1, -1), window), want))
    assert ops.ext().take_status() == 0


def _bad_blocks(device, new):
    """NaN exactly for the queries that see a bad block, for a bad key and a bad value, with and without a window,
    and the other rows as if the block were sound."""
    from myk_llm_b200 import ops

    b, n, hk, d = 2, 64, 2, 64
    q = _data((b, new, 4, d), 3, device) * 0.5
    zero = torch.zeros(b, dtype=torch.int32, device=device)
    at = torch.arange(n - new, n, device=device)
    for bad, token in ((0, 40), (1, 40), (0, 63), (1, 63), (0, 3), (1, 3)):
        kv = [_data((b, n, hk, d), s, device, spread=False) for s in (1, 2)]
        caches = []
        for spoil in (False, True):
            if spoil:
                kv[bad][1, token, 0, 7] = math.nan if token != 3 else -math.inf
            caches.append(ops.kv8_cache(b, n + 9, hk, d, block=16, device=device))
            ops.kv8_append(caches[-1], *kv, cache_seqlens=zero)
        lo = token // 16 * 16
        for left in (-1, 20):
            want, got = (ops.flash_attn_with_kvcache8(q, c, cache_seqlens=zero + n, causal=True, window_size=(left, 0))
                         for c in caches)
            sees = (at >= lo) & ((at - left <= lo + 15) if left >= 0 else (at >= 0))
            assert got[1, sees, :2].isnan().all() and not got[1, ~sees, :2].isnan().any()
            for a, c in ((got[0], want[0]), (got[1, :, 2:], want[1, :, 2:]), (got[1, ~sees, :2], want[1, ~sees, :2])):
                assert torch.equal(a, c)


@pytest.mark.parametrize("new", [1, 20, 64])
def test_bad_blocks_cpu(new):
    _bad_blocks("cpu", new)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 20, 64])
def test_bad_blocks_gpu(new):
    _bad_blocks("cuda", new)


def _bad_queries(device):
    """A NaN in a query makes that row of that head NaN and no other; a row that sees nothing stays 0."""
    from myk_llm_b200 import ops

    b, n, new, hk, d = 2, 30, 40, 1, 64
    cache = ops.kv8_cache(b, n, hk, d, device=device)
    zero = torch.zeros(b, dtype=torch.int32, device=device)
    ops.kv8_append(cache, _data((b, n, hk, d), 1, device), _data((b, n, hk, d), 2, device), cache_seqlens=zero)
    q = _data((b, new, 2, d), 3, device)
    q[1, 35, 0, 3] = math.nan
    q[0, 5, 1, 3] = math.nan  # ten tokens before the first: sees nothing
    out = ops.flash_attn_with_kvcache8(q, cache, cache_seqlens=zero + n, causal=True)
    assert out[1, 35, 0].isnan().all() and out.isnan().sum() == d and not out[:, :10].any()


def test_bad_queries_cpu():
    _bad_queries("cpu")


@pytest.mark.gpu
def test_bad_queries_gpu():
    _bad_queries("cuda")



@pytest.mark.gpu
@pytest.mark.parametrize("case", [
    # (batch, new, heads, kv_heads, d, cached keys, window, whether the prefill kernel is the faster one)
    (16, 80, 16, 4, 64, 16000, 0, False),   # a wave of the prefill kernel's CTAs is mostly idle with one query tile
    (16, 184, 16, 8, 64, 4000, 512, True),  # items of two heads, and a window that bounds the keys of each
])
def test_prefill_rule(case):
    """Which kernel a call takes, by whether it holds a bf16 copy of the cache while it runs."""
    from myk_llm_b200 import ops

    b, new, heads, hk, d, cap, window, prefill = case
    cache = ops.kv8_cache(b, cap, hk, d, device="cuda")
    q = torch.zeros(b, new, heads, d, dtype=torch.bfloat16, device="cuda")
    lens = torch.full((b,), cap // 2, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    ops.flash_attn_with_kvcache8(q, cache, cache_seqlens=lens, causal=True, window_size=(window - 1, 0))
    copy = 2 * 2 * b * cap * hk * d
    assert (torch.cuda.max_memory_allocated() - before >= copy) == prefill


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("case", [c for c in ATTEND if c[3] // c[4] * c[1] > 64])
def test_attend_split_weights(case, dtype):
    """More than 64 rows a KV head over few keys: the split kernel, whose weights have f16's 11 bits (2^-10 sum p |v|)."""
    from myk_llm_b200 import ops

    lens, new, step, heads, hk, d, block, causal, window = case
    assert causal and step
    b, cap = len(lens), max(lens) + new + 5
    cache, plain = _cache(b, cap, hk, d, dtype, block, "cuda")
    held = [_data((b, cap, hk, d), s, "cuda", spread=False) for s in (1, 2)]
    kv = [_data((b, new, hk, d), s, "cuda", spread=False) for s in (4, 5)]
    zero = torch.zeros(b, dtype=torch.int32, device="cuda")
    ops.kv8_append(cache, *held, cache_seqlens=zero)
    q = _data((b, new, heads, d), 3, "cuda") * 0.5
    out = ops.flash_attn_with_kvcache8(q, cache, *kv, cache_seqlens=zero + torch.tensor(lens, device="cuda"), causal=True,
                                       window_size=window)
    for p, x, y in zip(plain, held, kv):
        p.append(x, [0] * b)
        p.append(y, lens)
    want, mag = _attend(q, plain[0].values(), plain[1].values(), [n + new for n in lens], window[0], 0, 1 / math.sqrt(d))
    assert bool(((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * mag).all())


# ------------------------------------------------------------------------- refusals
def test_cache_refusals():
    from myk_llm_b200 import ops

    with pytest.raises(TypeError):
        ops.kv8_cache(1, 8, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ops.kv8_cache(1, 8, 1, 96)
    for block in (0, 3, 2048):
        with pytest.raises(ValueError):
            ops.kv8_cache(1, 8, 1, 64, block=block)
    cache = ops.kv8_cache(1, 8, 1, 64)
    with pytest.raises(ValueError):
        ops.kv8_read(cache, cache_seqlens=torch.ones(1), start=-1)
    with pytest.raises(ValueError):
        ops.kv8_read(cache, cache_seqlens=torch.ones(1), length=-1)


def test_attend_new_keys_and_values_together_cpu():
    """As on the GPU, new keys without values (or the reverse) are refused and nothing is written."""
    from myk_llm_b200 import ops

    cache = ops.kv8_cache(1, 8, 1, 64)
    x = torch.ones(1, 1, 1, 64)
    lens = torch.zeros(1, dtype=torch.int32)
    for k, v in ((x, None), (None, x)):
        with pytest.raises(ValueError):
            ops.flash_attn_with_kvcache8(x, cache, k, v, cache_seqlens=lens)
    assert not cache.keys.view(torch.uint8).any() and not cache.key_scales.any()


@pytest.mark.gpu
def test_kernel_refusals():
    from myk_llm_b200 import ops

    cache = ops.kv8_cache(2, 32, 2, 64, device="cuda")
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    x = torch.zeros(2, 3, 2, 64, dtype=torch.bfloat16, device="cuda")
    bad_new = [(x.float(), x), (x[:1], x[:1]), (x[..., :32], x[..., :32]), (x[:, :, :1], x[:, :, :1]), (x, x[:, :2]),
               (x.cpu(), x)]
    for k, v in bad_new:
        with pytest.raises(RuntimeError):
            ops.kv8_append(cache, k, v, cache_seqlens=lens)
    for n in (lens[:1], lens.cpu(), lens[:, None]):
        with pytest.raises(RuntimeError):
            ops.kv8_append(cache, x, x, cache_seqlens=n)
    q = torch.zeros(2, 1, 4, 64, dtype=torch.bfloat16, device="cuda")
    for bad in (q.float(), q[..., :32], q[:1], q[:, :, :3]):
        with pytest.raises(RuntimeError):
            ops.flash_attn_with_kvcache8(bad, cache, cache_seqlens=lens)
    with pytest.raises(RuntimeError):
        ops.flash_attn_with_kvcache8(q, cache, x, cache_seqlens=lens)
    with pytest.raises(RuntimeError):
        ops.flash_attn_with_kvcache8(q, cache, cache_seqlens=lens, softmax_scale=math.nan)
    broken = [ops.KVCache8(cache.keys[:, :, :16], cache.values[:, :, :16], cache.key_scales, cache.value_scales, 16),
              ops.KVCache8(cache.keys, cache.values, cache.key_scales, cache.value_scales, 8),
              ops.KVCache8(cache.keys, cache.values, cache.key_scales, cache.value_scales, 12),
              ops.KVCache8(cache.keys, cache.values.view(INT8), cache.key_scales, cache.value_scales, 16),
              ops.KVCache8(cache.keys, cache.values, cache.key_scales.cpu(), cache.value_scales, 16),
              ops.KVCache8(cache.keys.view(torch.uint8), cache.values.view(torch.uint8), cache.key_scales,
                           cache.value_scales, 16)]
    for c in broken:
        with pytest.raises(RuntimeError):
            ops.kv8_read(c, cache_seqlens=lens)
    # nothing to do is not an error
    ops.kv8_append(cache, x[:, :0], x[:, :0], cache_seqlens=lens)
    assert ops.flash_attn_with_kvcache8(q[:, :0], cache, cache_seqlens=lens).shape == (2, 0, 4, 64)
    assert not ops.flash_attn_with_kvcache8(q, cache, cache_seqlens=lens).any()
    assert ops.kv8_read(cache, cache_seqlens=lens, length=0)[0].shape == (2, 0, 2, 64)
