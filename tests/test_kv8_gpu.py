"""The 8-bit KV cache operators against 64-bit references: append, decode, weight sums, eviction, and a run of them."""
import math

import pytest
import torch

import kv8_ref as ref
from gpu_util import assert_clean_status

pytestmark = pytest.mark.gpu
D = 128
SCALE = 1.0 / math.sqrt(D)


def _ops():
    import cuda_llm_ops_b200 as ops
    return ops


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(seed, *shape):
    g = _gen(seed)
    x = torch.randn(*shape, generator=g, device="cuda")
    x *= torch.exp(torch.randn(*shape[:-1], 1, generator=g, device="cuda"))
    return x.to(torch.bfloat16)


def _shape(layout, B, S, H):
    return (B, S, H, D) if layout == 0 else (B, H, S, D)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _garbage_cache(seed, B, S, H, dtype, layout, block):
    """A cache whose bytes are arbitrary (NaN codes among them) and whose scales are NaN: what nothing has written yet."""
    cache = _ops().kv8_cache(B, S, H, dtype, layout, block)
    for t in (cache.k, cache.v):
        t.view(torch.uint8).copy_(torch.randint(0, 256, t.shape, generator=_gen(seed), device="cuda"))
    cache.k_scale.fill_(math.nan)
    cache.v_scale.fill_(math.nan)
    return cache


def _filled_cache(seed, B, S, H, dtype, layout, block, lens):
    cache = _garbage_cache(seed, B, S, H, dtype, layout, block)
    n = max(1, max(lens))
    _ops().kv8_append(cache, _rows(seed + 1, *_shape(layout, B, n, H)), _rows(seed + 2, *_shape(layout, B, n, H)),
                      _ints([0] * B), new_lens=_ints(lens))
    return cache


def _bits(cache):
    return [t.view(torch.uint8).clone() if t.element_size() == 1 else t.view(torch.int32).clone()
            for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]


# ------------------------------------------------------------------------------------------------------------------
# append
# ------------------------------------------------------------------------------------------------------------------
def _check_append(cache, before, rows, held, new):
    """Every byte of the cache after an append: new and old rows as the reference has them, the rest untouched."""
    for name, scale_name, x in (("k", "k_scale", rows[0]), ("v", "v_scale", rows[1])):
        codes, scales = getattr(cache, name), getattr(cache, scale_name)
        was = before[name].clone()
        was_values = ref.heads_first(was.view(codes.dtype), cache.kv_layout).double()
        was_scale = before[scale_name].double()
        want, want_scale = was_values.clone(), was_scale.clone()
        xs = ref.heads_first(x, cache.kv_layout)
        for b in range(cache.batch):
            ref.append(want[b], want_scale[b], xs[b], held[b], new[b], cache.block_tokens, codes.dtype)
        got = ref.heads_first(codes, cache.kv_layout).double()
        assert torch.equal(torch.nan_to_num(got, nan=1e9), torch.nan_to_num(want, nan=1e9)), name
        assert torch.equal(torch.nan_to_num(scales.double(), nan=-1.0), torch.nan_to_num(want_scale, nan=-1.0)), scale_name
        # behind the sequence: the very bytes that were there
        after = ref.heads_first(codes.view(torch.uint8), cache.kv_layout)
        for b in range(cache.batch):
            end = min(held[b] + max(0, min(new[b], xs.shape[2])), cache.capacity)
            assert torch.equal(after[b, :, end:], ref.heads_first(was, cache.kv_layout)[b, :, end:])


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("B,S,H,T,block,layout,held,new", [
    (1, 64, 1, 1, 16, 0, [0], [1]),                              # first token of a sequence
    (3, 200, 2, 1, 64, 1, [63, 64, 199], [1, 1, 1]),             # ends a block, starts one, fills the cache
    (2, 100, 3, 37, 32, 0, [5, 31], [37, 20]),                   # ragged chunk behind partly filled blocks
    (4, 130, 2, 130, 128, 1, [0, 0, 129, 130], [130, 0, 130, 1]),  # whole, nothing, one row of room, no room
    (2, 333, 5, 300, 16, 1, [7, 32], [300, 299]),
    (1, 40, 1, 9, 64, 0, [3], [9]),                              # capacity below one block
])
def test_append(dtype, B, S, H, T, block, layout, held, new):
    ops = _ops()
    cache = _filled_cache(10, B, S, H, dtype, layout, block, held)
    before = {n: getattr(cache, n).view(torch.uint8).clone() if n in "kv" else getattr(cache, n).clone()
              for n in ("k", "v", "k_scale", "v_scale")}
    rows = [_rows(20 + i, *_shape(layout, B, T, H)) for i in range(2)]
    # one sequence's rows large, so that old rows must be re-rounded; another's small, so that they must not
    ref.heads_first(rows[0], layout)[0].mul_(50)
    ref.heads_first(rows[1], layout)[-1].mul_(2.0 ** -20)
    ops.kv8_append(cache, rows[0], rows[1], _ints(held), new_lens=_ints(new))
    _check_append(cache, before, rows, held, new)
    assert_clean_status()


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("layout", [0, 1])
def test_append_of_strided_rows_and_default_lengths(dtype, layout):
    """K and V as slices of one projection output; all T rows real; lengths outside the cache are held to it."""
    ops = _ops()
    B, S, H, T = 2, 96, 2, 40
    cache = _garbage_cache(3, B, S, H, dtype, layout, 32)
    fused = _rows(4, *(_shape(layout, B, T, 3 * H)))
    k, v = (fused[:, :, H:2 * H], fused[:, :, 2 * H:]) if layout == 0 else (fused[:, H:2 * H], fused[:, 2 * H:])
    assert not k.is_contiguous()
    before = {n: getattr(cache, n).view(torch.uint8).clone() if n in "kv" else getattr(cache, n).clone()
              for n in ("k", "v", "k_scale", "v_scale")}
    ops.kv8_append(cache, k, v, _ints([0, -5]))
    _check_append(cache, before, [k, v], [0, 0], [T, T])
    now = _bits(cache)
    ops.kv8_append(cache, k, v, _ints([96, 2 ** 31 - 1]))
    assert all(torch.equal(a, b) for a, b in zip(now, _bits(cache)))


@pytest.mark.parametrize("dtype", ref.DTYPES)
def test_append_of_special_values(dtype):
    """Zero blocks, subnormals, the largest bf16 numbers, infinities and NaN; amax on either side of a scale's limit."""
    ops = _ops()
    B, H, T, block = 1, 1, 16 * 9, 16
    x = torch.zeros(B, H, T, D, device="cuda")
    x[0, 0, 16:32, :] = 1e-39
    x[0, 0, 32:48, 5] = 3.3e38
    x[0, 0, 48:64, :] = torch.randn(16, D, generator=_gen(1), device="cuda")
    x[0, 0, 50, 3], x[0, 0, 51, 4], x[0, 0, 52, 9] = math.inf, -math.inf, math.nan
    x[0, 0, 64:80, 0] = 448.0
    x[0, 0, 80:96, 0] = 450.0
    x[0, 0, 96:112, 0] = 127.0
    x[0, 0, 112:128, 0] = 127.5
    x[0, 0, 128:144, :] = torch.linspace(-7, 7, 16 * D, device="cuda").view(16, D)  # ties among them
    x = x.to(torch.bfloat16)
    cache = _garbage_cache(2, B, T, H, dtype, 1, block)
    before = {n: getattr(cache, n).view(torch.uint8).clone() if n in "kv" else getattr(cache, n).clone()
              for n in ("k", "v", "k_scale", "v_scale")}
    ops.kv8_append(cache, x, -x, _ints([0]))
    _check_append(cache, before, [x, -x], [0], [T])


# ------------------------------------------------------------------------------------------------------------------
# decode
# ------------------------------------------------------------------------------------------------------------------
def _check_decode(cache, q, lens, scale, out, lse=None, added=None):
    """Bounds, per value.  Scores: fp32 sums of 128 products, off by at most 128 * 2^-24 of the sum of magnitudes, plus
    2^-19 for rounding and the exponential.  out: half a bf16 step (2^-8 relative), the probabilities' rounding to f16
    (2^-11) and the normaliser's error, relative to sum p|v|.  The probabilities times their V scales are brought to
    [2^11, 2^15] (the largest one) before they become f16, whose steps are 2^-24 at least: half of that, 2^-36 of the
    largest, times |v8| is what any token can be off by where that is more than 2^-11 of its own."""
    want, want_lse, p, mag, size, floor = ref.decode(q, cache, lens, scale)
    ds = size * (128 * 2.0 ** -24) + 2.0 ** -19
    tol = want.abs() * 2.0 ** -8 + mag * (2.0 ** -11 + 2 * ds[..., None] + 2.0 ** -16) + 2.0 ** -36 * floor + 1e-30
    worst = ((out.double() - want).abs() / tol).max().item()
    assert worst <= 1, worst
    if lse is not None:
        empty = want_lse == -math.inf
        assert torch.equal(lse.double() == -math.inf, empty)
        err = torch.where(empty, torch.zeros_like(want_lse), (lse.double() - want_lse).abs())
        assert (err <= ds + 2.0 ** -22 * want_lse.abs().nan_to_num(posinf=0)).all(), err.max()
    if added is not None:
        B, Hq, S = p.shape
        H = cache.num_kv_heads
        group = p.view(B, H, Hq // H, S)
        bound = (group * (2 * ds.view(B, H, -1, 1) + 2.0 ** -20)).sum(2) + 1e-30
        base, got = added
        err = (got.double() - (base.double() + group.sum(2))).abs()
        assert (err <= bound + 2.0 ** -23 * got.double().abs()).all(), (err / bound).max()
        seen = torch.arange(S, device="cuda") < lens[:, None]
        same = torch.where(seen[:, None], torch.zeros_like(got), (got - base).abs())
        assert same.max() == 0, "a weight behind the sequence changed"


DECODE_CASES = [
    # B, S, Hq, H, block, layout, lens
    (1, 1, 1, 1, 16, 0, [1]),
    (2, 64, 4, 4, 16, 1, [64, 1]),
    (3, 100, 8, 2, 32, 0, [0, 100, 33]),              # an empty sequence
    (2, 257, 32, 2, 64, 1, [257, 256]),               # group 16, one token into a tile
    (1, 1000, 40, 2, 128, 0, [999]),                  # group 20: two blocks of query heads
    (5, 512, 10, 2, 64, 1, [1, 17, 0, 500, 512]),
    (2, 5000, 64, 8, 64, 0, [5000, 4321]),            # cut between blocks
    (1, 20000, 7, 1, 16, 1, [19999]),                 # one head, cut many times
    (70, 130, 8, 8, 32, 1, None),                     # many short sequences
]


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("B,S,Hq,H,block,layout,lens", DECODE_CASES)
def test_decode(dtype, B, S, Hq, H, block, layout, lens):
    ops = _ops()
    lens = lens if lens is not None else [(37 * b) % (S + 1) for b in range(B)]
    cache = _filled_cache(100, B, S, H, dtype, layout, block, lens)
    q = torch.randn(B, Hq, D, generator=_gen(7), device="cuda").to(torch.bfloat16)
    lse = torch.full((B, Hq), 5.0, device="cuda")
    out = ops.kv8_decode(q, cache, _ints(lens), lse=lse)
    _check_decode(cache, q, _ints(lens), SCALE, out, lse)
    base = torch.rand(B, H, S, generator=_gen(8), device="cuda")
    weights = base.clone()
    again = ops.kv8_decode(q, cache, _ints(lens), weights=weights)
    assert torch.equal(again.view(torch.int16), out.view(torch.int16)), "the weights change the output"
    _check_decode(cache, q, _ints(lens), SCALE, again, added=(base, weights))
    assert_clean_status()


@pytest.mark.parametrize("scale", [0.5, -0.3, 0.0, 1e-3])
def test_decode_scales(scale):
    ops = _ops()
    cache = _filled_cache(5, 2, 300, 2, torch.float8_e4m3fn, 1, 64, [300, 77])
    q = torch.randn(2, 6, D, generator=_gen(9), device="cuda").to(torch.bfloat16)
    lse = torch.empty(2, 6, device="cuda")
    out = ops.kv8_decode(q, cache, _ints([300, 77]), scale=scale, lse=lse)
    _check_decode(cache, q, _ints([300, 77]), scale, out, lse)


@pytest.mark.parametrize("dtype", ref.DTYPES)
def test_decode_of_scales_far_apart_and_queries_of_any_size(dtype):
    """Blocks whose values differ by many orders of magnitude, scales that are no powers of two, large and tiny queries."""
    ops = _ops()
    B, S, H, Hq = 3, 256, 2, 8
    cache = _garbage_cache(1, B, S, H, dtype, 1, 32)
    mag = torch.exp2(torch.tensor([0., -12., 9., -20., 3., -3., 14., 0.], device="cuda"))
    k = torch.randn(B, H, S, D, generator=_gen(2), device="cuda").to(torch.bfloat16)
    v = (torch.randn(B, H, S, D, generator=_gen(3), device="cuda") * mag.repeat_interleave(32)[:, None]).to(torch.bfloat16)
    ops.kv8_append(cache, k, v, _ints([0] * B))
    cache.k_scale.mul_(0.7)
    cache.v_scale.mul_(1.3)
    q = torch.randn(B, Hq, D, generator=_gen(4), device="cuda")
    q[1] *= 2.0 ** 30   # with the scale below: ordinary scores from queries far outside f16's range
    q[2] *= 2.0 ** -30
    q = q.to(torch.bfloat16)
    lens = _ints([S, 200, 131])
    for b, scale in enumerate((SCALE, SCALE * 2.0 ** -30, SCALE * 2.0 ** 30)):
        lse = torch.empty(B, Hq, device="cuda")
        out = ops.kv8_decode(q, cache, lens, scale=scale, lse=lse)
        one = ops.KV8Cache(*(t[b:b + 1].contiguous() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)),
                           kv_layout=1, block_tokens=32)
        _check_decode(one, q[b:b + 1], lens[b:b + 1], scale, out[b:b + 1], lse[b:b + 1])


def test_decode_puts_nan_only_where_nan_is():
    ops = _ops()
    cache = _filled_cache(5, 2, 200, 2, torch.float8_e4m3fn, 1, 64, [200, 200])
    cache.v.view(torch.uint8)[0, 1, 150, 7] = 0x7f
    q = torch.randn(2, 8, D, generator=_gen(9), device="cuda").to(torch.bfloat16)
    out = ops.kv8_decode(q, cache, _ints([200, 200]))
    nan = torch.isnan(out)
    assert nan[0, 4:, 7].all() and nan.sum() == 4
    clean = ops.kv8_decode(q, cache, _ints([150, 200]))
    assert not torch.isnan(clean).any()
    cache.k.view(torch.uint8)[1, 0, 3, 0] = 0xff
    out = ops.kv8_decode(q, cache, _ints([150, 200]))
    assert torch.isnan(out[1, :4]).all() and torch.isnan(out).sum() == 4 * D


def test_decode_is_repeatable_and_independent_of_the_number_of_workers():
    ops = _ops()
    lens = [3000, 1, 777]
    cache = _filled_cache(6, 3, 3000, 2, torch.float8_e4m3fn, 0, 64, lens)
    q = torch.randn(3, 16, D, generator=_gen(10), device="cuda").to(torch.bfloat16)
    first = ops.kv8_decode(q, cache, _ints(lens))
    for _ in range(3):
        assert torch.equal(ops.kv8_decode(q, cache, _ints(lens)).view(torch.int16), first.view(torch.int16))
    for workers in (1, 2, 3, 7, 64, 148, 300):
        _check_decode(cache, q, _ints(lens), SCALE, ops.kv8_decode(q, cache, _ints(lens), num_workers=workers))
    assert_clean_status()


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("B,S,Hq,H,workers", [
    (1, 12000, 16, 1, 0),     # one kv head over all blocks: merged in two steps
    (1, 3100, 5, 1, 25),      # one more than what is merged in one step
    (1, 3100, 5, 1, 24),
    (1, 1600, 3, 1, 13),
    (2, 40000, 20, 1, 512),   # more pieces than SMs; two blocks of query heads
    (3, 4000, 4, 2, 148),
])
def test_decode_of_units_that_many_blocks_share(dtype, B, S, Hq, H, workers):
    ops = _ops()
    lens = [S - 5 * b for b in range(B)]
    cache = _filled_cache(31, B, S, H, dtype, 1, 64, lens)
    q = torch.randn(B, Hq, D, generator=_gen(32), device="cuda").to(torch.bfloat16)
    first = None
    for _ in range(3):  # the counters are left as they were found
        lse = torch.empty(B, Hq, device="cuda")
        out = ops.kv8_decode(q, cache, _ints(lens), lse=lse, num_workers=workers)
        _check_decode(cache, q, _ints(lens), SCALE, out, lse)
        first = out if first is None else first
        assert torch.equal(out.view(torch.int16), first.view(torch.int16))
    assert_clean_status()


@pytest.mark.parametrize("dtype", ref.DTYPES)
def test_decode_of_blocks_that_nothing_was_written_to(dtype):
    """A new cache is all zeros, its scales too: tokens of value 0, whose scores are 0."""
    ops = _ops()
    cache = ops.kv8_cache(2, 300, 2, dtype, 1, 32)
    q = torch.randn(2, 8, D, generator=_gen(3), device="cuda").to(torch.bfloat16)
    lens = _ints([300, 1])
    lse = torch.empty(2, 8, device="cuda")
    weights = torch.zeros(2, 2, 300, device="cuda")
    out = ops.kv8_decode(q, cache, lens, lse=lse, weights=weights)
    assert (out == 0).all()
    _check_decode(cache, q, lens, SCALE, out, lse, added=(torch.zeros_like(weights), weights))
    ops.kv8_append(cache, _rows(4, 2, 2, 130, D), _rows(5, 2, 2, 130, D), _ints([40, 0]))
    lens = _ints([300, 210])
    base = weights.clone()
    out = ops.kv8_decode(q, cache, lens, lse=lse, weights=weights)
    _check_decode(cache, q, lens, SCALE, out, lse, added=(base, weights))
    kept, _, _, _ = ops.kv8_evict(cache, weights, lens, 200)
    out = ops.kv8_decode(q, kept, lens.clamp(max=200), lse=lse)
    _check_decode(kept, q, lens.clamp(max=200), SCALE, out, lse)


def test_decode_in_graphs_that_share_nothing():
    """Two captured calls replayed on two streams at once, lengths changed in between; an eager call beside them."""
    ops = _ops()
    caches = [_filled_cache(30 + i, 2, 4000, 4, torch.float8_e4m3fn, 1, 64, [4000, 3500]) for i in range(2)]
    qs = [torch.randn(2, 16, D, generator=_gen(40 + i), device="cuda").to(torch.bfloat16) for i in range(2)]
    lens = [_ints([4000, 100]), _ints([1500, 3500])]
    outs = [torch.empty_like(q) for q in qs]
    ops.kv8_decode(qs[0], caches[0], lens[0])
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.kv8_decode(qs[i], caches[i], lens[i], out=outs[i])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for step in range(4):
        lens[0].fill_(1000 + step)
        torch.cuda.synchronize()
        for _ in range(8):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        eager = ops.kv8_decode(qs[0], caches[0], lens[1])
        torch.cuda.synchronize()
        for i in range(2):
            _check_decode(caches[i], qs[i], lens[i], SCALE, outs[i])
        _check_decode(caches[0], qs[0], lens[1], SCALE, eager)
    assert_clean_status()


def test_decode_on_two_streams():
    ops = _ops()
    cache = _filled_cache(50, 3, 2500, 4, torch.int8, 0, 64, [2500, 2000, 10])
    lens = _ints([2500, 2000, 10])
    q = torch.randn(3, 16, D, generator=_gen(51), device="cuda").to(torch.bfloat16)
    want = ops.kv8_decode(q, cache, lens)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(ops.kv8_decode(q, cache, lens))
    torch.cuda.synchronize()
    assert all(torch.equal(o.view(torch.int16), want.view(torch.int16)) for o in outs)


# ------------------------------------------------------------------------------------------------------------------
# weight sums
# ------------------------------------------------------------------------------------------------------------------
def _check_sums(got, q, k, lse, scale, causal, base=None, **kw):
    """A term is off by its score's error (fp32 sum of 128 products, twice for the fused scale, and the exponential's
    2^-20), a sum of n terms by n * 2^-24 more."""
    want, big, terms = ref.weight_sums(q, k, lse, scale, causal, **kw)
    rel = big * 128 * 2.0 ** -24 + 2.0 ** -18 + terms * 2.0 ** -24
    full = want if base is None else want + base.double()
    err = (got.double() - full).abs()
    tol = want * rel + full.abs() * 2.0 ** -23 + 1e-30
    assert (err <= tol).all(), (err / tol).max().item()


SUMS_CASES = [
    # B, Sq, Skv, Hq, H, causal, q_start, lens, window
    (1, 1, 1, 1, 1, True, 0, None, None),
    (2, 64, 64, 4, 2, True, 0, None, None),
    (1, 300, 300, 8, 1, True, 0, None, None),
    (2, 257, 257, 6, 2, True, 0, [257, 100], 32),
    (3, 200, 200, 4, 4, True, 0, [0, 1, 199], None),     # an empty sequence, one of one token
    (1, 129, 700, 5, 1, True, 571, None, None),          # the last rows of a prompt
    (2, 40, 500, 4, 1, True, 300, [500, 320], 16),       # a chunk in the middle, a window that misses part of it
    (2, 70, 333, 8, 2, False, 0, [333, 50], None),       # no causal mask: encoder states of their own length
    (1, 150, 64, 2, 2, False, 0, None, 10),
    (1, 300, 100, 2, 1, True, 0, None, None),            # more queries than keys
    (1, 1100, 1100, 3, 1, True, 0, [1000], 900),
]


@pytest.mark.parametrize("B,Sq,Skv,Hq,H,causal,q_start,lens,window", SUMS_CASES)
def test_weight_sums(B, Sq, Skv, Hq, H, causal, q_start, lens, window):
    ops = _ops()
    q = torch.randn(B, Hq, Sq, D, generator=_gen(1), device="cuda").to(torch.bfloat16)
    k = torch.randn(B, H, Skv, D, generator=_gen(2), device="cuda").to(torch.bfloat16)
    s = SCALE * q.float().view(B, H, -1, Sq, D) @ k.float()[:, :, None].transpose(-1, -2)
    if causal:
        ahead = torch.arange(Skv, device="cuda")[None] > q_start + torch.arange(Sq, device="cuda")[:, None]
        s = s.masked_fill(ahead, -math.inf)
    lse = s.logsumexp(-1).view(B, Hq, Sq)
    lens = None if lens is None else _ints(lens)
    kw = dict(q_start=q_start, lens=lens, window=window)
    got = ops.attention_weight_sums(q, k, lse, causal=causal, q_start=q_start, seq_lens=lens, window=window)
    _check_sums(got, q, k, lse, SCALE, causal, **kw)
    again = ops.attention_weight_sums(q, k, lse, causal=causal, q_start=q_start, seq_lens=lens, window=window)
    assert torch.equal(got, again)
    base = torch.rand(B, H, Skv, generator=_gen(3), device="cuda")
    acc = base.clone()
    ops.attention_weight_sums(q, k, lse, causal=causal, q_start=q_start, seq_lens=lens, window=window, out=acc,
                              accumulate=True)
    _check_sums(acc, q, k, lse, SCALE, causal, base=base, **kw)
    assert_clean_status()


@pytest.mark.parametrize("window", [1, 31, 32, 33, 64, 65, 128, 129])
@pytest.mark.parametrize("group", [1, 2, 3, 5, 8])
def test_weight_sums_of_windows_whose_heads_share_a_tile(window, group):
    test_weight_sums(3, 700, 700, 2 * group, 2, True, 0, [700, 513, 20], window)


@pytest.mark.parametrize("Sq,Skv,q_start,lens", [(20, 600, 575, [595, 300]), (64, 64, 0, [64, 7]), (33, 900, 200, [233, 210])])
@pytest.mark.parametrize("causal", [True, False])
def test_weight_sums_of_few_queries(causal, Sq, Skv, q_start, lens):
    test_weight_sums(2, Sq, Skv, 7, 1, causal, q_start if causal else 0, lens, None)


def test_weight_sums_of_the_forward_add_up_to_its_rows():
    """With the forward's own lse the sums of a causal prompt add up to the number of (head, query) rows."""
    ops = _ops()
    B, Hq, H, S = 2, 8, 2, 500
    q = torch.randn(B, Hq, S, D, generator=_gen(1), device="cuda").to(torch.bfloat16)
    k = torch.randn(B, H, S, D, generator=_gen(2), device="cuda").to(torch.bfloat16)
    v = torch.randn(B, H, S, D, generator=_gen(3), device="cuda").to(torch.bfloat16)
    _, lse = ops.launch_flash_gqa_forward_bf16_kernel(q, k, v, causal=True)
    sums = ops.attention_weight_sums(q, k, lse)
    rows = sums.double().sum(-1) / (Hq // H * S)
    assert (rows - 1).abs().max() < 2e-3  # the forward's lse is good to 2e-3
    _check_sums(sums, q, k, lse, SCALE, True)


def test_weight_sums_skip_rows_without_keys_and_masked_infinities():
    ops = _ops()
    q = torch.randn(1, 2, 100, D, generator=_gen(1), device="cuda").to(torch.bfloat16)
    k = torch.randn(1, 1, 100, D, generator=_gen(2), device="cuda").to(torch.bfloat16)
    lse = (SCALE * q.float() @ k.float().transpose(-1, -2)).logsumexp(-1)
    lse[0, 0, 7] = -math.inf                  # a row that saw nothing
    k[0, 0, 60:] = math.nan                   # behind the sequence
    q[0, :, 60:] = math.inf
    lens = _ints([60])
    got = ops.attention_weight_sums(q, k, lse, seq_lens=lens)
    assert torch.isfinite(got).all()
    kz, qz = k.clone(), q.clone()
    kz[0, 0, 60:], qz[0, :, 60:] = 0, 0
    _check_sums(got, qz, kz, lse, SCALE, True, lens=lens)


# ------------------------------------------------------------------------------------------------------------------
# eviction
# ------------------------------------------------------------------------------------------------------------------
def _check_evict(cache, weights, lens, budget, sink, recent, result, before):
    out, out_weights, new_lens, indices = result
    B, H, block, dtype = cache.batch, cache.num_kv_heads, cache.block_tokens, cache.k.dtype
    k, v = ref.values(cache)
    w = weights.cpu().tolist()
    codes = [ref.heads_first(t, out.kv_layout) for t in (out.k, out.v)]
    for b in range(B):
        n = max(0, min(lens[b], cache.capacity))
        assert int(new_lens[b]) == min(n, budget)
        for h in range(H):
            keep = ref.kept_positions(w[b][h], n, budget, sink, recent)
            assert indices[b, h].tolist() == keep + [-1] * (budget - len(keep))
            at = torch.tensor(keep, dtype=torch.long, device="cuda")
            assert torch.equal(out_weights[b, h, :len(keep)].view(torch.int32), weights[b, h][at].view(torch.int32))
            for i, (vals, scales) in enumerate(((k, out.k_scale), (v, out.v_scale))):
                rows = vals[b, h][at]
                for j in range(0, len(keep), block):
                    part = rows[j:j + block]
                    s = ref.block_scale(ref.finite_amax(part, (0, 1)), dtype)
                    assert float(scales[b, h, j // block]) == float(s)
                    want = ref.to_code_values(part / s, dtype)
                    assert torch.equal(codes[i][b, h, j:j + part.shape[0]].double().nan_to_num(nan=1e9),
                                       want.nan_to_num(nan=1e9))
                # behind what was kept nothing was written
                old = ref.heads_first(before[i].view(dtype), out.kv_layout)
                assert torch.equal(codes[i][b, h, len(keep):].view(torch.uint8), old[b, h, len(keep):].view(torch.uint8))


EVICT_CASES = [
    # B, S, H, block, layout, lens, budget, sink, recent
    (1, 64, 1, 16, 0, [64], 1, 0, 0),
    (1, 64, 1, 16, 1, [64], 1, 1, 0),
    (2, 100, 2, 32, 0, [100, 40], 48, 4, 10),        # one within its budget
    (3, 200, 2, 64, 1, [0, 200, 65], 64, 0, 64),     # recent tokens only, an empty sequence
    (2, 1500, 3, 128, 0, [1500, 1499], 700, 3, 100),
    (1, 5000, 2, 64, 1, [4999], 4998, 1, 1),         # one token goes
    (1, 70000, 1, 64, 1, [70000], 4097, 4, 64),
    (2, 64, 2, 16, 0, [64, 64], 500, 4, 4),          # a budget beyond the capacity
]


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("B,S,H,block,layout,lens,budget,sink,recent", EVICT_CASES)
def test_evict(dtype, B, S, H, block, layout, lens, budget, sink, recent):
    ops = _ops()
    cache = _filled_cache(200, B, S, H, dtype, layout, block, lens)
    weights = torch.rand(B, H, S, generator=_gen(201), device="cuda").pow(6)
    weights[:, 0] = torch.round(weights[:, 0] * 8) / 4   # ties
    into = min(budget, S) + 5
    out = _garbage_cache(202, B, into, H, dtype, layout, block)
    before = [t.view(torch.uint8).clone() for t in (out.k, out.v)]
    out_weights = torch.full((B, H, into), 7.0, device="cuda")
    result = ops.kv8_evict(cache, weights, _ints(lens), budget, sink=sink, recent=recent, out=out,
                           out_weights=out_weights)
    assert result[0] is out and result[1] is out_weights
    _check_evict(cache, weights, lens, budget, sink, recent, result, before)
    for b in range(B):
        assert (out_weights[b, :, min(lens[b], budget):] == 7.0).all()
    assert_clean_status()


@pytest.mark.parametrize("B,S,H,budget", [
    (40, 2300, 4, 700),      # more rows than SMs, chunks beyond 2048 tokens
    (1, 2048, 3, 100),       # a chunk of 2048 tokens
    (1, 2049, 3, 2000),      # and of one more
    (3, 9000, 8, 1500),      # several blocks a row
])
def test_evict_in_blocks_of_either_size(B, S, H, budget):
    lens = [S - 3 * b for b in range(B)]
    test_evict(torch.int8, B, S, H, 32, 0, lens, budget, 4, 64)


def test_evict_of_special_weights():
    """All equal, negative, zeros of both signs, infinities, NaN."""
    ops = _ops()
    S = 300
    cache = _filled_cache(210, 5, S, 1, torch.float8_e4m3fn, 1, 32, [S] * 5)
    w = torch.zeros(5, 1, S, device="cuda")
    w[1, 0] = torch.linspace(-3, 3, S, device="cuda")
    w[2, 0, ::2] = -0.0
    w[2, 0, 100] = -1.0
    w[3, 0] = torch.rand(S, generator=_gen(1), device="cuda")
    w[3, 0, 5], w[3, 0, 6], w[3, 0, 7], w[3, 0, 8] = math.inf, -math.inf, math.nan, -math.nan
    w[4, 0] = -math.inf
    new = ops.kv8_cache(5, 128, 1, torch.float8_e4m3fn, 1, 32)
    before = [t.view(torch.uint8).clone() for t in (new.k, new.v)]
    result = ops.kv8_evict(cache, w, _ints([S] * 5), 120, sink=2, recent=7, out=new)
    _check_evict(cache, w, [S] * 5, 120, 2, 7, result, before)


def test_evict_makes_its_own_tensors_and_holds_lengths_to_the_cache():
    ops = _ops()
    cache = _filled_cache(220, 2, 100, 2, torch.int8, 0, 16, [100, 100])
    w = torch.rand(2, 2, 100, generator=_gen(1), device="cuda")
    out, out_weights, new_lens, indices = ops.kv8_evict(cache, w, _ints([1000, -4]), 50)
    assert out.capacity == 50 and new_lens.tolist() == [50, 0]
    assert (indices[1] == -1).all() and (out_weights[1] == 0).all()
    same = ops.kv8_evict(cache, w, _ints([100, 0]), 50)
    assert torch.equal(same[3], indices) and torch.equal(same[0].k.view(torch.uint8), out.k.view(torch.uint8))


# ------------------------------------------------------------------------------------------------------------------
# beyond 32 bits, captured, on other streams
# ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("layout", [0, 1])
def test_offsets_beyond_32_bits(layout):
    """A cache of 5 GB for K and 5 GB for V: the second sequence lies behind 2^31 bytes, its last heads behind 2^32."""
    ops = _ops()
    B, H, S, G, block = 2, 8, 2400000, 2, 64
    cache = ops.kv8_cache(B, S, H, torch.int8, layout, block)
    for i, t in enumerate((cache.k, cache.v)):
        t.random_(-127, 128, generator=_gen(i + 1))
    cache.k_scale.fill_(2.0 ** -6)
    cache.v_scale.fill_(2.0 ** -5)
    # the last rows come from an append
    held = [5, S - 70]
    rows = [_rows(3 + i, *_shape(layout, B, 70, H)) for i in range(2)]
    ops.kv8_append(cache, rows[0], rows[1], _ints(held))
    lens = _ints([75, S])
    q = torch.randn(B, H * G, D, generator=_gen(5), device="cuda").to(torch.bfloat16)
    weights = torch.zeros(B, H, S, device="cuda")
    lse = torch.empty(B, H * G, device="cuda")
    out = ops.kv8_decode(q, cache, lens, lse=lse, weights=weights)
    new, new_weights, new_lens, indices = ops.kv8_evict(cache, weights, lens, 300, sink=2, recent=80)
    assert new_lens.tolist() == [75, 300]
    for h in (0, 5, H - 1):
        one = [ref.heads_first(t, layout)[1:, h:h + 1].contiguous() for t in (cache.k, cache.v)]
        sub = ops.KV8Cache(one[0], one[1], *(t[1:, h:h + 1].contiguous() for t in (cache.k_scale, cache.v_scale)),
                           kv_layout=1, block_tokens=block)
        heads = slice(h * G, (h + 1) * G)
        _check_decode(sub, q[1:, heads], lens[1:], SCALE, out[1:, heads], lse[1:, heads],
                      added=(torch.zeros(1, 1, S, device="cuda"), weights[1:, h:h + 1]))
        w = weights[1, h].clone()
        w[:2], w[S - 80:] = math.inf, math.inf
        want = torch.sort(torch.sort(w, descending=True, stable=True).indices[:300]).values
        assert torch.equal(indices[1, h].long(), want)
        k, v = ref.values(sub)
        for vals, codes, scales in ((k, new.k, new.k_scale), (v, new.v, new.v_scale)):
            got = ref.heads_first(codes, layout)[1, h].double()
            s = scales[1, h].double().repeat_interleave(block)[:300, None]
            x = vals[0, 0][want]
            assert ((got * s - x).abs() <= s / 2).all()  # one rounding to the new scale
    assert_clean_status()


def test_every_call_in_one_graph_on_another_stream():
    """Append, decode with weights, weight sums and eviction captured into one graph; replayed twice with other inputs and
    compared with eager calls."""
    ops = _ops()
    B, H, Hq, cap, block = 2, 2, 8, 256, 32
    lens = _ints([100, 37])
    caches = [_filled_cache(60, B, cap, H, torch.float8_e4m3fn, 1, block, [cap, cap]) for _ in range(2)]
    kn, vn = _rows(61, B, H, 3, D), _rows(62, B, H, 3, D)
    q = torch.randn(B, Hq, D, generator=_gen(63), device="cuda").to(torch.bfloat16)
    qp = torch.randn(B, Hq, cap, D, generator=_gen(64), device="cuda").to(torch.bfloat16)
    kp = torch.randn(B, H, cap, D, generator=_gen(65), device="cuda").to(torch.bfloat16)
    lse = torch.full((B, Hq, cap), 6.0, device="cuda")
    after = torch.empty_like(lens)
    results = [dict(w=torch.zeros(B, H, cap, device="cuda")) for _ in range(2)]

    def work(cache, r):
        ops.kv8_append(cache, kn, vn, lens)
        torch.add(lens, 3, out=after)
        r["out"] = ops.kv8_decode(q, cache, after, weights=r["w"])
        ops.attention_weight_sums(qp, kp, lse, seq_lens=after, out=r["w"], accumulate=True)
        r["evicted"] = ops.kv8_evict(cache, r["w"], after, 40, sink=1, recent=8)

    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        work(caches[0], results[0])
    for step in range(2):
        kn.normal_()
        q.normal_()
        for c in results:
            c["w"].zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        work(caches[1], results[1])
        torch.cuda.synchronize()
        a, b = results
        assert torch.equal(a["out"].view(torch.int16), b["out"].view(torch.int16)) and torch.equal(a["w"], b["w"])
        assert torch.equal(a["evicted"][3], b["evicted"][3]) and torch.equal(a["evicted"][2], b["evicted"][2])
        n = int(b["evicted"][2].min())
        assert torch.equal(a["evicted"][0].k.view(torch.uint8)[:, :, :n], b["evicted"][0].k.view(torch.uint8)[:, :, :n])
        lens.copy_(_ints([200, 0]))
    assert_clean_status()


def test_weight_sums_on_two_streams_and_in_parts():
    ops = _ops()
    q = torch.randn(1, 8, 3000, D, generator=_gen(1), device="cuda").to(torch.bfloat16)
    k = torch.randn(1, 2, 3000, D, generator=_gen(2), device="cuda").to(torch.bfloat16)
    lse = torch.full((1, 8, 3000), 7.0, device="cuda")
    want = ops.attention_weight_sums(q, k, lse)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(6):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(ops.attention_weight_sums(q, k, lse))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    # a prompt in two chunks adds up to the whole one
    parts = ops.attention_weight_sums(q[:, :, :1111].contiguous(), k, lse[:, :, :1111].contiguous())
    ops.attention_weight_sums(q[:, :, 1111:].contiguous(), k, lse[:, :, 1111:].contiguous(), q_start=1111, out=parts,
                              accumulate=True)
    _check_sums(parts, q, k, lse, SCALE, True)
    assert_clean_status()


def test_own_workspaces():
    """A caller's workspace may hold anything; one too small or none of its size is refused."""
    ops = _ops()
    from cuda_llm_ops_b200 import _lib
    lib = _lib.load()
    lens = [3000, 2000]
    cache = _filled_cache(6, 2, 3000, 2, torch.int8, 0, 64, lens)
    q = torch.randn(2, 16, D, generator=_gen(10), device="cuda").to(torch.bfloat16)
    n = int(lib.cllo_kv8_decode_workspace_bytes(2, 3000, 16, 2, D, 1, 0))
    ws = torch.randint(0, 256, (n,), generator=_gen(1), device="cuda").to(torch.uint8)
    weights = torch.zeros(2, 2, 3000, device="cuda")
    out = ops.kv8_decode(q, cache, _ints(lens), weights=weights, workspace=ws)
    _check_decode(cache, q, _ints(lens), SCALE, out, added=(torch.zeros_like(weights), weights))
    with pytest.raises(RuntimeError, match="workspace"):
        ops.kv8_decode(q, cache, _ints(lens), weights=weights, workspace=ws[:n - 256])
    n = int(lib.cllo_attn_weight_sums_workspace_bytes())
    qp = torch.randn(1, 4, 700, D, generator=_gen(1), device="cuda").to(torch.bfloat16)
    lse = torch.full((1, 4, 700), 6.0, device="cuda")
    ws = torch.randint(0, 256, (n,), generator=_gen(1), device="cuda").to(torch.uint8)
    got = ops.attention_weight_sums(qp, qp[:, :2].contiguous(), lse, workspace=ws)
    _check_sums(got, qp, qp[:, :2].contiguous(), lse, SCALE, True)
    with pytest.raises(RuntimeError, match="workspace"):
        ops.attention_weight_sums(qp, qp[:, :2].contiguous(), lse, workspace=ws[:n - 256])


# ------------------------------------------------------------------------------------------------------------------
# together
# ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ref.DTYPES)
def test_prompt_decode_evict_decode(dtype):
    """A padded batch of prompts through the forward into the cache, its weight sums, steps that accumulate, an eviction,
    more steps: the cache at every step is what the references say, and the attention over it too."""
    ops = _ops()
    B, Hq, H, S, cap, block = 2, 8, 2, 300, 320, 64
    lens = [300, 211]
    q = torch.randn(B, Hq, S, D, generator=_gen(1), device="cuda").to(torch.bfloat16)
    k, v = (torch.randn(B, H, S, D, generator=_gen(2 + i), device="cuda").to(torch.bfloat16) for i in range(2))
    _, lse = ops.launch_flash_gqa_forward_bf16_kernel(q, k, v, causal=True)
    cache = ops.kv8_cache(B, cap, H, dtype, block_tokens=block)
    ops.kv8_append(cache, k, v, _ints([0, 0]), new_lens=_ints(lens))
    weights = torch.zeros(B, H, cap, device="cuda")
    sums = ops.attention_weight_sums(q, k, lse, seq_lens=_ints(lens), window=64)
    weights[:, :, :S] = sums
    dev = _ints(lens)
    for step in range(12):
        if step == 6:
            want = dev.tolist()
            before = [torch.zeros_like(t.view(torch.uint8)) for t in (cache.k[:, :, :256], cache.v[:, :, :256])]
            new = ops.kv8_cache(B, 256, H, dtype, block_tokens=block)
            result = ops.kv8_evict(cache, weights, dev, 200, sink=4, recent=32, out=new)
            _check_evict(cache, weights, want, 200, 4, 32, result, before)
            cache, weights, dev, _ = result
        kn, vn = (torch.randn(B, H, 1, D, generator=_gen(50 + 2 * step + i), device="cuda").to(torch.bfloat16)
                  for i in range(2))
        held = dev.tolist()
        before = {n: getattr(cache, n).view(torch.uint8).clone() if n in "kv" else getattr(cache, n).clone()
                  for n in ("k", "v", "k_scale", "v_scale")}
        ops.kv8_append(cache, kn, vn, dev)
        _check_append(cache, before, [kn, vn], held, [1, 1])
        dev = dev + 1
        qn = torch.randn(B, Hq, D, generator=_gen(90 + step), device="cuda").to(torch.bfloat16)
        base = weights.clone()
        out = ops.kv8_decode(qn, cache, dev, weights=weights)
        _check_decode(cache, qn, dev, SCALE, out, added=(base, weights))
    assert_clean_status()


# ------------------------------------------------------------------------------------------------------------------
# refusals
# ------------------------------------------------------------------------------------------------------------------
def test_refusals():
    ops = _ops()
    e4m3 = torch.float8_e4m3fn
    cache = ops.kv8_cache(2, 64, 2, e4m3)
    row = torch.zeros(2, 2, 1, D, dtype=torch.bfloat16, device="cuda")
    lens = _ints([0, 0])
    with pytest.raises(ValueError, match="seq_lens"):
        ops.kv8_append(cache, row, row, lens.long())
    with pytest.raises(ValueError, match="seq_lens"):
        ops.kv8_append(cache, row, row, lens.cpu())
    with pytest.raises(ValueError, match="new_lens"):
        ops.kv8_append(cache, row, row, lens, new_lens=_ints([1]))
    with pytest.raises(ValueError, match="match the cache"):
        ops.kv8_append(cache, row[:, :1], row[:, :1], lens)
    with pytest.raises(ValueError, match="16-byte"):
        wide = torch.zeros(2, 2, 1, D + 4, dtype=torch.bfloat16, device="cuda")
        ops.kv8_append(cache, wide[..., 4:], wide[..., 4:], lens)
    q = torch.zeros(2, 4, D, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="divisible"):
        ops.kv8_decode(q[:, :3].contiguous(), cache, lens)
    with pytest.raises(ValueError, match="weights"):
        ops.kv8_decode(q, cache, lens, weights=torch.zeros(2, 2, 65, device="cuda"))
    with pytest.raises(ValueError, match="lse"):
        ops.kv8_decode(q, cache, lens, lse=torch.zeros(2, 4, dtype=torch.float64, device="cuda"))
    with pytest.raises(RuntimeError, match="workspace"):
        ops.kv8_decode(q, cache, lens, workspace=torch.zeros(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(RuntimeError, match="bad argument"):
        ops.kv8_decode(q, cache, lens, scale=math.inf)
    w = torch.zeros(2, 2, 64, device="cuda")
    with pytest.raises(ValueError, match="budget"):
        ops.kv8_evict(cache, w, lens, 4, sink=3, recent=2)
    with pytest.raises(ValueError, match="room"):
        ops.kv8_evict(cache, w, lens, 40, out=ops.kv8_cache(2, 39, 2, e4m3))
    with pytest.raises(ValueError, match="match the cache"):
        ops.kv8_evict(cache, w, lens, 40, out=ops.kv8_cache(2, 40, 2, torch.int8))
    with pytest.raises(RuntimeError, match="bad argument"):
        ops.kv8_evict(cache, w, lens, 40, out=cache)
    k4 = torch.zeros(1, 2, 8, D, dtype=torch.bfloat16, device="cuda")
    lse = torch.zeros(1, 2, 8, device="cuda")
    with pytest.raises(ValueError, match="window"):
        ops.attention_weight_sums(k4, k4, lse, window=0)
    with pytest.raises(ValueError, match="accumulate"):
        ops.attention_weight_sums(k4, k4, lse, accumulate=True)
    with pytest.raises(ValueError, match="lse"):
        ops.attention_weight_sums(k4, k4, lse[:, :1])
