"""Checks of the 8-bit KV cache operators that need no GPU: the cache's tensors, the refusals of both interfaces."""
import ctypes

import pytest
import torch

import cuda_llm_ops_b200 as ops
import kv8_ref as ref

E4M3 = torch.float8_e4m3fn


def _tensors(B=2, S=100, H=3, dtype=E4M3, layout=ops.KV_BHSD, block=32):
    c = ops.kv8_cache(B, S, H, dtype, layout, block, device="cpu")
    return c.k, c.v, c.k_scale, c.v_scale


def test_cache_shapes():
    for layout, shape in ((ops.KV_BHSD, (2, 3, 100, 128)), (ops.KV_BSHD, (2, 100, 3, 128))):
        for dtype in ref.DTYPES:
            c = ops.kv8_cache(2, 100, 3, dtype, layout, 32, device="cpu")
            assert c.k.shape == shape and c.k.dtype == dtype and c.k_scale.shape == (2, 3, 4)
            assert (c.batch, c.capacity, c.num_kv_heads) == (2, 100, 3)


def test_cache_refusals():
    k, v, ks, vs = _tensors()
    kw = dict(kv_layout=ops.KV_BHSD, block_tokens=32)
    ops.KV8Cache(k, v, ks, vs, **kw)
    with pytest.raises(ValueError, match="float8_e4m3fn or both int8"):
        ops.KV8Cache(k.view(torch.int8), v, ks, vs, **kw)
    with pytest.raises(ValueError, match="float8_e4m3fn or both int8"):
        ops.KV8Cache(k.view(torch.uint8), v.view(torch.uint8), ks, vs, **kw)
    with pytest.raises(ValueError, match="block_tokens"):
        ops.KV8Cache(k, v, ks, vs, ops.KV_BHSD, 48)
    with pytest.raises(ValueError, match="kv_layout"):
        ops.KV8Cache(k, v, ks, vs, 7, 32)
    with pytest.raises(ValueError, match="4-D shape"):
        ops.KV8Cache(k, v[:, :, :50], ks, vs, **kw)
    with pytest.raises(ValueError, match="k_scale"):
        ops.KV8Cache(k, v, ks[:, :, :3], vs[:, :, :3], **kw)
    with pytest.raises(ValueError, match="k_scale"):
        ops.KV8Cache(k, v, ks.double(), vs, **kw)
    with pytest.raises(ValueError, match="contiguous"):
        ops.KV8Cache(*(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v)), ks, vs, **kw)
    with pytest.raises(ValueError, match="block_tokens"):
        ops.kv8_cache(1, 16, 1, block_tokens=8, device="cpu")


def test_no_cpu_path():
    cache = ops.kv8_cache(2, 64, 2, device="cpu")
    row = torch.zeros(2, 2, 1, 128, dtype=torch.bfloat16)
    lens = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.kv8_append(cache, row, row, lens)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.kv8_decode(torch.zeros(2, 4, 128, dtype=torch.bfloat16), cache, lens)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.kv8_evict(cache, torch.zeros(2, 2, 64), lens, 8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.attention_weight_sums(row, row, torch.zeros(2, 2, 1))


def test_c_interface_refusals(built_library):
    """Every bad argument is answered before a device is looked for."""
    from cuda_llm_ops_b200 import _lib
    lib = _lib.load()
    x = 1 << 20
    st = (ctypes.c_longlong * 3)(256, 128, 128)
    odd = (ctypes.c_longlong * 3)(256, 129, 128)

    def append(k=x, ks=st, cache=x, B=1, T=1, cap=64, H=1, Dh=128, layout=1, block=64, fmt=0):
        return lib.cllo_kv8_append_bf16(k, ks, x, st, x, None, cache, x, x, x, B, T, cap, H, Dh, layout, block, fmt, None)
    for bad in (dict(k=None), dict(k=x + 8), dict(ks=odd), dict(cache=x + 1), dict(B=0), dict(T=0), dict(cap=0), dict(layout=2),
                dict(block=24), dict(fmt=2)):
        assert append(**bad) == _lib.E_BAD_ARG, bad
    for bad in (dict(Dh=64), dict(cap=(1 << 30) + 1), dict(T=(1 << 30) + 1)):
        assert append(**bad) == _lib.E_UNSUPPORTED, bad

    def decode(q=x, lens=x, scale=1.0, ws=x, nbytes=1 << 30, B=1, cap=64, Hq=2, H=1, Dh=128, layout=1, block=64, fmt=0,
               workers=0):
        return lib.cllo_kv8_decode_bf16(q, x, x, x, x, lens, scale, x, None, None, ws, nbytes, B, cap, Hq, H, Dh, layout, block,
                                        fmt, workers, None)
    for bad in (dict(q=None), dict(q=x + 2), dict(lens=None), dict(scale=float("nan")), dict(scale=float("inf")), dict(B=0),
                dict(Hq=3, H=2), dict(layout=3), dict(block=8), dict(fmt=-1), dict(workers=-1)):
        assert decode(**bad) == _lib.E_BAD_ARG, bad
    for bad in (dict(Dh=64), dict(cap=(1 << 30) + 1)):
        assert decode(**bad) == _lib.E_UNSUPPORTED, bad
    assert lib.cllo_kv8_decode_workspace_bytes(1, 64, 3, 2, 128, 0, 0) == 0
    assert lib.cllo_kv8_decode_workspace_bytes(1, 64, 2, 2, 64, 0, 0) == 0

    def sums(q=x, lse=x, scale=1.0, q_start=0, window=0, flags=0, B=1, Sq=8, Skv=8, Hq=2, H=1, Dh=128):
        return lib.cllo_attn_weight_sums_bf16(q, x, lse, None, scale, 1, q_start, window, flags, x, x, 1 << 30, B, Sq, Skv, Hq, H, Dh,
                                              None)
    for bad in (dict(q=None), dict(q=x + 4), dict(lse=None), dict(scale=float("nan")), dict(q_start=-1), dict(window=-1),
                dict(flags=2), dict(Sq=0), dict(Skv=0), dict(Hq=3, H=2)):
        assert sums(**bad) == _lib.E_BAD_ARG, bad
    for bad in (dict(Dh=64), dict(Sq=(1 << 30) + 1)):
        assert sums(**bad) == _lib.E_UNSUPPORTED, bad

    far = 1 << 30

    def evict(k=x, k_to=far, w=x, w_to=None, new_lens=far, cap=64, cap_to=32, budget=32, sink=0, recent=0, Dh=128, layout=1,
              block=16, fmt=0, scale_to=far + (1 << 27)):
        return lib.cllo_kv8_evict(k, x + (1 << 20), x + (1 << 21), x + (1 << 22), w, x, k_to, far + (1 << 26), scale_to,
                                  scale_to + 4096, w_to, new_lens, far, 1, cap, cap_to, 1, Dh, budget, sink, recent,
                                  layout, block, fmt, None)
    for bad in (dict(k=None), dict(new_lens=None), dict(budget=0), dict(sink=-1), dict(sink=20, recent=13), dict(cap_to=31),
                dict(layout=4), dict(block=17), dict(fmt=5), dict(k_to=x), dict(k_to=x + 64 * 128 - 16),
                dict(w_to=x + 16), dict(scale_to=x + (1 << 21))):
        assert evict(**bad) == _lib.E_BAD_ARG, bad
    assert evict(Dh=64) == _lib.E_UNSUPPORTED


def test_reference_scales_and_codes():
    """The reference's own format, at its borders."""
    s = ref.block_scale(torch.tensor([0.0, 448.0, 448.1, 127.0, 1e-30, 1e38], dtype=torch.float64), E4M3)
    assert s.tolist() == [2.0 ** -60, 1.0, 2.0, 0.5, 2.0 ** -60, 2.0 ** 60]
    s = ref.block_scale(torch.tensor([127.0, 127.5, 63.5], dtype=torch.float64), torch.int8)
    assert s.tolist() == [1.0, 2.0, 0.5]
    x = torch.arange(-32000, 32001, dtype=torch.float64) / 64  # exact in fp32, ties among them
    mine = ref.to_code_values(x, E4M3)
    assert torch.equal(mine, x.clamp(-448, 448).to(E4M3).double())
