"""The 8-bit KV cache operators at sizes, values and calls that are easy to get wrong."""
import ctypes
import math
import threading
import time

import pytest
import torch

import kv8_ref as ref
from gpu_util import assert_clean_status
from test_kv8_gpu import (SCALE, _bits, _check_decode, _check_evict, _check_sums, _filled_cache, _garbage_cache, _gen, _ints,
                          _ops)

pytestmark = pytest.mark.gpu
D = 128
E4M3 = torch.float8_e4m3fn


# ------------------------------------------------------------------------------------------------------------------
# eviction: chunks of a row that are no multiple of four tokens
# ------------------------------------------------------------------------------------------------------------------
class _KernelNodeParams(ctypes.Structure):  # CUDA_KERNEL_NODE_PARAMS of the driver interface
    _fields_ = [("func", ctypes.c_void_p)] + [(n, ctypes.c_uint) for n in ("gx", "gy", "gz", "bx", "by", "bz", "smem")] + \
               [("params", ctypes.c_void_p), ("extra", ctypes.c_void_p), ("kern", ctypes.c_void_p), ("ctx", ctypes.c_void_p)]


def _captured_kernels(call):
    """(grid, block, dynamic shared memory) of every kernel that `call` launches; it is captured and never run."""
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    cuda = ctypes.CDLL("libcuda.so.1")
    raw = ctypes.c_void_p(graph.raw_cuda_graph())
    n = ctypes.c_size_t(0)
    assert cuda.cuGraphGetNodes(raw, None, ctypes.byref(n)) == 0
    nodes = (ctypes.c_void_p * n.value)()
    assert cuda.cuGraphGetNodes(raw, nodes, ctypes.byref(n)) == 0
    found = []
    for node in nodes:
        kind = ctypes.c_int(-1)
        assert cuda.cuGraphNodeGetType(ctypes.c_void_p(node), ctypes.byref(kind)) == 0
        if kind.value == 0:
            p = _KernelNodeParams()
            assert cuda.cuGraphKernelNodeGetParams_v2(ctypes.c_void_p(node), ctypes.byref(p)) == 0
            found.append((p.gx, p.bx, p.smem))
    return found


@pytest.mark.parametrize("B,S,H", [(1, 1, 1), (1, 30, 1), (1, 2049, 3), (1, 2050, 1), (3, 4099, 50), (1, 4999, 40), (2, 20483, 2)])
def test_evict_has_shared_memory_for_every_key_that_it_writes(B, S, H):
    """The keys of a chunk are written and read in groups of four: the last group belongs to what the launch asks for."""
    ops = _ops()
    cache = ops.kv8_cache(B, S, H)
    weights, lens = torch.zeros(B, H, S, device="cuda"), _ints([S] * B)
    out = ops.kv8_cache(B, 1, H)
    select = [k for k in _captured_kernels(lambda: ops.kv8_evict(cache, weights, lens, 1, out=out)) if k[2]]
    assert len(select) == 1
    grid, _, smem = select[0]
    chunk = -(-S // (grid // (B * H)))
    assert smem >= 4 * (-(-chunk // 4) * 4), (chunk, smem)


@pytest.mark.parametrize("dtype", ref.DTYPES)
@pytest.mark.parametrize("B,S,H,budget", [
    (1, 29, 1, 9), (2, 2049, 3, 1000), (1, 2050, 1, 77), (1, 2051, 2, 2050), (3, 4099, 50, 65), (2, 20483, 2, 3000),
    (1, 8 * 48 * 1024 + 3, 1, 513),  # chunks of one more than what shared memory holds
])
def test_evict_of_rows_of_any_length(dtype, B, S, H, budget):
    ops = _ops()
    lens = [S - 2 * b for b in range(B)]
    cache = _filled_cache(300, B, S, H, dtype, 1, 64, lens)
    weights = torch.rand(B, H, S, generator=_gen(301), device="cuda")
    weights[:, :, -5:] += 1  # the tail of the last group among the kept
    out = _garbage_cache(302, B, budget, H, dtype, 1, 64)
    before = [t.view(torch.uint8).clone() for t in (out.k, out.v)]
    result = ops.kv8_evict(cache, weights, _ints(lens), budget, sink=1, recent=2, out=out)
    _check_evict(cache, weights, lens, budget, 1, 2, result, before)
    assert_clean_status()


# ------------------------------------------------------------------------------------------------------------------
# workspaces
# ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("make", [lambda n: torch.zeros(n, dtype=torch.uint8),
                                  lambda n: torch.zeros(2 * n, dtype=torch.uint8, device="cuda")[::2],
                                  lambda n: torch.zeros(n // 1024, 1024, dtype=torch.uint8, device="cuda").t()])
def test_workspaces_that_a_kernel_could_not_write_are_refused(make):
    ops = _ops()
    ws = make(1 << 24)
    cache = ops.kv8_cache(1, 64, 1)
    q = torch.zeros(1, 2, D, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="workspace"):
        ops.kv8_decode(q, cache, _ints([64]), workspace=ws)
    with pytest.raises(ValueError, match="workspace"):
        ops.attention_weight_sums(q[:, :, None], q[:, :1, None], torch.zeros(1, 2, 1, device="cuda"), workspace=ws)


def test_decode_with_weights_goes_through_its_launches_one_thread_at_a_time(monkeypatch):
    """A call with weights is two launches that hand scores over in the stream's scratch: no other thread's call, with
    weights or without, may come between them.  The library's function is replaced by one that notes who else is inside."""
    ops = _ops()
    from cuda_llm_ops_b200 import _lib
    inside, met, entered, note = {}, [], [], threading.Lock()

    class Library:
        def __getattr__(self, name):
            return getattr(real, name)

        def cllo_kv8_decode_bf16(self, *args):
            workspace = args[10]
            with note:
                met.append(inside.get(workspace, 0))
                inside[workspace] = inside.get(workspace, 0) + 1
                entered.append(workspace)
            time.sleep(0.05)  # where the real one is between its launches
            with note:
                inside[workspace] -= 1
            return _lib.OK

    cache = ops.kv8_cache(2, 300, 2)
    q = torch.zeros(2, 8, D, dtype=torch.bfloat16, device="cuda")
    weights = [torch.zeros(2, 2, 300, device="cuda"), None, torch.zeros(2, 2, 300, device="cuda")]
    lens = _ints([300, 7])
    own = torch.zeros(1 << 23, dtype=torch.uint8, device="cuda")
    real = _lib.load()
    monkeypatch.setattr(_lib, "_lib", Library())
    for workspace in (None, own):  # the stream's scratch, and one that the threads share
        threads = [threading.Thread(target=ops.kv8_decode, args=(q, cache, lens), kwargs=dict(weights=w, workspace=workspace))
                   for w in weights]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    assert len(entered) == 6 and len(set(entered)) == 2
    assert met == [0] * 6


def test_decode_with_weights_from_two_host_threads_on_one_stream():
    """Both threads' weights are those of the same calls made one after the other, bit for bit."""
    ops = _ops()
    calls, lens = 500, [[900, 40], [33, 700, 512]]
    busy = torch.zeros(8192, 8192, dtype=torch.bfloat16, device="cuda")
    caches = [_filled_cache(400 + 10 * i, len(n), 1024, 2, E4M3, 1, 64, n) for i, n in enumerate(lens)]
    qs = [torch.randn(len(n), 8, D, generator=_gen(430 + i), device="cuda").to(torch.bfloat16) for i, n in enumerate(lens)]
    dev = [_ints(n) for n in lens]

    def work(i, weights, outs):
        for _ in range(calls):
            outs.append(ops.kv8_decode(qs[i], caches[i], dev[i], weights=weights))

    def run(together):
        weights = [torch.zeros(len(n), 2, 1024, device="cuda") for n in lens]
        outs = [[], []]
        torch.cuda.synchronize()
        for _ in range(30):  # the stream's queue runs full, so that the threads meet inside their launches
            torch.mm(busy, busy)
        start = threading.Barrier(2 if together else 1)

        def thread(i):
            start.wait()
            work(i, weights[i], outs[i])
        threads = [threading.Thread(target=thread, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
            if not together:
                t.join()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert all(len(o) == calls for o in outs)
        return weights, outs

    want, want_out = run(False)
    for _ in range(3):
        got, got_out = run(True)
        for i in range(2):
            assert torch.equal(got[i], want[i]), "thread %d: weights off by %g" % (i, (got[i] - want[i]).abs().max())
            assert all(torch.equal(o.view(torch.int16), want_out[i][0].view(torch.int16)) for o in got_out[i])
    assert_clean_status()


# ------------------------------------------------------------------------------------------------------------------
# weight sums: rows that saw nothing
# ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("causal,window,group", [(False, None, 2), (True, None, 2), (True, 64, 4), (True, 20, 3), (False, 100, 1)])
def test_weight_sums_of_rows_without_keys_whose_queries_are_not_finite(causal, window, group):
    """lse = -inf says that a row saw no key (padding, a mask that left nothing): it adds nothing, whatever its query holds."""
    ops = _ops()
    B, H, S = 2, 2, 400
    q = torch.randn(B, group * H, S, D, generator=_gen(1), device="cuda").to(torch.bfloat16)
    k = torch.randn(B, H, S, D, generator=_gen(2), device="cuda").to(torch.bfloat16)
    s = SCALE * q.float().view(B, H, -1, S, D) @ k.float()[:, :, None].transpose(-1, -2)
    if causal:
        s = s.masked_fill(torch.ones(S, S, dtype=torch.bool, device="cuda").triu(1), -math.inf)
    lse = s.logsumexp(-1).view(B, group * H, S)
    clean = q.clone()
    for row, value in ((5, math.nan), (127, math.inf), (128, -math.inf), (255, math.nan), (383, math.nan), (390, math.inf), (399, math.nan)):
        q[0, :, row], lse[0, :, row], clean[0, :, row] = value, -math.inf, 0
    q[1, 0, 390, 3], lse[1, 0, 390], clean[1, 0, 390] = math.nan, -math.inf, 0  # of one head, in one place
    q[1, -1], lse[1, -1], clean[1, -1] = math.nan, -math.inf, 0                 # a whole head
    got = ops.attention_weight_sums(q, k, lse, causal=causal, window=window)
    _check_sums(got, clean, k, lse, SCALE, causal, window=window)
    assert_clean_status()


# ------------------------------------------------------------------------------------------------------------------
# eviction and what follows it
# ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ref.DTYPES)
def test_two_caches_and_two_weight_tensors_in_turn(dtype):
    """Evictions between two caches, the second weight tensor zeroed before each: a token that is appended afterwards starts with
    no weight, whatever its place held before, and is attended to."""
    ops = _ops()
    B, H, Hq, cap, budget = 2, 2, 8, 160, 100
    lens = [160, 90]
    caches = [_filled_cache(500, B, cap, H, dtype, 1, 32, lens), _garbage_cache(501, B, cap, H, dtype, 1, 32)]
    weights = [torch.rand(B, H, cap, generator=_gen(502), device="cuda"), torch.full((B, H, cap), 3.0, device="cuda")]
    dev = _ints(lens)
    for turn in range(3):
        held, before = dev.tolist(), [t.view(torch.uint8).clone() for t in (caches[1].k, caches[1].v)]
        weights[1].zero_()
        result = ops.kv8_evict(caches[0], weights[0], dev, budget, sink=2, recent=20, out=caches[1], out_weights=weights[1])
        _check_evict(caches[0], weights[0], held, budget, 2, 20, result, before)
        caches.reverse()
        weights.reverse()
        dev = result[2].clone()
        for step in range(3):
            new = [torch.randn(B, H, 1, D, generator=_gen(510 + 9 * turn + 3 * step + i), device="cuda").to(torch.bfloat16)
                   for i in range(2)]
            ops.kv8_append(caches[0], *new, dev)
            dev = dev + 1
            q = torch.randn(B, Hq, D, generator=_gen(512 + 9 * turn + 3 * step), device="cuda").to(torch.bfloat16)
            base = weights[0].clone()
            at = dev.long() - 1
            assert (base[torch.arange(B, device="cuda"), :, at] == 0).all(), "the new token brings weight along"
            out = ops.kv8_decode(q, caches[0], dev, weights=weights[0])
            _check_decode(caches[0], q, dev, SCALE, out, added=(base, weights[0]))
    assert_clean_status()


def test_the_cache_that_eviction_makes_has_no_room_and_one_with_room_takes_the_next_token():
    ops = _ops()
    cache = _filled_cache(520, 1, 100, 2, torch.int8, 1, 32, [100])
    weights = torch.rand(1, 2, 100, generator=_gen(521), device="cuda")
    row = torch.randn(1, 2, 1, D, generator=_gen(522), device="cuda").to(torch.bfloat16)
    for out, stored in ((None, False), (ops.kv8_cache(1, 64, 2, torch.int8, 1, 32), True)):
        kept, _, lens, _ = ops.kv8_evict(cache, weights, _ints([100]), 50, out=out)
        before = _bits(kept)
        ops.kv8_append(kept, row, row, lens)
        assert all(torch.equal(a, b) for a, b in zip(before, _bits(kept))) != stored


# ------------------------------------------------------------------------------------------------------------------
# after a kernel that gave up
# ------------------------------------------------------------------------------------------------------------------
class _GaveUp:
    """The library, whose next status says that a kernel gave up half-way (none did)."""

    def __init__(self, real):
        self.real = real

    def __getattr__(self, name):
        return getattr(self.real, name)

    def cllo_device_status(self, detail):
        return -6


def test_status_after_calls_in_inference_mode(monkeypatch):
    """Scratch that a call made in inference mode is cleared like any other."""
    ops = _ops()
    from cuda_llm_ops_b200 import _lib, kv8
    cache = _filled_cache(600, 1, 300, 2, E4M3, 1, 64, [300])
    q = torch.randn(1, 8, D, generator=_gen(601), device="cuda").to(torch.bfloat16)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.inference_mode(), torch.cuda.stream(stream):
        want = ops.kv8_decode(q, cache, _ints([300]))
    torch.cuda.synchronize()
    scratch = kv8._workspaces[("decode", 0, stream.cuda_stream)]
    with monkeypatch.context() as m:
        m.setattr(_lib, "_lib", _GaveUp(_lib.load()))
        assert ops.device_status()[0] == -6
    torch.cuda.synchronize()
    assert (scratch == 0).all()
    with torch.cuda.stream(stream):
        again = ops.kv8_decode(q, cache, _ints([300]))
    torch.cuda.synchronize()
    assert torch.equal(again.view(torch.int16), want.view(torch.int16))


def test_status_clears_every_streams_scratch_before_it_returns(monkeypatch):
    """Scratch is kept per stream: a call on another stream, made right after the status, finds no counts of lost pieces."""
    ops = _ops()
    from cuda_llm_ops_b200 import _lib, kv8
    cache = _filled_cache(610, 1, 300, 2, E4M3, 1, 64, [300])
    q = torch.randn(1, 8, D, generator=_gen(611), device="cuda").to(torch.bfloat16)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        ops.kv8_decode(q, cache, _ints([300]))
    torch.cuda.synchronize()
    scratch = kv8._workspaces[("decode", 0, stream.cuda_stream)]
    scratch[:4096].fill_(1)
    elsewhere = torch.ones(4096, dtype=torch.uint8)  # of a device that was not asked about
    busy = torch.zeros(8192, 8192, dtype=torch.bfloat16, device="cuda")
    torch.mm(busy, busy)
    torch.cuda.synchronize()
    with monkeypatch.context() as m:
        m.setattr(_lib, "_lib", _GaveUp(_lib.load()))
        m.setitem(kv8._workspaces, ("decode", 99, 0), elsewhere)
        for _ in range(30):
            torch.mm(busy, busy)
        assert ops.device_status()[0] == -6
    with torch.cuda.stream(stream):
        found = scratch[:4096].clone()
    torch.cuda.synchronize()
    assert (found == 0).all()
    assert (elsewhere == 1).all()
