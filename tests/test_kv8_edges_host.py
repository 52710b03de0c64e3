"""The 8-bit KV cache operators at calls that are easy to get wrong, as far as they are answered without a GPU."""
import itertools

import pytest
import torch

# cllo_kv8_evict with B = 1, one kv head, 64 tokens cut to 32, blocks of 16: what is read, what is written, and their bytes
READ = dict(k=64 * 128, v=64 * 128, k_scale=16, v_scale=16, weights=256, seq_lens=4)
WRITTEN = dict(k_to=32 * 128, v_to=32 * 128, k_scale_to=8, v_scale_to=8, weights_to=128, new_lens=4, indices=128)


def _evict(lib, **at):
    """The status of the call with every tensor in a place of its own, except where `at` says."""
    place = {n: (i + 1) << 24 for i, n in enumerate([*READ, *WRITTEN])}
    place.update(at)
    return lib.cllo_kv8_evict(*(place[n] for n in (*READ, "k_to", "v_to", "k_scale_to", "v_scale_to", "weights_to", "new_lens",
                                                   "indices")), 1, 64, 32, 1, 128, 32, 0, 0, 1, 16, 0, None)


def test_evict_refuses_tensors_that_share_memory(built_library):
    """Lengths updated in place among them: blocks read the old lengths while another writes the new ones."""
    from cuda_llm_ops_b200 import _lib
    lib = _lib.load()
    if torch.cuda.is_available():
        pytest.skip("the calls that are not refused would launch on these addresses")
    assert _evict(lib) not in (_lib.OK, _lib.E_BAD_ARG)  # no device
    sizes = {**READ, **WRITTEN}
    place = {n: (i + 1) << 24 for i, n in enumerate(sizes)}
    pairs = list(itertools.product(WRITTEN, READ)) + list(itertools.permutations(WRITTEN, 2))
    for w, other in pairs:
        step = 16 if w in ("k_to", "v_to") else 4
        for at in (place[other], place[other] + sizes[other] - sizes[other] % 16 - (step if sizes[other] % 16 == 0 else 0),
                   place[other] - sizes[w] + step):
            if step == 16:
                at -= at % 16
            if at < place[other] + sizes[other] and place[other] < at + sizes[w]:
                assert _evict(lib, **{w: at}) == _lib.E_BAD_ARG, (w, other, at - place[other])
        if step == 4 or sizes[other] % 16 == 0:  # next to each other is fine
            assert _evict(lib, **{w: place[other] + sizes[other]}) not in (_lib.OK, _lib.E_BAD_ARG), (w, other)
    assert _evict(lib, seq_lens=1 << 20, new_lens=1 << 20) == _lib.E_BAD_ARG
    assert _evict(lib, weights_to=None) not in (_lib.OK, _lib.E_BAD_ARG)


def test_evict_refuses_misaligned_tensors(built_library):
    """Rows move 16 bytes at a time, everything else is read and written as 32-bit words."""
    from cuda_llm_ops_b200 import _lib
    lib = _lib.load()
    place = {n: (i + 1) << 24 for i, n in enumerate([*READ, *WRITTEN])}
    for name, at in place.items():
        for off in (8, 4) if name in ("k", "v", "k_to", "v_to") else (1, 2, 3):
            assert _evict(lib, **{name: at + off}) == _lib.E_BAD_ARG, (name, off)


def test_workspaces_that_a_kernel_could_not_write(built_library):
    """One of another device, or with gaps between its elements, is refused before its address is taken."""
    from cuda_llm_ops_b200 import kv8
    cpu, cuda = torch.device("cpu"), torch.device("cuda", 0)
    kv8._check_workspace(torch.zeros(4096, dtype=torch.uint8), cpu)
    kv8._check_workspace(torch.zeros(4, 1024), cpu)
    for t, device in ((torch.zeros(4096, dtype=torch.uint8), cuda), (torch.zeros(4096, dtype=torch.uint8, device="meta"), cpu),
                      (torch.zeros(4096, dtype=torch.uint8)[::2], cpu), (torch.zeros(64, 64).t(), cpu), (bytearray(4096), cpu),
                      (4096, cpu)):
        with pytest.raises(ValueError, match="workspace"):
            kv8._check_workspace(t, device)


def test_evict_refuses_budgets_beyond_what_its_counts_hold(built_library):
    """Positions are counted in 32 bits, in steps of several thousand: a budget near 2^31 would carry them past it."""
    from cuda_llm_ops_b200 import _lib
    lib = _lib.load()
    place = [(i + 1) << 40 for i in range(len(READ) + len(WRITTEN))]

    def evict(budget):
        return lib.cllo_kv8_evict(*place, 1, 64, 64, 1, 128, budget, 0, 0, 1, 16, 0, None)
    for budget in ((1 << 30) + 1, (1 << 31) - 8192, (1 << 31) - 1):
        assert evict(budget) == _lib.E_UNSUPPORTED, budget
    if not torch.cuda.is_available():
        assert evict(1 << 30) not in (_lib.OK, _lib.E_UNSUPPORTED, _lib.E_BAD_ARG)  # no device


@pytest.mark.parametrize("default", [torch.bfloat16, torch.float64])
def test_caches_under_another_default_dtype(default):
    """Serving programs set torch's default dtype to their model's; the scales are fp32 all the same."""
    import cuda_llm_ops_b200 as ops
    before = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        cache = ops.kv8_cache(2, 100, 3, device="cpu")
    finally:
        torch.set_default_dtype(before)
    assert cache.k_scale.dtype is torch.float32 and cache.v_scale.dtype is torch.float32
