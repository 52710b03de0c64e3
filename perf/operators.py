"""What is measured of the 8-bit KV cache operators: cases, inputs, plain forms in torch, and 64-bit results.

Four operators that follow one another in serving: ``kv8_append`` writes K/V rows into an 8-bit cache with one
power-of-two scale per (sequence, kv head, block of tokens); ``kv8_decode`` attends over it for one query token per
sequence; ``attention_weight_sums`` adds up how much weight a prompt's queries gave to every key; ``kv8_evict`` keeps the
tokens of the largest accumulated weight and moves them to another cache.  head_dim is 128 throughout.
"""
import math
import random

import numpy as np
import torch

own = False  # set by whoever imports this: run() calls the framework's kernels instead of the plain forms

D = 128
QMAX = {"e4m3": 448.0, "int8": 127.0}
MANTISSA_LIMIT = {"e4m3": (0.875, 9), "int8": (0.9921875, 7)}  # qmax = 2 * first * 2^(second - 1)
STORED = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


# ------------------------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token for every sequence of a batch of 60 at different lengths: the append of a serving step
        dict(name="append_step", op="append", batch=60, tokens=1, kv_heads=8, capacity=4096, block=64, format="e4m3",
             layout="bshd", ragged=True),
        # four prompts of 16384 tokens written at once
        dict(name="append_prompt", op="append", batch=4, tokens=16384, kv_heads=8, capacity=16384, block=64,
             format="e4m3", layout="bhsd", ragged=False),
        # chunks of up to 1000 tokens behind lengths that end inside a block
        dict(name="append_chunk_int8", op="append", batch=7, tokens=1000, kv_heads=4, capacity=4160, block=32,
             format="int8", layout="bshd", ragged=True),
        # one short conversation: latency
        dict(name="decode_short", op="decode", batch=1, capacity=1024, q_heads=32, kv_heads=8, block=64, format="e4m3",
             layout="bhsd", ragged=False, weights=False),
        # the README's decode shape
        dict(name="decode_b60", op="decode", batch=60, capacity=4096, q_heads=128, kv_heads=8, block=64, format="e4m3",
             layout="bshd", ragged=False, weights=False),
        # one sequence of a million tokens
        dict(name="decode_long_int8", op="decode", batch=1, capacity=1 << 20, q_heads=64, kv_heads=8, block=128,
             format="int8", layout="bshd", ragged=False, weights=False),
        # a mixed batch, one slot of it empty, that keeps the statistic for eviction
        dict(name="decode_ragged_weights", op="decode", batch=17, capacity=16384, q_heads=40, kv_heads=8, block=16,
             format="e4m3", layout="bhsd", ragged=True, weights=True),
        # the last 64 queries of four prompts: what a prompt's eviction looks at
        dict(name="sums_window", op="sums", batch=4, seq=8192, q_heads=32, kv_heads=8, window=64, ragged=True),
        # every query of one prompt
        dict(name="sums_all", op="sums", batch=1, seq=8192, q_heads=32, kv_heads=4, window=0, ragged=False),
        # four prompts of 32768 tokens cut down to 4096
        dict(name="evict_prompt", op="evict", batch=4, capacity=32768, budget=4096, sink=4, recent=256, kv_heads=8,
             block=64, format="e4m3", layout="bhsd", ragged=False),
        # a running batch, some of it within its budget, that sheds what a few hundred steps added
        dict(name="evict_running_int8", op="evict", batch=33, capacity=2304, budget=2001, sink=4, recent=128, kv_heads=8,
             block=32, format="int8", layout="bshd", ragged=True),
        # one sequence, two kv heads: latency
        dict(name="evict_short", op="evict", batch=1, capacity=1536, budget=512, sink=1, recent=33, kv_heads=2, block=64,
             format="e4m3", layout="bhsd", ragged=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "decode", "sums", "evict"])
    case = dict(op=op, kv_heads=rng.choice([1, 2, 4, 5, 8]), ragged=rng.random() < 0.5)
    if op != "sums":
        case.update(block=rng.choice([16, 32, 64, 128]), format=rng.choice(["e4m3", "int8"]),
                    layout=rng.choice(["bshd", "bhsd"]))
    if op == "append":
        case["tokens"] = 1 if rng.random() < 0.3 else _log_int(rng, 2, 16384)
        case["batch"] = min(_log_int(rng, 1, 256), max(1, 65536 // case["tokens"]))
        case["capacity"] = case["block"] * (-(-case["tokens"] // case["block"]) + _log_int(rng, 1, 32))
    elif op == "decode":
        case["capacity"] = case["block"] * max(1, _log_int(rng, 1, 262144) // case["block"])
        case["batch"] = min(_log_int(rng, 1, 128), max(1, 524288 // case["capacity"]))
        case["q_heads"] = case["kv_heads"] * rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16, 20])
        case["weights"] = rng.random() < 0.5
    elif op == "sums":
        case["seq"] = _log_int(rng, 1, 8192)
        case["batch"] = min(_log_int(rng, 1, 16), max(1, 8192 // case["seq"]))
        case["q_heads"] = case["kv_heads"] * rng.choice([1, 2, 3, 4])
        case["window"] = rng.choice([0, 0, 1, 17, 64, 300])
    else:
        case["capacity"] = case["block"] * max(1, _log_int(rng, 64, 131072) // case["block"])
        case["batch"] = min(_log_int(rng, 1, 64), max(1, 131072 // case["capacity"]))
        case["budget"] = max(1, int(case["capacity"] * rng.uniform(0.05, 1.0)))
        case["sink"] = rng.choice([0, 1, 4]) if case["budget"] >= 16 else 0
        case["recent"] = int((case["budget"] - case["sink"]) * rng.choice([0.0, 0.1, 0.5, 1.0]))
    return case


def _ragged(case, lo, hi):
    """Sequence lengths of a case: all ``hi``, or spread over [lo, hi] in a way that belongs to the case."""
    if not case["ragged"]:
        return [hi] * case["batch"]
    r = random.Random(case["batch"] * 1000003 + hi)
    return [r.randint(lo, hi) for _ in range(case["batch"])]


def _append_lengths(case):
    held_max = case["capacity"] - case["tokens"]
    held = _ragged(case, 0, held_max)
    r = random.Random(case["tokens"])
    new = [case["tokens"] if not case["ragged"] or case["tokens"] == 1 else r.randint(0, case["tokens"])
           for _ in range(case["batch"])]
    return held, new


def _decode_lengths(case):
    lens = _ragged(case, 1, case["capacity"])
    if case["ragged"] and case["batch"] > 2:
        lens[1] = 0  # a free slot of the batch
    return lens


# ------------------------------------------------------------------------------------------------------------------
# the 8-bit format: a block's scale is the smallest power of two 2^e, -60 <= e <= 60, with amax <= qmax * 2^e
# ------------------------------------------------------------------------------------------------------------------
def _scale_of(amax, fmt):
    limit, shift = MANTISSA_LIMIT[fmt]
    mantissa, exponent = torch.frexp(amax)
    e = exponent - shift + (mantissa > limit).to(exponent.dtype)
    e = torch.where(amax > 0, e, torch.full_like(e, -60)).clamp(-60, 60)
    return torch.ldexp(torch.ones_like(amax), e)


def _to_codes(x, fmt):
    """fp32 values in units of the scale -> stored values (round to nearest even, saturating)."""
    x = x.clamp(-QMAX[fmt], QMAX[fmt])
    return x.to(torch.float8_e4m3fn) if fmt == "e4m3" else torch.round(x).to(torch.int8)


def _blocks(x, block):
    """[..., S, D] -> [..., n_blocks, block, D]; S is a multiple of block."""
    return x.view(*x.shape[:-2], x.shape[-2] // block, block, x.shape[-1])


def _heads_first(x, layout):
    return x.transpose(1, 2) if layout == "bshd" else x


def _values(codes, scale, layout, block):
    """The fp32 values a cache stands for, [B, Hkv, S, D]."""
    x = _heads_first(codes, layout).float()
    s = scale.repeat_interleave(block, dim=2)[:, :, :x.shape[2], None]
    return x * s


# ------------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------------
def _rows(gen, *shape):
    """K or V rows: N(0,1) with a magnitude of its own per token, as activations have it."""
    x = torch.randn(*shape, generator=gen, device="cuda")
    x *= torch.exp(0.3 * torch.randn(*shape[:-1], 1, generator=gen, device="cuda"))
    return x.to(torch.bfloat16)


def _cache(gen, case):
    """A filled cache: codes in the case's layout and block scales, for K and for V."""
    B, S, H, block, fmt = case["batch"], case["capacity"], case["kv_heads"], case["block"], case["format"]
    made = {}
    for name in ("k", "v"):
        x = _blocks(_rows(gen, B, H, S, D).float(), block)
        scale = _scale_of(x.abs().amax(dim=(-1, -2)), fmt)
        codes = _to_codes(x / scale[..., None, None], fmt).view(B, H, S, D)
        made[name] = codes.transpose(1, 2).contiguous() if case["layout"] == "bshd" else codes
        made[name + "_scale"] = scale
    return made


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, H = case["batch"], case["kv_heads"]

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    state = dict(case=case)
    if case["op"] == "append":
        held, new = _append_lengths(case)
        state.update(_cache(gen, case))
        shape = (B, case["tokens"], H, D) if case["layout"] == "bshd" else (B, H, case["tokens"], D)
        state.update(k_new=_rows(gen, *shape), v_new=_rows(gen, *shape), lens=ints(held), new=ints(new))
    elif case["op"] == "decode":
        state.update(_cache(gen, case))
        state["q"] = torch.randn(B, case["q_heads"], D, generator=gen, device="cuda").to(torch.bfloat16)
        state["lens"] = ints(_decode_lengths(case))
        state["lse"] = torch.empty(B, case["q_heads"], device="cuda")
        if case["weights"]:  # what earlier steps have added up
            state["weights"] = torch.rand(B, H, case["capacity"], generator=gen, device="cuda")
    elif case["op"] == "sums":
        S, Hq = case["seq"], case["q_heads"]
        lens = _ragged(case, (S + 1) // 2, S)
        q = torch.randn(B, Hq, S, D, generator=gen, device="cuda").to(torch.bfloat16)
        k = torch.randn(B, H, S, D, generator=gen, device="cuda").to(torch.bfloat16)
        lse = torch.empty(B, Hq, S, device="cuda")  # of the causal forward over the padded batch
        causal = torch.ones(S, S, dtype=torch.bool, device="cuda").tril()
        for b in range(B):
            for h in range(Hq):
                s = (q[b, h].float() @ k[b, h // (Hq // H)].float().T) / math.sqrt(D)
                lse[b, h] = s.masked_fill_(~causal, -math.inf).logsumexp(-1)
        state.update(q=q, k=k, lse=lse, lens=ints(lens), out=torch.empty(B, H, S, device="cuda"))
    else:
        state.update(_cache(gen, case))
        lens = _ragged(case, max(1, case["capacity"] // 2), case["capacity"])
        # accumulated weight: a few heavy tokens, many light ones, and ties
        w = torch.rand(B, H, case["capacity"], generator=gen, device="cuda").pow(8)
        state.update(lens=ints(lens), weights=torch.round(w * 4096) / 1024)
        into = -(-case["budget"] // case["block"]) * case["block"]
        shape = (B, into, H, D) if case["layout"] == "bshd" else (B, H, into, D)
        for name in ("k", "v"):
            state[name + "_to"] = torch.zeros(shape, device="cuda").to(STORED[case["format"]])
            state[name + "_scale_to"] = torch.zeros(B, H, into // case["block"], device="cuda")
        state["weights_to"] = torch.zeros(B, H, into, device="cuda")
    return state


# ------------------------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "decode": _own_decode, "sums": _own_sums, "evict": _own_evict}[op](state)
    return {"append": _plain_append, "decode": _plain_decode, "sums": _plain_sums, "evict": _plain_evict}[op](state)


def _own_cache(state, suffix=""):
    import cuda_llm_ops_b200 as ops
    layout = ops.KV_BSHD if state["case"]["layout"] == "bshd" else ops.KV_BHSD
    return ops.KV8Cache(state["k" + suffix], state["v" + suffix], state["k_scale" + suffix], state["v_scale" + suffix],
                        kv_layout=layout, block_tokens=state["case"]["block"])


def _own_append(state):
    import cuda_llm_ops_b200 as ops
    ops.kv8_append(_own_cache(state), state["k_new"], state["v_new"], state["lens"], new_lens=state["new"])
    return {n: state[n] for n in ("k", "v", "k_scale", "v_scale")}


def _own_decode(state):
    import cuda_llm_ops_b200 as ops
    out = ops.kv8_decode(state["q"], _own_cache(state), state["lens"], lse=state["lse"], weights=state.get("weights"))
    return {"out": out, "lse": state["lse"], "weights": state.get("weights")}


def _own_sums(state):
    import cuda_llm_ops_b200 as ops
    window = state["case"]["window"] or None
    return ops.attention_weight_sums(state["q"], state["k"], state["lse"], causal=True, seq_lens=state["lens"],
                                     window=window, out=state["out"])


def _own_evict(state):
    import cuda_llm_ops_b200 as ops
    case = state["case"]
    _, weights, lens, indices = ops.kv8_evict(_own_cache(state), state["weights"], state["lens"], case["budget"],
                                              sink=case["sink"], recent=case["recent"], out=_own_cache(state, "_to"),
                                              out_weights=state["weights_to"])
    return {"k": state["k_to"], "v": state["v_to"], "k_scale": state["k_scale_to"], "v_scale": state["v_scale_to"],
            "weights": weights, "lens": lens, "indices": indices}


def _plain_append(state):
    case = state["case"]
    block, fmt, layout, T = case["block"], case["format"], case["layout"], case["tokens"]
    B, H = case["batch"], case["kv_heads"]
    lens, new = state["lens"].long(), state["new"].long()
    # the blocks that T tokens can touch, as a window of whole blocks inside the cache
    n_all = case["capacity"] // block
    n_win = min(n_all, -(-T // block) + 1)
    first = torch.minimum(lens // block, torch.full_like(lens, n_all - n_win))
    blk = first[:, None] + torch.arange(n_win, device="cuda")                          # [B, n_win]
    pos = first[:, None] * block + torch.arange(n_win * block, device="cuda")          # [B, n_win * block]
    is_new = (pos >= lens[:, None]) & (pos < (lens + new)[:, None])
    is_old = pos < lens[:, None]
    src = (pos - lens[:, None]).clamp(0, T - 1)
    b_at, h_at = torch.arange(B, device="cuda")[:, None, None], torch.arange(H, device="cuda")[None, :, None]
    for name in ("k", "v"):
        codes, scale = _heads_first(state[name], layout), state[name + "_scale"]
        fresh = _heads_first(state[name + "_new"], layout)[b_at, h_at, src[:, None, :]].float()   # [B,H,n_win*block,D]
        fresh = torch.where(is_new[:, None, :, None], fresh, torch.zeros_like(fresh))
        held = codes.view(torch.uint8)[b_at, h_at, pos[:, None, :]]                        # stored bytes
        old_scale = scale[b_at, h_at, blk[:, None, :]]                                  # [B,H,n_win]
        has_new = is_new.view(B, 1, n_win, block).any(-1)
        has_old = is_old.view(B, 1, n_win, block).any(-1)
        need = _scale_of(_blocks(fresh, block).abs().amax(dim=(-1, -2)), fmt)
        to = torch.where(has_old, torch.maximum(old_scale, need), need)
        to = torch.where(has_new, to, old_scale)
        row_scale, row_old = (t.repeat_interleave(block, dim=2)[..., None] for t in (to, old_scale))
        moved = _to_codes(held.view(STORED[fmt]).float() * (row_old / row_scale), fmt).view(torch.uint8)
        put = _to_codes(fresh / row_scale, fmt).view(torch.uint8)
        held = torch.where((is_old & has_new[:, 0].repeat_interleave(block, dim=1))[:, None, :, None], moved, held)
        held = torch.where(is_new[:, None, :, None], put, held)
        codes.view(torch.uint8)[b_at, h_at, pos[:, None, :]] = held
        scale[b_at, h_at, blk[:, None, :]] = to
    return {n: state[n] for n in ("k", "v", "k_scale", "v_scale")}


def _plain_decode(state):
    case = state["case"]
    B, H, Hq, S = case["batch"], case["kv_heads"], case["q_heads"], case["capacity"]
    k = _values(state["k"], state["k_scale"], case["layout"], case["block"])
    s = (state["q"].float() / math.sqrt(D)).view(B, H, Hq // H, D) @ k.transpose(-1, -2)     # [B,H,G,S]
    del k
    seen = torch.arange(S, device="cuda") < state["lens"][:, None]
    s = s.masked_fill_(~seen[:, None, None, :], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    norm = p.sum(-1, keepdim=True)
    lse = torch.where(norm > 0, m + torch.log(norm), torch.full_like(m, -math.inf))
    p = p / torch.where(norm > 0, norm, torch.ones_like(norm))
    if case["weights"]:
        state["weights"] += p.sum(2)
    v = _values(state["v"], state["v_scale"], case["layout"], case["block"])
    v = torch.where(seen[:, None, :, None], v, torch.zeros_like(v))
    out = (p @ v).view(B, Hq, D).to(torch.bfloat16)
    return {"out": out, "lse": lse.view(B, Hq), "weights": state.get("weights")}


def _plain_sums(state):
    case = state["case"]
    B, H, Hq, S = case["batch"], case["kv_heads"], case["q_heads"], case["seq"]
    rows = min(case["window"], S) if case["window"] else S
    lens = state["lens"].long()
    # the last `rows` queries of each sequence; those before its start count for nothing
    at = lens[:, None] - rows + torch.arange(rows, device="cuda")                              # [B, rows]
    idx = at.clamp(min=0)
    b_at, h_at = torch.arange(B, device="cuda")[:, None, None], torch.arange(Hq, device="cuda")[None, :, None]
    q = state["q"][b_at, h_at, idx[:, None, :]].float() / math.sqrt(D)                        # [B,Hq,rows,D]
    lse = state["lse"][b_at, h_at, idx[:, None, :]].view(B, H, Hq // H, rows, 1)
    s = q.view(B, H, (Hq // H) * rows, D) @ state["k"].float().transpose(-1, -2)
    s = s.view(B, H, Hq // H, rows, S)
    p = torch.exp_(s.sub_(lse))
    t = torch.arange(S, device="cuda")
    seen = (t <= at[..., None]) & (t < lens[:, None, None]) & (at >= 0)[..., None]             # [B,rows,S]
    p.masked_fill_(~seen[:, None, None], 0.0)
    return p.sum((2, 3))


def _plain_evict(state):
    case = state["case"]
    block, fmt, layout, budget = case["block"], case["format"], case["layout"], case["budget"]
    B, H, S = case["batch"], case["kv_heads"], case["capacity"]
    lens = state["lens"].long()
    t = torch.arange(S, device="cuda")
    forced = (t < case["sink"]) | (t >= (lens - case["recent"])[:, None])
    rank = torch.where(forced[:, None, :], torch.full_like(state["weights"], math.inf), state["weights"])
    rank = torch.where((t < lens[:, None])[:, None, :], rank, torch.full_like(rank, -math.inf))
    take = min(budget, S)
    chosen = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :take]
    kept = torch.minimum(lens, torch.full_like(lens, budget))
    chosen = torch.where(torch.arange(take, device="cuda") < kept[:, None, None], chosen, torch.full_like(chosen, S))
    chosen = torch.sort(chosen, dim=-1).values                                                # S stands for none
    real = chosen < S
    into = state["weights_to"].shape[2]
    indices = torch.full((B, H, budget), -1, dtype=torch.int32, device="cuda")
    indices[..., :take] = torch.where(real, chosen, torch.full_like(chosen, -1)).to(torch.int32)
    src = torch.zeros(B, H, into, dtype=torch.long, device="cuda")
    src[..., :take] = torch.where(real, chosen, torch.zeros_like(chosen))
    live = torch.zeros(B, H, into, dtype=torch.bool, device="cuda")
    live[..., :take] = real
    b_at, h_at = torch.arange(B, device="cuda")[:, None, None], torch.arange(H, device="cuda")[None, :, None]
    for name in ("k", "v"):
        codes = _heads_first(state[name], layout).view(torch.uint8)[b_at, h_at, src].view(STORED[fmt])
        x = codes.float() * state[name + "_scale"][b_at, h_at, src // block][..., None]
        x = _blocks(torch.where(live[..., None], x, torch.zeros_like(x)), block)
        scale = _scale_of(x.abs().amax(dim=(-1, -2)), fmt)
        put = _to_codes(x / scale[..., None, None], fmt).view(torch.uint8).view(B, H, into, D)
        to, scale_to = _heads_first(state[name + "_to"], layout).view(torch.uint8), state[name + "_scale_to"]
        to.copy_(torch.where(live[..., None], put, to))
        scale_to.copy_(torch.where(live.view(B, H, -1, block).any(-1), scale, scale_to))
    moved = state["weights"][b_at, h_at, src]
    state["weights_to"].copy_(torch.where(live, moved, state["weights_to"]))
    return {"k": state["k_to"], "v": state["v_to"], "k_scale": state["k_scale_to"], "v_scale": state["v_scale_to"],
            "weights": state["weights_to"], "lens": kept.to(torch.int32), "indices": indices}


# ------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------------------------
def work(case):
    H = case["kv_heads"]
    if case["op"] == "append":
        _, new = _append_lengths(case)
        values = sum(new) * H * D * 2
        blocks = sum(-(-n // case["block"]) for n in new) * H * 2
        return {"bytes": 3.0 * values + 4.0 * blocks + 8.0 * case["batch"], "flops": 2.0 * values}
    if case["op"] == "decode":
        total, Hq = sum(_decode_lengths(case)), case["q_heads"]
        n = total * H * 2 * (D + 4.0 / case["block"]) + case["batch"] * (Hq * (4 * D + 4) + 4)
        if case["weights"]:
            n += 8.0 * total * H
        return {"bytes": float(n), "flops": 4.0 * total * Hq * D}
    if case["op"] == "sums":
        S, Hq = case["seq"], case["q_heads"]
        lens = _ragged(case, (S + 1) // 2, S)
        rows = [min(case["window"] or S, n) for n in lens]
        pairs = sum(r * (n - r) + r * (r + 1) / 2 for r, n in zip(rows, lens)) * Hq
        n = sum(rows) * Hq * (2 * D + 4) + sum(lens) * H * 2 * D + case["batch"] * H * S * 4
        return {"bytes": float(n), "flops": pairs * (2.0 * D + 2)}
    lens = _ragged(case, max(1, case["capacity"] // 2), case["capacity"])
    kept = sum(min(n, case["budget"]) for n in lens)
    ranked = sum(n for n in lens if n > case["budget"])
    n = H * (4.0 * ranked + kept * (4 * D + 16.0 / case["block"] + 8) + 4.0 * case["batch"] * case["budget"])
    return {"bytes": n, "flops": 2.0 * kept * H * 2 * D}


# ------------------------------------------------------------------------------------------------------------------
# 64-bit results, from the definitions
# ------------------------------------------------------------------------------------------------------------------
def _exact_scale(amax, fmt):
    # an amax of exactly qmax * 2^e must give e: the margin is far above the error of log2 and far below the distance to the
    # next fp32 amax (2^-24)
    e = torch.ceil(torch.log2(amax.double() / QMAX[fmt]) - 1e-9)
    e = torch.where(amax > 0, e, torch.full_like(e, -60.0)).clamp(-60, 60)
    return torch.exp2(e)


def _exact_codes(x, fmt):
    """Doubles in units of the scale -> the nearest representable value, ties to even."""
    if fmt == "int8":
        return torch.round(x).clamp(-127, 127)
    _, e = torch.frexp(x.abs())
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def exact(case, seed):
    state = prepare(case, seed)
    return {"append": _exact_append, "decode": _exact_decode, "sums": _exact_sums, "evict": _exact_evict}[case["op"]](state)


def _exact_append(state):
    case = state["case"]
    held, new = _append_lengths(case)
    block, fmt = case["block"], case["format"]
    result = {}
    for name in ("k", "v"):
        codes = _heads_first(state[name], case["layout"]).double().contiguous()
        scales = state[name + "_scale"].double()
        rows = _heads_first(state[name + "_new"], case["layout"])
        for b in range(case["batch"]):
            if new[b] == 0:
                continue
            lo, hi = held[b], held[b] + new[b]
            b0, b1 = lo // block, -(-hi // block)
            vals = torch.zeros(case["kv_heads"], (b1 - b0) * block, D, dtype=torch.float64, device="cuda")
            vals[:, lo - b0 * block:hi - b0 * block] = rows[b, :, :new[b]].double()
            s = _exact_scale(vals.view(case["kv_heads"], b1 - b0, -1).abs().amax(-1), fmt)
            if lo % block:
                s[:, 0] = torch.maximum(s[:, 0], scales[b, :, b0])
                old = codes[b, :, b0 * block:lo] * (scales[b, :, b0] / s[:, 0])[:, None, None]
                codes[b, :, b0 * block:lo] = _exact_codes(old, fmt)
            put = _exact_codes(vals / s.repeat_interleave(block, dim=1)[..., None], fmt)
            codes[b, :, lo:hi] = put[:, lo - b0 * block:hi - b0 * block]
            scales[b, :, b0:b1] = s
        result[name] = codes.transpose(1, 2) if case["layout"] == "bshd" else codes
        result[name + "_scale"] = scales
    return result


def _exact_decode(state):
    case = state["case"]
    B, H, Hq, S = case["batch"], case["kv_heads"], case["q_heads"], case["capacity"]
    G = Hq // H
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device="cuda")
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64, device="cuda")
    weights = state["weights"].double() if case["weights"] else None
    for b, n in enumerate(_decode_lengths(case)):
        if n == 0:
            continue
        for h in range(H):
            part = {}
            for name in ("k", "v"):
                codes = state[name][b, :n, h] if case["layout"] == "bshd" else state[name][b, h, :n]
                s = state[name + "_scale"][b, h].double().repeat_interleave(case["block"])[:n, None]
                part[name] = codes.double() * s
            heads = slice(h * G, (h + 1) * G)
            score = state["q"][b, heads].double() @ part["k"].T / math.sqrt(D)
            lse[b, heads] = torch.logsumexp(score, -1)
            p = torch.softmax(score, -1)
            out[b, heads] = p @ part["v"]
            if weights is not None:
                weights[b, h, :n] += p.sum(0)
    return {"out": out, "lse": lse, "weights": weights}


def _exact_sums(state):
    case = state["case"]
    B, H, Hq, S = case["batch"], case["kv_heads"], case["q_heads"], case["seq"]
    out = torch.zeros(B, H, S, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_ragged(case, (S + 1) // 2, S)):
        first = max(0, n - case["window"]) if case["window"] else 0
        mask = torch.arange(n, device="cuda")[None, :] <= torch.arange(first, n, device="cuda")[:, None]
        for h in range(Hq):
            kh = h // (Hq // H)
            s = state["q"][b, h, first:n].double() @ state["k"][b, kh, :n].double().T / math.sqrt(D)
            out[b, kh, :n] += (torch.exp(s - state["lse"][b, h, first:n, None].double()) * mask).sum(0)
    return out


def _exact_evict(state):
    case = state["case"]
    block, fmt, budget, B, H = case["block"], case["format"], case["budget"], case["batch"], case["kv_heads"]
    lens = _ragged(case, max(1, case["capacity"] // 2), case["capacity"])
    w = state["weights"].cpu().numpy().astype(np.float64)
    indices = np.full((B, H, budget), -1, dtype=np.int64)
    for b in range(B):
        for h in range(H):
            n = lens[b]
            if n <= budget:
                indices[b, h, :n] = np.arange(n)
                continue
            middle = np.arange(case["sink"], n - case["recent"])
            order = middle[np.lexsort((middle, -w[b, h, middle]))][:budget - case["sink"] - case["recent"]]
            keep = np.concatenate([np.arange(case["sink"]), order, np.arange(n - case["recent"], n)])
            indices[b, h] = np.sort(keep)
    at = torch.from_numpy(indices).cuda()
    live = at >= 0
    into = state["weights_to"].shape[2]
    result = {}
    for name in ("k", "v"):
        codes = _heads_first(state[name], case["layout"]).double()
        x = torch.zeros(B, H, into, D, dtype=torch.float64, device="cuda")
        src = at.clamp(min=0)
        vals = torch.gather(codes, 2, src[..., None].expand(-1, -1, -1, D))
        vals *= torch.gather(state[name + "_scale"].double(), 2, src // block)[..., None]
        x[:, :, :budget] = vals * live[..., None]
        x = x.view(B, H, into // block, block * D)
        used = torch.zeros(B, H, into, dtype=torch.bool, device="cuda")
        used[..., :budget] = live
        s = _exact_scale(x.abs().amax(-1), fmt) * used.view(B, H, -1, block).any(-1)
        put = _exact_codes(x / torch.where(s > 0, s, torch.ones_like(s))[..., None], fmt).view(B, H, into, D)
        result[name] = put.transpose(1, 2) if case["layout"] == "bshd" else put
        result[name + "_scale"] = s
    weights = torch.zeros(B, H, into, dtype=torch.float64, device="cuda")
    weights[..., :budget] = torch.gather(state["weights"].double(), 2, at.clamp(min=0)) * live
    result["weights"] = weights
    result["lens"] = torch.tensor([min(n, budget) for n in lens])
    result["indices"] = at
    return result
