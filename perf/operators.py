"""The attention step of a ragged serving batch, as cases that can be timed.

A batch mixes sequences that bring one token with sequences that bring many
(prompts, chunks of prompts, speculated tokens). Three operators run its
attention step, and each case is one pass through one of them:

* ``slots``: positions, cache slots and newly taken cache blocks of every token,
  from the request lengths (``build_slot_mapping``);
* ``norm``: the RMS norm of each query and key head, the rotation by the token's
  position and the cache write (``qk_norm_rotary_embedding`` and
  ``qk_norm_rotary_embedding_and_cache``);
* ``attn``: attention of the new tokens over the paged cache, causal, with a
  window, a prefix that every token sees, capped scores and a bias by distance
  (``paged_attention_varlen``).

``own`` selects the package's kernels; without it ``run`` evaluates the same
operators with elementary torch operations in 32 bits. ``exact`` evaluates them
in 64 bits. ``listed()`` holds the fixed cases, ``draw(rng)`` gives others of
the same ranges.
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
ROPE_BASE = 10000.0
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
DEVICE = "cuda"


def listed():
    return [
        # --- slots -----------------------------------------------------------
        # One decode step's bookkeeping: the smallest call, latency only.
        dict(name="slots_decode_64", kind="slots", seqs=64, new_low=1, new_high=1, ctx_low=100, ctx_high=4096,
             block=16),
        # A large mixed step: prompts of up to a few hundred tokens that take
        # fresh blocks, beside sequences that bring no token at all.
        dict(name="slots_prefill_300", kind="slots", seqs=300, new_low=0, new_high=400, ctx_low=0, ctx_high=2000,
             block=16),
        # --- norm ------------------------------------------------------------
        # A small decode batch: latency.
        dict(name="norm_decode_8", kind="norm", tokens=8, hq=32, hkv=8, d=128, rot=128, neox=True, dtype="bf16",
             cache="same", block=16),
        # A prompt chunk of odd length into an fp8 cache, half of each head
        # rotated in the interleaved layout.
        dict(name="norm_fp8_1003", kind="norm", tokens=1003, hq=28, hkv=4, d=128, rot=64, neox=False, dtype="fp16",
             cache="fp8", block=32),
        # A full prefill step, into the cache of the model's type.
        dict(name="norm_prefill_16384", kind="norm", tokens=16384, hq=32, hkv=8, d=128, rot=128, neox=True,
             dtype="bf16", cache="same", block=16),
        # --- attn ------------------------------------------------------------
        # Four short chats, one token each: latency.
        dict(name="attn_decode_short_4", kind="attn", seqs=4, new_low=1, new_high=1, ctx_low=30, ctx_high=250, hq=32,
             hkv=8, d=128, block=16, layout="vllm", dtype="bf16", fp8=False, window=0, prefix=0, softcap=0.0,
             alibi=False),
        # The ordinary decode batch, scores biased by distance.
        dict(name="attn_decode_alibi_64", kind="attn", seqs=64, new_low=1, new_high=1, ctx_low=512, ctx_high=4095,
             hq=32, hkv=8, d=128, block=16, layout="vllm", dtype="bf16", fp8=False, window=0, prefix=0, softcap=0.0,
             alibi=True),
        # Long contexts of which each token sees a window and the first few
        # tokens; a small model's heads.
        dict(name="attn_decode_window_32", kind="attn", seqs=32, new_low=1, new_high=1, ctx_low=8000, ctx_high=40000,
             hq=14, hkv=2, d=64, block=16, layout="nhd", dtype="fp16", fp8=False, window=4096, prefix=20, softcap=0.0,
             alibi=False),
        # One 128K-token context, capped scores: work split over the cache.
        dict(name="attn_decode_128k_cap", kind="attn", seqs=1, new_low=1, new_high=1, ctx_low=131071, ctx_high=131071,
             hq=32, hkv=8, d=128, block=16, layout="hnd", dtype="bf16", fp8=False, window=0, prefix=0, softcap=50.0,
             alibi=False),
        # Verification of one to four speculated tokens over an fp8 cache.
        dict(name="attn_spec_fp8_48", kind="attn", seqs=48, new_low=1, new_high=4, ctx_low=200, ctx_high=8000, hq=28,
             hkv=4, d=128, block=16, layout="nhd", dtype="bf16", fp8=True, window=0, prefix=0, softcap=0.0,
             alibi=False),
        # Ragged prompts with wide heads, windowed and capped, some of them
        # continuing a cached prefix.
        dict(name="attn_prompts_d256_9", kind="attn", seqs=9, new_low=17, new_high=2003, ctx_low=0, ctx_high=1500,
             hq=16, hkv=2, d=256, block=32, layout="nhd", dtype="bf16", fp8=False, window=1024, prefix=0,
             softcap=30.0, alibi=False),
        # Two long prompts from scratch, the largest call: bound by the products.
        dict(name="attn_prompts_8192", kind="attn", seqs=2, new_low=8192, new_high=8192, ctx_low=0, ctx_high=0, hq=32,
             hkv=8, d=128, block=16, layout="nhd", dtype="bf16", fp8=False, window=0, prefix=0, softcap=0.0,
             alibi=False),
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5))))))


# (query heads, KV heads, head size)
HEADS = [(32, 8, 128), (28, 4, 128), (14, 2, 64), (16, 2, 256), (8, 8, 96), (12, 4, 192), (5, 5, 128), (16, 1, 64)]
MOST_SCORES = 4 * 10**9  # query heads x new tokens x keys, about the largest listed case's
MOST_CACHE = 10**9  # bytes


def draw(rng):
    kind = rng.choice(["slots", "norm", "norm", "attn", "attn", "attn", "attn"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    block = rng.choice([16, 16, 32, 64])
    if kind == "slots":
        seqs = _log(rng, 1, 1024)
        new_high = rng.choice([1, 1, _log(rng, 1, max(1, 32768 // seqs))])
        return dict(kind=kind, seqs=seqs, new_low=rng.choice([0, 1]), new_high=new_high,
                    ctx_low=0, ctx_high=_log(rng, 1, 8192), block=rng.choice([block, 1, 48]))
    if kind == "norm":
        hq, hkv, d = rng.choice(HEADS)
        cache = rng.choice(["same", "same", "fp8", "none"])
        return dict(kind=kind, tokens=_log(rng, 1, 16384), hq=hq, hkv=hkv, d=d, rot=rng.choice([d, d, d // 2]),
                    neox=rng.random() < 0.7, dtype=dtype, cache=cache, block=block)
    fp8 = rng.random() < 0.25
    hq, hkv, d = rng.choice([h for h in HEADS if not (fp8 and h[2] == 96)])
    shape = rng.choice(["decode", "decode", "spec", "prompts", "mixed"])
    row = 2 * hkv * d * (1 if fp8 else 2)  # cache bytes a token
    seqs = _log(rng, 1, 200) if shape in ("decode", "spec") else _log(rng, 1, 16)
    ctx_high = _log(rng, 1, max(1, min(100000, MOST_CACHE // (row * seqs))))
    chunk = 0
    if shape == "decode":
        low, high = rng.choice([0, 1, 1]), 1
    elif shape == "spec":
        low, high = 1, rng.randint(2, 8)
    else:
        ctx_high = rng.choice([0, min(ctx_high, 20000)])
        most = 1
        while most < 8192 and 2 * most * (2 * most + ctx_high) * hq * seqs <= MOST_SCORES:
            most *= 2
        high = _log(rng, 1, most)
        low = max(1, high // 8)
        if shape == "mixed":  # one sequence brings a chunk, the others a token
            chunk, low, high = high, 1, 1
    return dict(kind="attn", seqs=seqs, new_low=low, new_high=high, chunk=chunk,
                ctx_low=rng.choice([0, ctx_high // 8, ctx_high]), ctx_high=ctx_high, hq=hq, hkv=hkv, d=d, block=block,
                layout=rng.choice(["nhd", "hnd", "vllm"]), dtype=dtype, fp8=fp8,
                window=rng.choice([0, 0, _log(rng, 1, 8192)]), prefix=rng.choice([0, 0, _log(rng, 1, 600)]),
                softcap=rng.choice([0.0, 0.0, 30.0, 50.0]), alibi=rng.random() < 0.25)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _spread(low, high, n):
    """n whole numbers evenly over [low, high]."""
    if n == 1:
        return [high]
    return [low + (high - low) * i // (n - 1) for i in range(n)]


def _lengths(case, seed):
    """New tokens and cached tokens of every sequence. Their numbers are the
    case's; which sequence has which is the seed's."""
    g = torch.Generator().manual_seed(seed)
    n = case["seqs"]
    new = _spread(case["new_low"], case["new_high"], n)
    ctx = _spread(case["ctx_low"], case["ctx_high"], n)
    # Paired in the case's own order, so that the work is the same for every seed.
    fixed = torch.Generator().manual_seed(1234 + n)
    ctx = [ctx[i] for i in torch.randperm(n, generator=fixed).tolist()]
    if case.get("chunk"):
        new[0] = case["chunk"]
    order = torch.randperm(n, generator=g).tolist()
    return [new[i] for i in order], [ctx[i] for i in order]


def _starts(new):
    out = [0]
    for n in new:
        out.append(out[-1] + n)
    return out


def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEVICE)


def _randn(shape, seed, dtype, scale=1.0):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEVICE) * scale).to(dtype)


def _cache(case, blocks, seed):
    """K and V caches [blocks, block, hkv, d] as views of the case's layout."""
    dtype = torch.float8_e4m3fn if case["fp8"] else DTYPES[case["dtype"]]
    b, h, d = case["block"], case["hkv"], case["d"]
    if case["layout"] == "nhd":
        return tuple(_randn((blocks, b, h, d), seed + i, dtype) for i in range(2))
    if case["layout"] == "hnd":
        return tuple(_randn((blocks, h, b, d), seed + i, dtype).transpose(1, 2) for i in range(2))
    kv = _randn((blocks, h, b, 2 * d), seed, dtype).transpose(1, 2)
    return kv[..., :d], kv[..., d:]


def _cos_sin(positions, rot):
    freq = ROPE_BASE ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], dim=1).float().to(DEVICE)


def prepare(case, seed):
    kind = case["kind"]
    if kind == "slots":
        new, ctx = _lengths(case, seed)
        block = case["block"]
        held = [-(-c // block) for c in ctx]
        need = [-(-(c + n) // block) for c, n in zip(ctx, new)]
        g = torch.Generator().manual_seed(seed + 1)
        blocks = torch.randperm(sum(need) + 7, generator=g, dtype=torch.int32)
        tables = torch.zeros(case["seqs"], max(max(need), 1), dtype=torch.int32)
        at = 0
        for s, n in enumerate(held):
            tables[s, :n] = blocks[at:at + n]
            at += n
        return dict(case=case, starts=_int32(_starts(new)), lens=_int32([c + n for c, n in zip(ctx, new)]),
                    tables=tables.to(DEVICE), free=blocks[at:].to(DEVICE), tokens=sum(new))
    if kind == "norm":
        dtype = DTYPES[case["dtype"]]
        t, hq, hkv, d, block = case["tokens"], case["hq"], case["hkv"], case["d"], case["block"]
        g = torch.Generator().manual_seed(seed)
        st = dict(case=case, qkv=_randn((t, (hq + 2 * hkv) * d), seed + 1, dtype),
                  qw=(1 + _randn((d,), seed + 2, torch.float32, 0.1)).to(dtype),
                  kw=(1 + _randn((d,), seed + 3, torch.float32, 0.1)).to(dtype),
                  table=_cos_sin(8192, case["rot"]),
                  positions=torch.randint(0, 8192, (t,), generator=g).to(DEVICE),
                  q_out=torch.empty((t, hq * d), dtype=dtype, device=DEVICE))
        if case["cache"] == "none":
            st["k_out"] = torch.empty((t, hkv * d), dtype=dtype, device=DEVICE)
        else:
            blocks = -(-t // block) + 1
            store = torch.float8_e4m3fn if case["cache"] == "fp8" else dtype
            st["kc"], st["vc"] = (torch.zeros((blocks, block, hkv, d), dtype=store, device=DEVICE) for _ in range(2))
            st["slots"] = torch.randperm(blocks * block, generator=g)[:t].to(DEVICE)
            st["scales"] = (0.02, 0.015) if case["cache"] == "fp8" else (1.0, 1.0)
        return st
    new, ctx = _lengths(case, seed)
    lens = [n + c for n, c in zip(new, ctx)]
    block = case["block"]
    need = [-(-n // block) for n in lens]
    g = torch.Generator().manual_seed(seed + 1)
    blocks = torch.randperm(sum(need) + 3, generator=g, dtype=torch.int32)
    tables = torch.zeros(case["seqs"], max(max(need), 1), dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        tables[s, :n] = blocks[at:at + n]
        at += n
    kc, vc = _cache(case, len(blocks), seed + 2)
    st = dict(case=case, new=new, lens=lens, starts=_int32(_starts(new)), seq_lens=_int32(lens), tables=tables.to(DEVICE),
              kc=kc, vc=vc, scales=(0.9, 1.1) if case["fp8"] else (1.0, 1.0),
              q=_randn((sum(new), case["hq"], case["d"]), seed + 4, DTYPES[case["dtype"]]), slopes=None, prefix=None)
    st["out"] = torch.empty_like(st["q"])
    if case["alibi"]:
        st["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / case["hq"]) for h in range(case["hq"])], device=DEVICE)
    if case["prefix"]:
        st["prefix"] = _int32([min(case["prefix"] + s % 3, n) for s, n in enumerate(lens)])
    return st


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"slots": _own_slots, "norm": _own_norm, "attn": _own_attn}[kind](state)
    return {"slots": _plain_slots, "norm": _plain_norm, "attn": _plain_attn}[kind](state)


def _own_slots(st):
    import decodekernels_amd as dk

    positions, slots, taken = dk.build_slot_mapping(st["starts"], st["lens"], st["tables"], st["case"]["block"],
                                                    st["tokens"], free_blocks=st["free"])
    return {"positions": positions, "slots": slots, "tables": st["tables"], "taken": taken}


def _own_norm(st):
    import decodekernels_amd as dk

    case = st["case"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    q, k, v = st["qkv"].split([hq * d, hkv * d, hkv * d], dim=1)
    if case["cache"] == "none":
        dk.qk_norm_rotary_embedding(st["positions"], q, k, st["qw"], st["kw"], EPS, d, st["table"], case["neox"],
                                    query_out=st["q_out"], key_out=st["k_out"])
        return {"q": st["q_out"], "k": st["k_out"]}
    dk.qk_norm_rotary_embedding_and_cache(st["positions"], q, k, v, st["qw"], st["kw"], EPS, d, st["table"],
                                          case["neox"], st["kc"], st["vc"], st["slots"], k_scale=st["scales"][0],
                                          v_scale=st["scales"][1], query_out=st["q_out"])
    return {"q": st["q_out"], "k_cache": st["kc"], "v_cache": st["vc"]}


def _own_attn(st):
    import decodekernels_amd as dk

    case = st["case"]
    out = dk.paged_attention_varlen(st["q"], st["kc"], st["vc"], st["tables"], st["seq_lens"], st["starts"],
                                    max_query_len=max(st["new"]), max_seq_len=max(st["lens"]), window=case["window"],
                                    prefix_lens=st["prefix"], softcap=case["softcap"], alibi_slopes=st["slopes"],
                                    out=st["out"], k_scale=st["scales"][0], v_scale=st["scales"][1])
    return {"out": out}


def _plain_slots(st):
    block = st["case"]["block"]
    starts, lens, tables, free = st["starts"].long(), st["lens"].long(), st["tables"], st["free"]
    new = starts[1:] - starts[:-1]
    held = (lens - new + block - 1) // block
    need = (lens + block - 1) // block
    taken = need - held
    first = taken.cumsum(0) - taken  # of the free blocks
    # Blocks that the new tokens need beyond those that hold the cached ones.
    col = torch.arange(tables.shape[1], device=DEVICE)
    fresh = (col >= held[:, None]) & (col < need[:, None])
    index = (first[:, None] + col - held[:, None]).clamp(0, max(free.numel() - 1, 0))
    tables.copy_(torch.where(fresh, free[index], tables))
    token = torch.arange(st["tokens"], device=DEVICE)
    seq = torch.searchsorted(starts[1:].contiguous(), token, right=True)
    positions = (lens - new)[seq] + token - starts[seq]
    slots = tables[seq, positions // block].long() * block + positions % block
    return {"positions": positions, "slots": slots, "tables": tables, "taken": taken.sum().int().reshape(1)}


def _plain_norm_rotate(x, weight, cos, sin, neox):
    """x [tokens, heads, d] in 32 bits: normed, then the first columns rotated."""
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    half = cos.shape[-1]
    r = x[..., :2 * half]
    a, b = (r[..., :half], r[..., half:]) if neox else (r[..., 0::2], r[..., 1::2])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    r = torch.cat([ra, rb], -1) if neox else torch.stack([ra, rb], -1).flatten(-2)
    return torch.cat([r, x[..., 2 * half:]], -1)


def _plain_norm(st):
    case = st["case"]
    hq, hkv, d, t = case["hq"], case["hkv"], case["d"], case["tokens"]
    q, k, v = (x.float().view(t, -1, d) for x in st["qkv"].split([hq * d, hkv * d, hkv * d], dim=1))
    cos, sin = st["table"][st["positions"]][:, None].chunk(2, dim=-1)
    q = _plain_norm_rotate(q, st["qw"], cos, sin, case["neox"])
    k = _plain_norm_rotate(k, st["kw"], cos, sin, case["neox"])
    st["q_out"].copy_(q.flatten(1))
    if case["cache"] == "none":
        st["k_out"].copy_(k.flatten(1))
        return {"q": st["q_out"], "k": st["k_out"]}
    for cache, x, scale in ((st["kc"], k, st["scales"][0]), (st["vc"], v, st["scales"][1])):
        if case["cache"] == "fp8":
            x = (x / scale).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
            cache.view(torch.uint8).view(-1, hkv, d)[st["slots"]] = x.view(torch.uint8)
        else:
            cache.view(-1, hkv, d)[st["slots"]] = x.to(cache.dtype)
    return {"q": st["q_out"], "k_cache": st["kc"], "v_cache": st["vc"]}


def _plain_attn(st):
    case = st["case"]
    hq, hkv, d, block = case["hq"], case["hkv"], case["d"], case["block"]
    group = hq // hkv
    out = st["out"]
    at = 0
    for s, (n, length) in enumerate(zip(st["new"], st["lens"])):
        if n == 0:
            continue
        table = st["tables"][s, :-(-length // block)].long()
        k = st["kc"][table].float().flatten(0, 1)[:length] * st["scales"][0]  # [keys, hkv, d]
        v = st["vc"][table].float().flatten(0, 1)[:length] * st["scales"][1]
        key = torch.arange(length, device=DEVICE)
        query = torch.arange(length - n, length, device=DEVICE)[:, None]
        sees = key <= query
        if case["window"]:
            sees &= key > query - case["window"]
        if st["prefix"] is not None:
            sees |= key < st["prefix"][s]
        for h in range(hkv):
            q = st["q"][at:at + n, h * group:(h + 1) * group].float().transpose(0, 1).reshape(group * n, d)
            x = (q @ k[:, h].t().contiguous()).view(group, n, length) * d**-0.5
            if case["softcap"]:
                x = case["softcap"] * torch.tanh(x / case["softcap"])
            if st["slopes"] is not None:
                x = x - st["slopes"][h * group:(h + 1) * group, None, None] * (query - key).abs()
            x = x.masked_fill(~sees, -math.inf)
            top = x.amax(-1, keepdim=True).clamp_min(-3e38)
            p = torch.exp(x - top)
            del x
            total = p.sum(-1, keepdim=True)
            y = (p.view(group * n, length) @ v[:, h].contiguous()).view(group, n, d) / total.clamp_min(1e-30)
            out[at:at + n, h * group:(h + 1) * group] = y.transpose(0, 1)
        at += n
    return {"out": out}


# ---------------------------------------------------------------------------
# Work and exact results
# ---------------------------------------------------------------------------
def _visible(n, length, window, prefix):
    """(pairs of a token and a key that it sees, keys that some token sees)."""
    pairs, low = 0, length
    for i in range(length - n, length):
        first = max(0, i - window + 1) if window else 0
        pairs += i + 1 - first + (min(prefix, first) + max(0, prefix - i - 1) if prefix else 0)
        low = min(low, first)
    return pairs, (length - low + min(prefix, low)) if n else 0


def work(case):
    kind = case["kind"]
    if kind == "slots":
        new, ctx = _lengths(case, 0)
        b = case["block"]
        fresh = sum(-(-(c + n) // b) - -(-c // b) for n, c in zip(new, ctx))
        held = sum(1 for n, c in zip(new, ctx) if n and c % b)  # entries of partly filled blocks
        return {"bytes": 16 * sum(new) + 4 * (2 * case["seqs"] + 2) + 8 * fresh + 4 * held,
                "flops": sum(new)}
    if kind == "norm":
        t, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["d"]
        store = {"same": 2, "fp8": 1, "none": 2}[case["cache"]]
        values = 0 if case["cache"] == "none" else hkv * d * (2 + store)
        table = 4 * case["rot"] * min(t, 8192)
        return {"bytes": t * (hq * d * 4 + hkv * d * (2 + store) + values + 8 + (0 if case["cache"] == "none" else 8))
                + table, "flops": t * (hq + hkv) * (4 * d + 3 * case["rot"])}
    new, ctx = _lengths(case, 0)
    pairs = keys = 0
    for s, (n, c) in enumerate(zip(new, ctx)):
        p, k = _visible(n, n + c, case["window"], min(case["prefix"] + s % 3, n + c) if case["prefix"] else 0)
        pairs, keys = pairs + p, keys + k
    elt = 1 if case["fp8"] else 2
    return {"bytes": 2 * keys * case["hkv"] * case["d"] * elt + 4 * sum(new) * case["hq"] * case["d"],
            "flops": 4 * pairs * case["hq"] * case["d"]}


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "slots":
        return None  # whole numbers: the plain form is exact
    if kind == "norm":
        t, hq, hkv, d, half = case["tokens"], case["hq"], case["hkv"], case["d"], case["rot"] // 2
        heads = st["qkv"].double().view(t, hq + 2 * hkv, d)
        gain = torch.cat([st["qw"].double().expand(hq, d), st["kw"].double().expand(hkv, d)])
        y = heads[:, :hq + hkv]
        y = y * gain / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / d + EPS)
        turn = torch.complex(*(st["table"].double()[st["positions"]].split(half, dim=1)))[:, None]
        first = torch.arange(half, device=DEVICE) * (1 if case["neox"] else 2)
        second = first + (half if case["neox"] else 1)
        z = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        if case["cache"] == "none":
            return {"q": y[:, :hq].flatten(1), "k": y[:, hq:].flatten(1)}
        kc = torch.zeros(st["kc"].shape, dtype=torch.float64, device=DEVICE)
        vc = torch.zeros_like(kc)
        kc.view(-1, hkv, d)[st["slots"]] = y[:, hq:] / st["scales"][0]
        vc.view(-1, hkv, d)[st["slots"]] = heads[:, hq + hkv:] / st["scales"][1]
        if case["cache"] == "fp8":
            kc, vc = kc.clamp(-448, 448), vc.clamp(-448, 448)
        return {"q": y[:, :hq].flatten(1), "k_cache": kc, "v_cache": vc}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEVICE)
    starts = _starts(st["new"])
    for s, length in enumerate(st["lens"]):
        n, c = st["new"][s], length - st["new"][s]
        rows = max(1, 2**27 // max(length, 1))  # queries at a time
        j = torch.arange(length, device=DEVICE)
        page = st["tables"][s].long()[j // case["block"]]
        for h in range(hq if n else 0):
            kv = h // (hq // hkv)
            k = st["kc"][page, j % case["block"], kv].double() * (st["scales"][0] / math.sqrt(d))
            v = st["vc"][page, j % case["block"], kv].double() * st["scales"][1]
            for i0 in range(0, n, rows):
                i = torch.arange(i0, min(n, i0 + rows), device=DEVICE)
                x = torch.mm(st["q"][starts[s] + i, h].double(), k.t().contiguous())
                away = (c + i)[:, None] - j[None]
                if case["softcap"]:
                    x = torch.tanh(x / case["softcap"]) * case["softcap"]
                if st["slopes"] is not None:
                    x = x - st["slopes"][h].double() * away.abs()
                hidden = away < 0
                if case["window"]:
                    hidden |= away >= case["window"]
                if st["prefix"] is not None:
                    hidden &= j[None] >= st["prefix"][s]
                x[hidden] = -math.inf
                out[starts[s] + i, h] = torch.softmax(x, -1) @ v
    return {"out": out}
