"""GPU tests of the attention step of a ragged batch: ``build_slot_mapping``,
``qk_norm_rotary_embedding(_and_cache)`` and ``paged_attention_varlen`` against
their 64-bit definitions (``oracle/ragged_step.py``), one by one and in a row.

Tolerances, with h = finfo(dtype).eps / 2, the most that one rounding is off,
relative to the value:

* head norms: the output's own rounding, h |y|, and the fp32 arithmetic before
  it. A rotated element is a cos - b sin of normed values, each off by a few
  2^-24 relative, so the sum is off by at most 2^-20 (|a| + |b|).
* e4m3 cache rows: h = 2^-4 of the value, half the smallest step (2^-10) below
  the normal range, and the fp32 part, which can move a value over a rounding
  border: the two together bound it.
* attention: the output's rounding h |y|; weights rounded to the dtype before
  the products with v, h sum(p |v|); and the fp32 scores. A score is a sum of
  head_dim products of magnitude at most ~ 20 in all, off by some 20 x 20 x
  2^-24 = 2.4e-5 (MFMA adds 16 or 32 products at a time), a tanh cap of 50 adds
  50 x 2^-22 = 1.2e-5; weights, numerator and sum, are off by twice that
  relative: 2^-13 sum(p |v|).
"""

import ctypes

import pytest
import torch

import decodekernels_amd as dk
from decodekernels_amd import capi
from oracle import ragged_step as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, FP16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def int32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def starts_of(new):
    out = [0]
    for n in new:
        out.append(out[-1] + n)
    return out


# ---------------------------------------------------------------------------
# Slot maps
# ---------------------------------------------------------------------------
def check_slots(new, lens, block, columns=None, free_short=0, with_free=True, pad=0, seed=0):
    g = torch.Generator().manual_seed(seed)
    starts = starts_of(new)
    held = [-(-max(n - m, 0) // block) for m, n in zip(new, lens)]
    need = [-(-max(n, 0) // block) for n in lens]
    columns = max([1, *need]) if columns is None else columns
    perm = torch.randperm(sum(need) + 5, generator=g).tolist()
    tables, at = [], 0
    for h, w in zip(held, need):
        k = min(h if with_free else w, columns)
        tables.append(perm[at:at + k] + [-9] * (columns - k))
        at += k
    free = perm[at:]
    if free_short:
        free = free[:max(0, sum(need) - sum(held) - free_short)]
    total = starts[-1] + pad
    want = oracle.slot_mapping(starts, lens, tables, block, total, free if with_free else None)
    dev_tables = torch.full((len(new), columns + 3), -77, dtype=torch.int32, device=DEV)[:, :columns]  # strided rows
    if new:
        dev_tables.copy_(int32(tables))
    positions, slots, taken = dk.build_slot_mapping(int32(starts), int32(lens), dev_tables, block, total,
                                                    free_blocks=int32(free) if with_free else None)
    assert positions.tolist() == want[0]
    assert slots.tolist() == want[1]
    assert dev_tables.tolist() == want[2]
    if dev_tables.numel():
        assert bool((dev_tables.as_strided((len(new), 3), (columns + 3, 1), columns) == -77).all())
    assert taken.tolist() == [want[3]]


@pytest.mark.parametrize("block", [1, 16, 48])
@pytest.mark.parametrize("seqs", [1, 3, 64, 257, 1023, 1024, 1025, 2500])
def test_slots_ragged(seqs, block):
    g = torch.Generator().manual_seed(seqs + block)
    new = torch.randint(0, 9, (seqs,), generator=g).tolist()
    ctx = torch.randint(0, 200, (seqs,), generator=g).tolist()
    check_slots(new, [n + c for n, c in zip(new, ctx)], block, seed=seqs)


@pytest.mark.parametrize("with_free", [True, False])
def test_slots_one_token_each_and_long_prompts(with_free):
    check_slots([1] * 300, [1 + 7 * i % 900 for i in range(300)], 16, with_free=with_free)
    check_slots([5000, 0, 1, 4097], [5000, 12, 1, 9000], 16, with_free=with_free)
    check_slots([0, 0, 0], [3, 0, 40], 16, with_free=with_free)


def test_slots_padding_and_shortages():
    check_slots([3, 1, 0, 20], [3, 90, 5, 40], 16, pad=37)  # rows behind the last sequence: -1
    check_slots([40, 1, 33, 2], [40, 17, 50, 2], 16, free_short=3)  # the free list ends early
    check_slots([40, 1, 33, 2], [40, 17, 50, 2], 16, free_short=100)  # and is empty
    check_slots([70, 20], [70, 100], 16, columns=3)  # the table ends early
    check_slots([9, 4], [5, 0], 16)  # lengths below the new tokens: no position for the first ones
    check_slots([], [], 16, columns=1, pad=5)


def test_slots_without_rows_or_tokens():
    tables = torch.zeros((2, 4), dtype=torch.int32, device=DEV)
    positions, slots, taken = dk.build_slot_mapping(int32([0, 0, 0]), int32([5, 0]), tables, 16, 0, free_blocks=int32([1]))
    assert positions.numel() == 0 and slots.numel() == 0 and taken.tolist() == [0]


# ---------------------------------------------------------------------------
# Head norms, rotation, cache write
# ---------------------------------------------------------------------------
def rope_table(rot, positions=64, dtype=torch.float32):
    freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).to(dtype).to(DEV)


def norm_case(tokens, hq, hkv, d, rot, neox, dtype, seed=0, offset=0, pad=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    width = (hq + 2 * hkv) * d + pad
    buf = torch.randn(tokens * width + offset, generator=g, device=DEV).to(dtype)
    qkv = buf[offset:].view(tokens, width)
    q, k, v = qkv[:, :hq * d], qkv[:, hq * d:(hq + hkv) * d], qkv[:, (hq + hkv) * d:(hq + 2 * hkv) * d]
    qw, kw = ((1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(dtype) for _ in range(2))
    pos = torch.randint(0, 64, (tokens,), generator=g, device=DEV)
    return q, k, v, qw, kw, pos


def want_norm(x, w, d, pos, table, neox, eps=1e-6):
    """The 64-bit result and what its fp32 arithmetic may be off by."""
    xs = x.cpu().reshape(x.shape[0], -1, d)
    ok = ((pos >= 0) & (pos < table.shape[0])).cpu()
    y = oracle.norm_rotate(xs, w.cpu(), eps, pos.cpu().clamp(0, table.shape[0] - 1), table.cpu(), neox)
    y[~ok] = xs[~ok].double()
    n = xs.double() / (xs.double().pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.cpu().double()
    half = table.shape[1] // 2
    size = n.abs()
    for i in range(half):
        a, b = (i, i + half) if neox else (2 * i, 2 * i + 1)
        size[..., a] = size[..., b] = n[..., a].abs() + n[..., b].abs()
    return y, size * 2.0**-20


def check_close(got, want, slack, dtype):
    got = got.cpu().double().reshape(want.shape)
    err = (got - want).abs()
    bound = half_step(dtype) * (want.abs() + slack) + slack
    if dtype == FP8:
        bound = bound + 2.0**-10
    elif dtype == FP16:
        bound = bound + 2.0**-25  # half of the smallest fp16
    assert bool((err <= bound).all()), f"max error / bound {(err / bound.clamp_min(1e-30)).max().item()}"


NORM_SHAPES = [(1, 4, 2, 128, 128), (5, 28, 4, 128, 64), (3, 14, 2, 64, 64), (7, 8, 8, 96, 96), (2, 6, 2, 192, 96),
               (4, 16, 2, 256, 256), (33, 5, 1, 80, 80), (3, 3, 1, 40, 24), (2, 3, 3, 18, 6), (2, 2, 2, 512, 128),
               (2, 3, 1, 7, 2), (130, 32, 8, 128, 128), (4, 3, 2, 128, 48), (3, 2, 1, 128, 8)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("shape", NORM_SHAPES, ids=str)
def test_norm_rotates_in_place_and_out_of_place(shape, neox, dtype):
    tokens, hq, hkv, d, rot = shape
    q, k, v, qw, kw, pos = norm_case(tokens, hq, hkv, d, rot, neox, dtype)
    table = rope_table(rot)
    wq, sq = want_norm(q, qw, d, pos, table, neox)
    wk, sk = want_norm(k, kw, d, pos, table, neox)
    q_out, k_out = torch.empty(tokens, hq, d, dtype=dtype, device=DEV), torch.empty(tokens, hkv * d, dtype=dtype, device=DEV)
    before = q.clone()
    dk.qk_norm_rotary_embedding(pos, q, k, qw, kw, 1e-6, d, table, neox, query_out=q_out, key_out=k_out)
    check_close(q_out, wq, sq, dtype)
    check_close(k_out, wk, sk, dtype)
    assert torch.equal(q, before)
    v_before = v.clone()
    got = dk.qk_norm_rotary_embedding(pos, q, k, qw, kw, 1e-6, d, table, neox)
    assert got[0].data_ptr() == q.data_ptr()
    assert torch.equal(q.reshape(-1), q_out.view(-1)) and torch.equal(k.reshape(-1), k_out.view(-1))
    assert torch.equal(v, v_before)


@pytest.mark.parametrize("cache_dtype", ["same", "fp8"])
@pytest.mark.parametrize("layout", ["nhd", "vllm", "odd"])
@pytest.mark.parametrize("shape", NORM_SHAPES, ids=str)
def test_norm_with_cache_write(shape, layout, cache_dtype):
    tokens, hq, hkv, d, rot = shape
    dtype = BF16 if tokens % 2 else FP16
    neox = d != 64
    offset, pad = (0, 0) if layout != "odd" else (1, 3)  # rows at odd addresses
    q, k, v, qw, kw, pos = norm_case(tokens, hq, hkv, d, rot, neox, dtype, seed=1, offset=offset, pad=pad)
    table = rope_table(rot, dtype=dtype if layout == "vllm" else torch.float32)
    block, blocks = 4, tokens // 4 + 2
    store = FP8 if cache_dtype == "fp8" else dtype
    raw = torch.full((blocks * block * hkv * 2 * d + 1,), 7, dtype=torch.uint8, device=DEV) if store == FP8 else \
        torch.full((blocks * block * hkv * 2 * d + 1,), 7.0, dtype=dtype, device=DEV)
    raw = raw[1:] if layout == "odd" else raw[:-1]
    kv = raw.view(blocks, hkv, block, 2 * d).transpose(1, 2)
    kc, vc = (kv[..., :d], kv[..., d:]) if layout != "nhd" else \
        tuple(x.view(blocks, block, hkv, d) for x in raw.view(2, -1))
    before_k, before_v = kc.clone(), vc.clone()
    if store == FP8:
        kc, vc = kc.view(FP8), vc.view(FP8)
    slots = torch.randperm(blocks * block, generator=torch.Generator().manual_seed(2))[:tokens].to(DEV)
    if tokens > 2:
        slots[1], slots[2] = -1, blocks * block + 5  # padding, and past the cache
    k_before = k.clone()
    q_out = torch.empty(tokens, hq * d, dtype=dtype, device=DEV)
    ks, vs = (0.02, 0.015) if store == FP8 else (1.0, 1.0)
    dk.qk_norm_rotary_embedding_and_cache(pos, q, k, v, qw, kw, 1e-6, d, table, neox, kc, vc, slots, k_scale=ks,
                                          v_scale=vs, query_out=q_out)
    wq, sq = want_norm(q, qw, d, pos, table, neox)
    wk, sk = want_norm(k, kw, d, pos, table, neox)
    check_close(q_out, wq, sq, dtype)
    assert torch.equal(k, k_before)
    put = torch.zeros(blocks * block, dtype=torch.bool)
    live = [t for t in range(tokens) if 0 <= slots[t] < blocks * block]
    at = slots[live].cpu()
    put[at] = True
    flat = lambda c: c.view(torch.uint8).cpu().reshape(-1, hkv, d).view(FP8) if store == FP8 else c.cpu().reshape(-1, hkv, d)
    got_k, got_v = flat(kc).float(), flat(vc).float()
    limit = (lambda x: x.clamp(-448, 448)) if store == FP8 else (lambda x: x)
    check_close(got_k[at], limit(wk[live] / ks), sk[live] / ks, store)
    vw = v.reshape(tokens, hkv, d)[live].cpu().double() / vs
    check_close(got_v[at], limit(vw), vw.abs() * (2.0**-24 if store == FP8 else 0.0), store)
    for c, b in ((kc, before_k), (vc, before_v)):
        same = (c.view(torch.uint8) if store == FP8 else c).cpu().reshape(-1, hkv, d)[~put]
        assert torch.equal(same, b.cpu().reshape(-1, hkv, d)[~put])


def test_norm_leaves_padding_as_it_was():
    d, rot = 128, 128
    q, k, v, qw, kw, pos = norm_case(6, 4, 2, d, rot, True, BF16)
    table = rope_table(rot)
    pos[1], pos[4] = -1, 64
    kc = torch.zeros(3, 4, 2, d, dtype=BF16, device=DEV)
    vc = torch.zeros_like(kc)
    slots = torch.arange(6, device=DEV) + 2
    q0, k0 = q.clone(), k.clone()
    dk.qk_norm_rotary_embedding_and_cache(pos, q, k, v, qw, kw, 1e-6, d, table, True, kc, vc, slots)
    for t in (1, 4):
        assert torch.equal(q[t], q0[t])
        assert not kc.view(-1, 2, d)[t + 2].any() and not vc.view(-1, 2, d)[t + 2].any()
    assert not torch.equal(q[0], q0[0])
    dk.qk_norm_rotary_embedding(pos, q, k, qw, kw, 1e-6, d, table, True)
    assert torch.equal(k[1], k0[1]) and torch.equal(k[4], k0[4]) and not torch.equal(k[0], k0[0])


def test_norm_zero_rows_infinities_and_saturation():
    d = 64
    q = torch.zeros(3, 2 * d, dtype=BF16, device=DEV)
    k = torch.zeros(3, d, dtype=BF16, device=DEV)
    q[1, 0] = float("inf")
    k[2] = 300.0
    w = torch.ones(d, dtype=BF16, device=DEV)
    table = rope_table(d)
    pos = torch.zeros(3, dtype=torch.int64, device=DEV)
    kc = torch.zeros(1, 4, 1, d, dtype=FP8, device=DEV)
    vc = torch.zeros(1, 4, 1, d, dtype=FP8, device=DEV)
    v = torch.full((3, d), 1e4, dtype=BF16, device=DEV)
    out = dk.qk_norm_rotary_embedding_and_cache(pos, q, k, v, w, w, 1e-6, d, table, True, kc, vc,
                                                torch.arange(3, device=DEV), k_scale=1e-3, v_scale=1.0)
    assert not out[0].any() and not out[2].any()
    assert bool(out[1, :d].isnan().any()) and not out[1, d:].any()  # that head only
    assert bool((vc.float()[0, :3] == 448).all()) and bool((kc.float()[0, 2] == 448).all())


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
class Batch:
    """A ragged batch over a paged cache whose blocks are shuffled."""

    def __init__(self, new, lens, hq, hkv, d, dtype=BF16, block=16, layout="nhd", fp8=False, seed=0, poison=True,
                 q_scale=1.0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.new, self.lens = new, lens
        self.starts = starts_of(new)
        need = [-(-n // block) for n in lens]
        blocks = sum(need) + 3
        perm = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed))
        self.tables = torch.full((len(new), max([1, *need])), -5, dtype=torch.int32)  # unused entries: nonsense
        at = 0
        for s, n in enumerate(need):
            self.tables[s, :n] = perm[at:at + n]
            at += n
        store = FP8 if fp8 else dtype
        randn = lambda *shape: torch.randn(*shape, generator=g, device=DEV)
        if layout == "nhd":
            k, v = randn(blocks, block, hkv, d), randn(blocks, block, hkv, d)
        elif layout == "hnd":
            k, v = (randn(blocks, hkv, block, d).transpose(1, 2) for _ in range(2))
        else:
            kv = randn(blocks, hkv, block, 2 * d).to(store).transpose(1, 2)
            k, v = kv[..., :d], kv[..., d:]
        self.k, self.v = (x if x.dtype == store else x.to(store) for x in (k, v))
        if poison:  # every place that holds no token
            flat = torch.zeros(blocks, block, dtype=torch.bool)
            for s, n in enumerate(lens):
                j = torch.arange(n)
                flat[self.tables[s].long()[j // block], j % block] = True
            for x in (self.k, self.v):
                bits = x.view(torch.uint8) if fp8 else x
                bits[~flat.to(DEV)] = 0x7F if fp8 else float("nan")
        self.tables = self.tables.to(DEV)
        self.q = (randn(self.starts[-1], hq, d) * q_scale).to(dtype)
        self.dtype, self.d, self.hq = dtype, d, hq
        self.scales = dict(k_scale=0.9, v_scale=1.1) if fp8 else {}

    def run(self, out=None, q=None, **kw):
        return dk.paged_attention_varlen(self.q if q is None else q, self.k, self.v, self.tables, int32(self.lens),
                                         int32(self.starts), out=out, **kw, **self.scales)

    def check(self, got, **kw):
        if "alibi_slopes" in kw:
            kw["slopes"] = kw.pop("alibi_slopes")
        if "prefix_lens" in kw:
            kw["prefix"] = kw.pop("prefix_lens").tolist()
        kw.setdefault("scale", self.d**-0.5)
        want, size = oracle.attention(self.q, self.k, self.v, self.tables, self.lens, self.starts, **kw, **self.scales)
        h = half_step(self.dtype)
        bound = h * want.abs() + (h + 2.0**-13) * size + 2.0**-25
        got = got.double()
        nan = want.isnan()
        assert bool((got.isnan() == nan).all())
        same_inf = want.isinf() & (got == want)
        ok = ((got - want).abs() <= bound) | nan | same_inf
        assert bool(ok.all()), f"max error / bound {((got - want).abs() / bound)[~nan].max().item()}, {int((~ok).sum())} off"


HEADS = [(4, 2, 128), (8, 2, 64), (3, 3, 96), (6, 2, 192), (8, 1, 256), (16, 1, 128), (7, 1, 128), (5, 5, 64), (9, 1, 192)]
RAGGED = {
    "decode": ([1, 1, 0, 1, 1, 1], [1, 17, 40, 700, 33, 1031]),
    "empty": ([1, 2, 1, 0, 3], [0, 1, 5, 0, 2]),  # lengths of zero, and below the new tokens
    "spec": ([3, 1, 5, 2, 4], [300, 64, 5, 1100, 33]),
    "prompts": ([1, 40, 129, 300], [1, 40, 500, 300]),
    "mixed": ([1, 260, 1, 33], [900, 700, 2, 100]),
}
FEATURES = {
    "plain": {},
    "window": dict(window=37),
    "window1": dict(window=1),
    "cap": dict(softcap=5.0),
    "alibi": dict(alibi=True),
    "prefix": dict(prefix=[9, 0, 70, 1000, 3, 18]),
    "all": dict(window=50, softcap=3.0, alibi=True, prefix=[5, 33, 7, 64, 0, 1]),
}


def features(name, hq, seqs):
    kw = dict(FEATURES[name])
    if kw.pop("alibi", False):
        kw["alibi_slopes"] = torch.tensor([2.0 ** (-1 - h % 7) for h in range(hq)], device=DEV)
    if "prefix" in kw:
        kw["prefix_lens"] = int32(kw.pop("prefix")[:seqs])
    return kw


@pytest.mark.parametrize("feature", FEATURES)
@pytest.mark.parametrize("shape", RAGGED)
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_attention(heads, shape, feature):
    hq, hkv, d = heads
    new, lens = RAGGED[shape]
    i = HEADS.index(heads) + list(RAGGED).index(shape)
    b = Batch(new, lens, hq, hkv, d, dtype=[BF16, FP16][i % 2], block=[16, 32, 1, 48, 8][i % 5],
              layout=["nhd", "hnd", "vllm"][i % 3], seed=i)
    kw = features(feature, hq, len(new))
    b.check(b.run(**kw), **kw)


@pytest.mark.parametrize("feature", ["plain", "all"])
@pytest.mark.parametrize("shape", RAGGED)
@pytest.mark.parametrize("heads", [h for h in HEADS if h[2] != 96], ids=str)
def test_attention_fp8_cache(heads, shape, feature):
    hq, hkv, d = heads
    new, lens = RAGGED[shape]
    i = HEADS.index(heads) + list(RAGGED).index(shape)
    b = Batch(new, lens, hq, hkv, d, dtype=[BF16, FP16][i % 2], block=[16, 64, 3][i % 3],
              layout=["nhd", "hnd", "vllm"][i % 3], fp8=True, seed=i)
    kw = features(feature, hq, len(new))
    b.check(b.run(**kw), **kw)


@pytest.mark.parametrize("heads", [(32, 8, 128), (2, 2, 64), (2, 1, 256)], ids=str)
def test_attention_long_contexts(heads):
    hq, hkv, d = heads
    b = Batch([1, 2, 1], [20000, 9000, 4097], hq, hkv, d, seed=3)
    b.check(b.run())
    kw = dict(window=3000, prefix_lens=int32([100, 0, 33]), softcap=20.0)
    b.check(b.run(**kw), **kw)
    b = Batch([600, 1], [9000, 12000], hq, hkv, d, seed=4)
    b.check(b.run())
    b.check(b.run(window=700), window=700)


def test_attention_many_sequences():
    g = torch.Generator().manual_seed(1)
    new = torch.randint(0, 3, (700,), generator=g).tolist()
    lens = [n + c for n, c in zip(new, torch.randint(0, 90, (700,), generator=g).tolist())]
    b = Batch(new, lens, 4, 1, 64, seed=5)
    b.check(b.run())
    new[350] = 150
    lens[350] += 150
    b = Batch(new, lens, 4, 1, 64, seed=5)
    b.check(b.run())


def test_attention_more_sequences_than_one_scan_takes():
    g = torch.Generator().manual_seed(2)
    new = torch.randint(0, 3, (2500,), generator=g).tolist()
    lens = [n + c for n, c in zip(new, torch.randint(0, 40, (2500,), generator=g).tolist())]
    b = Batch(new, lens, 2, 1, 64, seed=6)
    b.check(b.run(max_seq_len=5000))  # cut by shares
    b.check(b.run())
    for s in (3, 1023, 1024, 2047, 2048, 2499):
        new[s], lens[s] = 70, 90 + s % 7
    b = Batch(new, lens, 2, 1, 64, seed=6)
    b.check(b.run(max_seq_len=5000))


def test_attention_keys_and_values_laid_out_differently():
    for fp8 in (False, True):
        b = Batch([1, 90, 3], [700, 300, 50], 4, 2, 128, fp8=fp8)
        want = b.run()
        b.check(want)
        raw = b.v.view(torch.uint8) if fp8 else b.v
        b.v = raw.transpose(1, 2).contiguous().transpose(1, 2).view(b.v.dtype)
        assert b.v.stride() != b.k.stride() and torch.equal(b.run(), want)


def test_attention_shared_blocks():
    """Sequences that begin with the same cached blocks, and block size 1 to 100."""
    for block in (16, 7, 100):
        b = Batch([1, 40, 2], [400, 440, 402], 4, 2, 128, block=block, poison=False)
        b.tables[1:, :3 if block < 100 else 1] = b.tables[0, :3 if block < 100 else 1]
        b.check(b.run())


def test_attention_rows_behind_the_last_sequence_stay():
    b = Batch([3, 1, 40], [50, 9, 77], 4, 2, 128)
    q = torch.cat([b.q, torch.full((5, 4, 128), float("nan"), dtype=BF16, device=DEV)])
    out = torch.full_like(q, 3.0)
    b.run(out=out, q=q)
    assert bool((out[44:] == 3.0).all())
    b.check(out[:44])
    assert torch.equal(dk.paged_attention_varlen(q, b.k, b.v, b.tables, int32([]), int32([0]), out=torch.full_like(q, 2.0)),
                       torch.full_like(q, 2.0))


def test_attention_bounds_may_be_loose_and_rows_more_than_needed():
    b = Batch([3, 1, 40], [500, 9, 77], 4, 2, 128)
    want = b.run()
    b.check(want)
    b.check(b.run(max_query_len=1000, max_seq_len=40000))
    tables = torch.cat([b.tables, torch.full((3, b.tables.shape[1]), -1, dtype=torch.int32, device=DEV)])
    got = dk.paged_attention_varlen(b.q, b.k, b.v, tables, int32([*b.lens, 5, 6]), int32(b.starts))
    assert torch.equal(got, want)


def test_attention_strided_and_unaligned_queries_and_outputs():
    b = Batch([1, 33, 2], [40, 90, 700], 4, 2, 128)
    want = b.run()
    buf = torch.zeros(36 * (4 * 131 + 7) + 1, dtype=BF16, device=DEV)
    q = buf.as_strided((36, 4, 128), (4 * 131 + 7, 131, 1), 1)  # odd addresses and strides
    q.copy_(b.q)
    obuf = torch.full_like(buf, 9.0)
    out = obuf.as_strided((36, 4, 128), (4 * 131 + 7, 131, 1), 1)
    b.run(out=out, q=q)
    assert torch.equal(out, want)
    out.fill_(9.0)
    assert bool((obuf == 9.0).all())
    swapped = b.q.transpose(0, 1).contiguous().transpose(0, 1)  # head-major
    assert torch.equal(b.run(q=swapped, out=torch.empty_like(swapped)), want)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("heads", [(4, 2, 128), (2, 1, 256), (8, 2, 64)], ids=str)
def test_attention_hidden_values_have_no_influence(heads, bad):
    """Keys and values that some tokens of the batch see and others do not."""
    hq, hkv, d = heads
    for new, lens, at in (([4, 60, 1], [40, 200, 90], [(0, 38), (1, 150), (1, 199), (2, 3)]),
                          ([200], [200], [(0, 60), (0, 131)])):
        b = Batch(new, lens, hq, hkv, d, seed=7)
        kw = dict(window=24, prefix_lens=int32([2, 0, 0][:len(new)]))
        for s, j in at:
            page = int(b.tables[s, j // 16])
            b.v[page, j % 16, 0, 5] = bad
            b.v[page, j % 16, hkv - 1] = bad
        b.check(b.run(**kw), **kw)
        for s, j in at:
            page = int(b.tables[s, j // 16])
            b.k[page, j % 16, 0, 3] = float("nan")
        b.check(b.run(**kw), **kw)


def test_attention_block_entries_no_token_sees_are_not_used():
    b = Batch([1, 2, 40], [900, 1500, 1000], 4, 2, 128)
    kw = dict(window=64, prefix_lens=int32([10, 0, 16]))
    want = b.run(**kw)
    b.check(want, **kw)
    for s, (n, length, pre) in enumerate(zip(b.new, b.lens, [10, 0, 16])):
        first = (length - n - 63) // 16
        b.tables[s, -(-pre // 16):first] = 2**31 - 1
    assert torch.equal(b.run(**kw), want)


def test_attention_extreme_scores():
    b = Batch([1, 70], [300, 400], 4, 2, 128, q_scale=60.0)
    b.check(b.run(scale=1.0), scale=1.0)  # one key takes all
    b.check(b.run(scale=1.0, softcap=30.0), scale=1.0, softcap=30.0)
    b.check(b.run(scale=-0.2), scale=-0.2)
    b.check(b.run(scale=0.0), scale=0.0)  # the mean


@pytest.mark.parametrize("cap", [0.5, 50.0, 64.0, 65.0, 1e3, 1e4, 1e8])
def test_attention_caps_small_and_large(cap):
    b = Batch([1, 70], [300, 400], 4, 2, 128, dtype=FP16, q_scale=4.0)
    b.check(b.run(softcap=cap), softcap=cap)


def test_attention_of_an_empty_cache():
    q = torch.randn(3, 4, 64, device=DEV).to(BF16)
    cache = torch.empty(0, 16, 2, 64, dtype=BF16, device=DEV)
    for columns in (0, 2):
        tables = torch.zeros(2, columns, dtype=torch.int32, device=DEV)
        out = dk.paged_attention_varlen(q, cache, cache, tables, int32([5, 5]), int32([0, 1, 3]), out=torch.ones_like(q))
        assert not out.any()
    b = Batch([1], [9], 4, 2, 64)
    assert not dk.paged_attention_varlen(b.q, b.k, b.v, b.tables, int32([9]), int32([0, 1]), max_seq_len=0).any()
    assert dk.paged_attention_varlen(q[:0], b.k, b.v, b.tables, int32([9]), int32([0, 0])).shape == (0, 4, 64)


def test_attention_reads_every_e4m3_value():
    """V of all 254 e4m3fn numbers, each attended to alone (window 1), and q.K
    of a unit query with them."""
    codes = torch.tensor([c for c in range(256) if c % 128 != 127], dtype=torch.uint8)
    n = codes.numel()
    for dtype in (BF16, FP16):
        for new in ([1] * n, [n]):  # one token each, and a prompt
            seqs = len(new)
            v = codes.to(DEV).view(FP8)
            cache = torch.zeros(n, 1, 1, 64, dtype=torch.uint8, device=DEV).view(FP8)
            cache.view(torch.uint8)[:] = codes.to(DEV)[:, None, None, None]
            tables = torch.arange(n, dtype=torch.int32, device=DEV).view(seqs, -1)
            lens = [1] * n if seqs > 1 else [n]
            q = torch.zeros(n, 1, 64, dtype=dtype, device=DEV)
            q[..., 0] = 1
            out = dk.paged_attention_varlen(q, cache, cache, tables, int32(lens), int32(starts_of(new)), window=1,
                                            scale=1.0)
            assert torch.equal(out[:, 0, 0].float(), v.float()) and torch.equal(out[:, 0, 63].float(), v.float())


@pytest.mark.parametrize("seed", range(48))
def test_attention_random_batches(seed):
    """Any mixture of sizes, features, layouts and types."""
    g = torch.Generator().manual_seed(1000 + seed)
    pick = lambda *v: v[int(torch.randint(len(v), (1,), generator=g))]
    upto = lambda n: int(torch.randint(n, (1,), generator=g))
    fp8 = upto(3) == 0
    d = pick(64, 128, 192, 256) if fp8 else pick(64, 96, 128, 192, 256)
    hkv = pick(1, 2, 3)
    hq = hkv * pick(1, 2, 3, 5, 8, 16)
    seqs = pick(1, 2, 5, 9)
    style = pick("one", "few", "many", "mixed")
    new = [{"one": upto(2), "few": upto(6), "many": upto(200), "mixed": pick(0, 1, 1, upto(300))}[style] for _ in range(seqs)]
    top = pick(1, 40, 700, 3000)
    lens = [max(0, n + upto(top) - (2 if upto(9) == 0 else 0)) for n in new]
    b = Batch(new, lens, hq, hkv, d, dtype=pick(BF16, FP16), block=pick(1, 8, 16, 16, 32, 40, 48), fp8=fp8,
              layout=pick("nhd", "hnd", "vllm"), seed=seed)
    kw = {}
    if upto(2):
        kw["window"] = pick(1, 5, 64, 300, 5000)
    if upto(3) == 0:
        kw["softcap"] = pick(2.0, 30.0)
    if upto(3) == 0:
        kw["alibi_slopes"] = torch.rand(hq, generator=g).to(DEV)
    if upto(2):
        kw["prefix_lens"] = int32([upto(100) for _ in new])
    if b.starts[-1] == 0:
        return
    b.check(b.run(**kw), **kw)


def test_attention_through_the_c_interface_with_and_without_workspace():
    L = capi.lib()
    stream = torch.cuda.current_stream().cuda_stream
    for new, lens in (([1, 1, 1], [5000, 70, 3000]), ([300, 1], [4000, 2000]), ([3, 2], [2000, 900])):
        b = Batch(new, lens, 8, 2, 128)
        out = torch.full_like(b.q, 7.0)
        dlens, dstarts = int32(lens), int32(b.starts)
        p = capi.varlen_attn_params(out, b.q, b.k, b.v, b.tables, dlens, dstarts, 128**-0.5, window=1500)
        args = (capi.dtype_code(BF16), 128, max(new), max(lens))
        size = L.dk_paged_attention_varlen_workspace_bytes(ctypes.byref(p), *args[1:])
        assert size > 0
        ws = torch.full((size // 4 + 64,), float("nan"), device=DEV)  # nothing of it has to be set before
        guard = ws[size // 4:]
        guard.fill_(3.0)
        assert L.dk_paged_attention_varlen(ctypes.byref(p), *args, ws.data_ptr(), size, stream) == 0, capi.last_error()
        b.check(out, window=1500)
        assert bool((guard == 3.0).all())
        assert torch.equal(out, b.run(window=1500))
        for ptr, have in ((None, 0), (ws.data_ptr(), size - 4)):
            out.fill_(7.0)
            assert L.dk_paged_attention_varlen(ctypes.byref(p), *args, ptr, have, stream) == 0, capi.last_error()
            b.check(out, window=1500)


def test_norm_and_slots_through_the_c_interface():
    L = capi.lib()
    stream = torch.cuda.current_stream().cuda_stream
    q, k, v, qw, kw, pos = norm_case(9, 4, 2, 128, 128, True, BF16)
    table = rope_table(128)
    r = capi.rotary_params(pos, q, k, 128, table, True)
    q_out, k_out = (torch.empty(9, h * 128, dtype=BF16, device=DEV) for h in (4, 2))
    n = capi.qk_norm_params(qw, kw, 1e-6, 128, q_out, k_out)
    assert L.dk_qk_norm_rotary_embedding(ctypes.byref(r), ctypes.byref(n), capi.DK_BFLOAT16, stream) == 0
    want = dk.qk_norm_rotary_embedding(pos, q.clone(), k.clone(), qw, kw, 1e-6, 128, table, True)
    assert torch.equal(q_out, want[0]) and torch.equal(k_out, want[1])
    kc, vc = (torch.zeros(2, 8, 2, 128, dtype=BF16, device=DEV) for _ in range(2))
    slots = torch.arange(9, device=DEV) + 3
    c = capi.cache_write_params(k, v, kc, vc, slots)
    n = capi.qk_norm_params(qw, kw, 1e-6, 128, q_out.fill_(0))
    assert L.dk_qk_norm_rotary_embedding_and_cache(ctypes.byref(r), ctypes.byref(n), ctypes.byref(c), capi.DK_BFLOAT16,
                                                   stream) == 0
    assert torch.equal(q_out, want[0]) and torch.equal(kc.view(-1, 256)[3:12], want[1])
    starts, lens, tables = int32([0, 2, 3]), int32([20, 1]), int32([[4, 0], [0, 0]])
    p64, s64, taken = (torch.empty(3, dtype=t, device=DEV) for t in (torch.int64, torch.int64, torch.int32))
    s = capi.slot_mapping_params(starts, lens, tables, 16, p64, s64, int32([9, 8, 7]), taken)
    assert L.dk_build_slot_mapping(ctypes.byref(s), stream) == 0
    assert p64.tolist() == [18, 19, 0] and taken[0].item() == 1
    assert s64.tolist() == [2, 3, 9 * 16]  # block 1 of sequence 0 is held: entry 0; sequence 1 takes block 9


def test_attention_offsets_past_32_bits():
    """Blocks more than 2^32 elements into the cache."""
    hq, hkv, d, block = 4, 2, 128, 16
    b = Batch([1, 50], [200, 90], hq, hkv, d, poison=False)
    blocks = 2**32 // (block * hkv * d) + b.k.shape[0] + 1
    first = blocks - b.k.shape[0]
    k = torch.empty(blocks, block, hkv, d, dtype=BF16, device=DEV)
    v = torch.empty_like(k)
    k[first:], v[first:] = b.k, b.v
    got = dk.paged_attention_varlen(b.q, k, v, torch.where(b.tables >= 0, b.tables + first, b.tables), int32(b.lens),
                                    int32(b.starts))
    assert torch.equal(got, b.run())


def test_attention_repeats_bit_for_bit_and_runs_on_another_stream():
    b = Batch([1, 33, 2, 1], [4000, 90, 700, 2100], 4, 2, 128)
    want = b.run()
    assert torch.equal(b.run(), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = b.run()
    side.synchronize()
    assert torch.equal(got, want)


# ---------------------------------------------------------------------------
# The three in a row, as a layer of a serving step runs them
# ---------------------------------------------------------------------------
class Engine:
    """One layer's attention step with its cache, over static buffers."""

    def __init__(self, seqs, tokens, hq=8, hkv=2, d=128, block=16, columns=20, dtype=BF16, fp8=False, **kw):
        self.hq, self.hkv, self.d, self.block, self.dtype, self.kw = hq, hkv, d, block, dtype, kw
        blocks = seqs * columns
        store = FP8 if fp8 else dtype
        self.kc, self.vc = (torch.zeros(blocks, block, hkv, d, dtype=dtype, device=DEV).to(store) for _ in range(2))
        self.scales = dict(k_scale=0.02, v_scale=0.02) if fp8 else {}
        self.free = torch.randperm(blocks, generator=torch.Generator().manual_seed(0)).to(torch.int32).to(DEV)
        self.used = 0
        self.tables = torch.zeros(seqs, columns, dtype=torch.int32, device=DEV)
        self.starts = torch.zeros(seqs + 1, dtype=torch.int32, device=DEV)
        self.lens = torch.zeros(seqs, dtype=torch.int32, device=DEV)
        self.qkv = torch.zeros(tokens, (hq + 2 * hkv) * d, dtype=dtype, device=DEV)
        self.free_now = torch.zeros_like(self.free)
        self.out = torch.zeros(tokens, hq, d, dtype=dtype, device=DEV)
        g = torch.Generator(device=DEV).manual_seed(1)
        self.qw, self.kw_ = ((1 + 0.1 * torch.randn(d, generator=g, device=DEV)).to(dtype) for _ in range(2))
        self.table = rope_table(d, 512)
        self.taken = torch.zeros(1, dtype=torch.int32, device=DEV)

    def step(self):
        hq, hkv, d = self.hq, self.hkv, self.d
        pos, slots, _ = dk.build_slot_mapping(self.starts, self.lens, self.tables, self.block, self.qkv.shape[0],
                                              free_blocks=self.free_now, num_new_blocks=self.taken)
        q, k, v = self.qkv.split([hq * d, hkv * d, hkv * d], dim=1)
        dk.qk_norm_rotary_embedding_and_cache(pos, q, k, v, self.qw, self.kw_, 1e-6, d, self.table, True, self.kc,
                                              self.vc, slots, **self.scales)
        return dk.paged_attention_varlen(q.view(-1, hq, d), self.kc, self.vc, self.tables, self.lens, self.starts,
                                         max_query_len=self.qkv.shape[0], max_seq_len=320, out=self.out, **self.kw,
                                         **self.scales)

    def feed(self, new, lens, qkv):
        self.starts.copy_(int32(starts_of(new)))
        self.lens.copy_(int32(lens))
        self.qkv.zero_()
        self.qkv[:qkv.shape[0]] = qkv
        self.free_now.copy_(torch.roll(self.free, -self.used))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("captured", [False, True])
def test_step_of_a_serving_layer(captured, fp8):
    """A prompt step, then decode and speculation steps; captured, one graph
    serves them all, with the lengths, tables and tokens of each step in its
    buffers, replayed between eager work and checked each time."""
    seqs, tokens = 4, 160
    kw = dict(window=100, softcap=20.0)
    e = Engine(seqs, tokens, fp8=fp8, **kw)
    steps = [[100, 0, 37, 23], [1, 5, 1, 1], [1, 90, 4, 1], [1, 1, 0, 3], [0, 0, 0, 1]]
    hq, hkv, d = e.hq, e.hkv, e.d
    graph = None
    if captured:
        e.feed([0] * seqs, [0] * seqs, e.qkv[:0])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            e.step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            e.step()
    lens = [0] * seqs
    keys = [torch.zeros(0, hkv, d, dtype=torch.float64) for _ in range(seqs)]
    vals = [torch.zeros(0, hkv, d, dtype=torch.float64) for _ in range(seqs)]
    g = torch.Generator(device=DEV).manual_seed(2)
    for new in steps:
        lens = [a + b for a, b in zip(lens, new)]
        n = sum(new)
        qkv = torch.randn(n, (hq + 2 * hkv) * d, generator=g, device=DEV).to(e.dtype)
        e.feed(new, lens, qkv)
        e.out.fill_(5.0)
        if captured:
            graph.replay()
        else:
            e.step()
        torch.cuda.synchronize()
        e.used += int(e.taken)
        assert bool((e.out[n:] == 5.0).all()) and not e.qkv[n:].any()
        # 64-bit: norm, rotate and gather per sequence, over the caches as they were written.
        starts = starts_of(new)
        for s in range(seqs):
            rows = qkv[starts[s]:starts[s + 1]].cpu()
            pos = torch.arange(lens[s] - new[s], lens[s])
            k = oracle.norm_rotate(rows[:, hq * d:(hq + hkv) * d].reshape(-1, hkv, d), e.kw_.cpu(), 1e-6, pos,
                                   e.table.cpu(), True)
            keys[s] = torch.cat([keys[s], k])
            vals[s] = torch.cat([vals[s], rows[:, (hq + hkv) * d:].reshape(-1, hkv, d).double()])
            j = torch.arange(lens[s])
            page = e.tables[s].cpu().long()[j // e.block]
            store = FP8 if fp8 else e.dtype
            for cache, want in ((e.kc, keys[s]), (e.vc, vals[s])):
                got = cache.float().cpu()[page, j % e.block].double()
                scale = 0.02 if fp8 else 1.0
                w = (want / scale).clamp(-448, 448) if fp8 else want
                assert bool(((got - w).abs() <= half_step(store) * w.abs() * (1 + 2.0**-10) + 2.0**-9).all())
        q = e.qkv[:n].view(n, -1, d)[:, :hq].contiguous()
        want, size = oracle.attention(q, e.kc, e.vc, e.tables, lens, starts, d**-0.5, **kw, **e.scales)
        h = half_step(e.dtype)
        assert bool(((e.out[:n].double() - want).abs() <= h * want.abs() + (h + 2.0**-13) * size).all())


def test_two_captured_graphs_do_not_share_their_partial_results():
    bs = [Batch([1, 1, 1], lens, 8, 2, 128, seed=i) for i, lens in enumerate(([5000, 70, 3000], [4000, 4100, 9]))]
    graphs, outs, wants = [], [], []
    for b in bs:
        wants.append(b.run())
        lens, starts = int32(b.lens), int32(b.starts)
        out = torch.zeros_like(b.q)
        call = lambda: dk.paged_attention_varlen(b.q, b.k, b.v, b.tables, lens, starts, max_query_len=1,
                                                 max_seq_len=max(b.lens), out=out)
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        graphs.append((graph, lens, starts))
        outs.append(out)
    side = torch.cuda.Stream()
    for _ in range(3):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
        torch.cuda.synchronize()
        for out, want in zip(outs, wants):
            assert torch.equal(out, want)
        assert torch.equal(bs[0].run(), wants[0])


# ---------------------------------------------------------------------------
# Refusals
# ---------------------------------------------------------------------------
def refuse(match, call):
    with pytest.raises((RuntimeError, ValueError), match=match):
        call()


def test_refusals():
    b = Batch([1, 2], [20, 9], 4, 2, 128, poison=False)
    lens, starts = int32(b.lens), int32(b.starts)

    def attn(q=b.q, k=b.k, v=b.v, tables=b.tables, lens=lens, starts=starts, **kw):
        return lambda: dk.paged_attention_varlen(q, k, v, tables, lens, starts, **{"max_query_len": 2, "max_seq_len": 20, **kw})

    refuse("same shape", attn(out=b.q[:1]))
    refuse("dtype mismatch", attn(q=b.q.half()))
    refuse("float16 or bfloat16", attn(q=b.q.float(), k=b.k.float(), v=b.v.float()))
    refuse("shapes differ", attn(v=b.v[:1]))
    refuse("does not match q", attn(q=b.q[..., :64]))
    refuse("contiguous", attn(q=b.q.transpose(1, 2).contiguous().transpose(1, 2)))
    refuse("multiple of num_kv_heads", attn(q=b.q[:, :3]))
    refuse("head_dim", attn(q=b.q[..., :32].contiguous(), k=b.k[..., :32].contiguous(), v=b.v[..., :32].contiguous()))
    refuse("at least 2", attn(lens=lens[:1]))
    refuse("at least 2 rows", attn(tables=b.tables[:1]))
    refuse("int32", attn(lens=lens.long()))
    refuse("int32", attn(starts=starts.long()))
    refuse("int32", attn(tables=b.tables.long()))
    refuse("window", attn(window=-1))
    refuse("softcap", attn(softcap=-1.0))
    refuse("softcap", attn(softcap=float("nan")))
    refuse("scale", attn(scale=float("inf")))
    refuse("alibi_slopes", attn(alibi_slopes=torch.ones(3, device=DEV)))
    refuse("alibi_slopes", attn(alibi_slopes=torch.ones(4, device=DEV, dtype=BF16)))
    refuse("prefix_lens", attn(prefix_lens=int32([1])))
    refuse("non-negative", attn(max_seq_len=-1))
    refuse("fp8", attn(k_scale=2.0))
    refuse("multiples of 16 bytes", attn(k=torch.zeros(b.k.numel() + 1, dtype=BF16, device=DEV)[1:].view(b.k.shape)))
    refuse("same device", attn(lens=lens.cpu()))
    many = torch.zeros(3, 34, 128, dtype=BF16, device=DEV)
    refuse("GQA group", attn(q=many))

    table = rope_table(128)
    pos = torch.zeros(3, dtype=torch.int64, device=DEV)
    q, k = torch.zeros(3, 512, dtype=BF16, device=DEV), torch.zeros(3, 256, dtype=BF16, device=DEV)
    w = torch.ones(128, dtype=BF16, device=DEV)

    def norm(pos=pos, q=q, k=k, qw=w, kw=w, eps=1e-6, d=128, table=table, **kws):
        return lambda: dk.qk_norm_rotary_embedding(pos, q, k, qw, kw, eps, d, table, **kws)

    refuse("head_size", norm(qw=w[:64]))
    refuse("dtype mismatch", norm(kw=w.half()))
    refuse("int64", norm(pos=pos.int()))
    refuse("one row per position", norm(pos=pos[:2]))
    refuse("multiple of head_size", norm(d=96, qw=w[:96], kw=w[:96], table=rope_table(96)))
    refuse("rot_dim", norm(table=rope_table(256)))
    refuse("eps", norm(eps=-1.0))
    refuse("query's heads", norm(query_out=k))
    refuse("float32 or the query dtype", norm(table=table.half()))
    cache = torch.zeros(2, 4, 2, 128, dtype=BF16, device=DEV)
    slots = torch.zeros(3, dtype=torch.int64, device=DEV)

    def put(kc=cache, vc=cache, slots=slots, v=k, **kws):
        return lambda: dk.qk_norm_rotary_embedding_and_cache(pos, q, k, v, w, w, 1e-6, 128, table, True, kc, vc, slots, **kws)

    refuse("one key / value row per slot", put(slots=slots[:2]))
    refuse("head", put(kc=cache[:, :, :1], vc=cache[:, :, :1]))
    refuse("fp8", put(k_scale=0.5))
    refuse("k_scale", put(kc=cache.to(FP8), vc=cache.to(FP8), k_scale=0.0))

    def slot(starts=starts, lens=lens, tables=b.tables, block=16, n=3, **kws):
        return lambda: dk.build_slot_mapping(starts, lens, tables, block, n, **kws)

    refuse("block_size", slot(block=0))
    refuse("at least 2", slot(lens=lens[:1]))
    refuse("int32", slot(free_blocks=torch.zeros(3, dtype=torch.int64, device=DEV)))
    refuse("num_tokens", slot(positions=slots[:2]))
    refuse("same size", slot(slot_mapping=slots[:2]))
    refuse("int64", slot(slot_mapping=slots.int()))
