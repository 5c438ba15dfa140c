"""CPU tests of the ragged batch's attention step: argument checks of the C
entries (every call here is refused, or has nothing to do, before any HIP
call), the workspace's size, the Python wrappers under fake tensors, and the
64-bit definitions against plain formulas."""

import ctypes
import math

import pytest
import torch

import decodekernels_amd as dk
from decodekernels_amd import capi
from oracle import ragged_step as oracle

FAKE = 0x10000  # never dereferenced


def test_params_structs_match_the_header():
    assert ctypes.sizeof(capi.SlotMappingParams) == 7 * 8 + 8 + 5 * 4 + 4  # padded to 8
    assert ctypes.sizeof(capi.QkNormParams) == 4 * 8 + 4 * 8 + 8
    assert ctypes.sizeof(capi.VarlenAttnParams) == 9 * 8 + 11 * 8 + 8 * 4 + 2 * 4
    assert capi.VarlenAttnParams.softcap.offset == 196


def attn_params(**kw):
    p = capi.VarlenAttnParams()
    for name in ("out", "q", "k_cache", "v_cache", "block_tables", "seq_lens", "query_start_loc"):
        setattr(p, name, FAKE)
    p.q_stride_token, p.q_stride_head, p.out_stride_token, p.out_stride_head = 1024, 128, 1024, 128
    p.k_stride_block, p.k_stride_token, p.k_stride_head = 4096, 256, 128
    p.v_stride_block, p.v_stride_token, p.v_stride_head = 4096, 256, 128
    p.bt_stride, p.num_tokens, p.num_seqs, p.num_q_heads, p.num_kv_heads = 8, 4, 2, 8, 2
    p.block_size, p.num_blocks, p.max_blocks, p.scale = 16, 100, 8, 0.1
    for name, value in kw.items():
        setattr(p, name, value)
    return p


def attn(p, dtype=capi.DK_BFLOAT16, head_dim=128, most_new=1, most=100, ws=None, size=0):
    return capi.lib().dk_paged_attention_varlen(ctypes.byref(p), dtype, head_dim, most_new, most, ws, size, None)


@pytest.mark.parametrize(
    "fields,call,message",
    [
        (dict(num_q_heads=34), {}, "GQA group"),
        (dict(num_q_heads=7), {}, "multiple of num_kv_heads"),
        (dict(num_kv_heads=0), {}, "multiple of num_kv_heads"),
        ({}, dict(head_dim=80), "head_dim"),
        ({}, dict(head_dim=512), "head_dim"),
        ({}, dict(dtype=2), "float16 or bfloat16"),
        (dict(block_size=0), {}, "block_size"),
        (dict(num_tokens=-1), {}, "non-negative"),
        ({}, dict(most=-1), "non-negative"),
        (dict(window=-1), {}, "window"),
        (dict(softcap=-1.0), {}, "softcap"),
        (dict(softcap=math.inf), {}, "softcap"),
        (dict(softcap=1e-44, scale=1e30), {}, "fp32's range"),
        (dict(scale=math.nan), {}, "scale"),
        (dict(q=None), {}, "NULL"),
        (dict(query_start_loc=None), {}, "NULL"),
        (dict(block_tables=None), {}, "NULL"),
        (dict(k_cache=FAKE + 8), {}, "16 bytes"),
        (dict(v_stride_token=132), {}, "16 bytes"),
        (dict(k_stride_block=-4096), {}, "strides"),
        (dict(bt_stride=1 << 31), {}, "strides"),
        (dict(num_tokens=1 << 30), {}, "too many"),
        ({}, dict(most=5000, ws=FAKE + 4, size=1 << 30), "workspace must be 16-byte aligned"),
    ],
)
def test_attention_refusals(fields, call, message):
    if message.startswith("workspace"):
        fields = dict(max_blocks=400)
    assert attn(attn_params(**fields), **call) == capi.HIP_ERROR_INVALID_VALUE
    assert message in capi.last_error()


def test_attention_fp8_refusals():
    call = capi.lib().dk_paged_attention_varlen_fp8
    p = attn_params()
    for k_scale, v_scale, d, message in ((0.0, 1.0, 128, "k_scale"), (1.0, math.inf, 128, "v_scale"), (1.0, 1.0, 96, "head_dim")):
        assert call(ctypes.byref(p), capi.DK_FLOAT16, d, 1, 100, k_scale, v_scale, None, 0, None) == 1
        assert message in capi.last_error()
    p.k_stride_token = 8  # 8 bytes of e4m3fn
    assert call(ctypes.byref(p), capi.DK_FLOAT16, 128, 1, 100, 1.0, 1.0, None, 0, None) == 1
    assert "16 bytes" in capi.last_error()


def test_attention_with_nothing_to_do():
    for fields in (dict(num_tokens=0), dict(num_seqs=0), dict(num_tokens=0, q=None, out=None)):
        assert attn(attn_params(**fields)) == 0
    assert capi.lib().dk_paged_attention_varlen(None, 1, 128, 1, 1, None, 0, None) == 1


def test_workspace_size():
    def size(d=128, most_new=1, most=100, **kw):
        return capi.lib().dk_paged_attention_varlen_workspace_bytes(ctypes.byref(attn_params(**kw)), d, most_new, most)

    assert size(most=512, max_blocks=400) == 0  # never cut
    # 256 shares a KV head and 2 sequences, 4 rows a slot of 128 sums and 2 more floats, 2 numbers a (sequence, head).
    assert size(most=5000, max_blocks=400) == 4 * ((256 + 2) * 2 * 4 * 130 + 2 * 2 * 2)
    assert size(most=5000, max_blocks=30) == 0  # the tables hold 480 tokens
    assert size(most=5000, max_blocks=400, window=100) == 0
    assert size(most=5000, max_blocks=400, window=100, prefix_lens=FAKE) > 0
    assert size(most_new=4, most=5000, max_blocks=400) > size(most=5000, max_blocks=400)
    assert size(most_new=4, most=5000, max_blocks=400, num_q_heads=34) == 0  # refused by the call
    assert size(most=5000, max_blocks=400, num_seqs=0) == 0


def norm_params(**kw):
    r, n, c = capi.RotaryParams(), capi.QkNormParams(), capi.CacheWriteParams()
    r.positions = r.query = r.key = r.cos_sin_cache = FAKE
    r.q_stride_token, r.q_stride_head, r.k_stride_token, r.k_stride_head, r.cache_stride = 1024, 128, 1024, 128, 128
    r.num_tokens, r.num_q_heads, r.num_kv_heads, r.head_size, r.rot_dim, r.max_position = 3, 4, 2, 128, 128, 10
    r.cache_dtype = capi.DK_FLOAT32
    n.q_weight = n.k_weight = n.query_out = n.key_out = FAKE
    n.eps = 1e-6
    c.key = c.value = c.key_cache = c.value_cache = c.slot_mapping = FAKE
    c.k_stride_token, c.k_stride_head, c.v_stride_token, c.v_stride_head = 1024, 128, 1024, 128
    c.num_tokens, c.num_kv_heads, c.head_size, c.block_size, c.num_blocks = 3, 2, 128, 16, 4
    for name, value in kw.items():
        which, field = name.split("_", 1)
        setattr(dict(r=r, n=n, c=c)[which], field, value)
    return r, n, c


@pytest.mark.parametrize(
    "fields,cached,message",
    [
        (dict(r_rot_dim=130), False, "rot_dim"),
        (dict(r_rot_dim=7), False, "rot_dim"),
        (dict(r_head_size=0), False, "head_size"),
        (dict(r_cache_dtype=capi.DK_FLOAT16), False, "cos_sin_cache"),
        (dict(n_eps=-1.0), False, "eps"),
        (dict(n_eps=math.nan), False, "eps"),
        (dict(n_q_weight=None), False, "q_weight"),
        (dict(n_key_out=None), False, "key_out"),
        (dict(r_positions=None), False, "positions"),
        (dict(r_num_tokens=-1), False, "non-negative"),
        (dict(r_num_tokens=2**30), False, "too many"),
        (dict(c_num_tokens=2), True, "token counts"),
        (dict(c_num_kv_heads=3), True, "head counts"),
        (dict(c_key=FAKE + 64), True, "same tensor"),
        (dict(c_block_size=0), True, "block_size"),
        (dict(c_slot_mapping=None), True, "slot_mapping"),
    ],
)
def test_norm_refusals(fields, cached, message):
    r, n, c = norm_params(**fields)
    L = capi.lib()
    if cached:
        rc = L.dk_qk_norm_rotary_embedding_and_cache(ctypes.byref(r), ctypes.byref(n), ctypes.byref(c), 1, None)
    else:
        rc = L.dk_qk_norm_rotary_embedding(ctypes.byref(r), ctypes.byref(n), 1, None)
    assert rc == capi.HIP_ERROR_INVALID_VALUE and message in capi.last_error()


def test_norm_scales_and_nothing_to_do():
    L = capi.lib()
    r, n, c = norm_params()
    for scales in ((0.0, 1.0), (1.0, math.nan), (math.inf, 1.0)):
        rc = L.dk_qk_norm_rotary_embedding_and_cache_fp8(ctypes.byref(r), ctypes.byref(n), ctypes.byref(c), 1, *scales, None)
        assert rc == 1 and "k_scale and v_scale" in capi.last_error()
    r, n, c = norm_params(r_num_tokens=0, c_num_tokens=0)
    assert L.dk_qk_norm_rotary_embedding_and_cache(ctypes.byref(r), ctypes.byref(n), ctypes.byref(c), 1, None) == 0
    assert L.dk_qk_norm_rotary_embedding(ctypes.byref(r), ctypes.byref(n), 1, None) == 0
    assert L.dk_qk_norm_rotary_embedding(None, None, 1, None) == 1


@pytest.mark.parametrize(
    "fields,message",
    [
        (dict(block_size=0), "block_size"),
        (dict(num_seqs=-1), "non-negative"),
        (dict(num_tokens=2**31 - 1), "too many"),
        (dict(query_start_loc=None), "query_start_loc"),
        (dict(block_tables=None), "block_tables"),
        (dict(slot_mapping=None), "slot_mapping"),
        (dict(bt_stride=3), "overlap"),
        (dict(num_free_blocks=4), "free_blocks"),
    ],
)
def test_slot_refusals(fields, message):
    p = capi.SlotMappingParams()
    p.query_start_loc = p.seq_lens = p.block_tables = p.positions = p.slot_mapping = FAKE
    p.num_seqs, p.num_tokens, p.block_size, p.max_blocks, p.bt_stride = 2, 5, 16, 4, 4
    for name, value in fields.items():
        setattr(p, name, value)
    assert capi.lib().dk_build_slot_mapping(ctypes.byref(p), None) == capi.HIP_ERROR_INVALID_VALUE
    assert message in capi.last_error()


def test_fake_tensors_trace_through():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        q = torch.empty(5, 8, 128, dtype=torch.bfloat16, device="cuda")
        cache = torch.empty(9, 16, 2, 128, dtype=torch.bfloat16, device="cuda")
        i32 = lambda *shape: torch.empty(shape, dtype=torch.int32, device="cuda")
        pos, slots, taken = dk.build_slot_mapping(i32(3), i32(2), i32(2, 4), 16, 5, free_blocks=i32(7))
        assert pos.shape == slots.shape == (5,) and pos.dtype == torch.int64 and taken.shape == (1,)
        kv = torch.empty(5, 256, dtype=torch.bfloat16, device="cuda")
        w, table = torch.empty(128, dtype=torch.bfloat16, device="cuda"), torch.empty(64, 128, device="cuda")
        out = dk.qk_norm_rotary_embedding_and_cache(pos, q, kv, kv, w, w, 1e-6, 128, table, True, cache, cache, slots)
        assert out.shape == q.shape
        assert dk.qk_norm_rotary_embedding(pos, q, kv, w, w, 1e-6, 128, table)[1].shape == kv.shape
        out = dk.paged_attention_varlen(q, cache, cache, i32(2, 4), i32(2), i32(3), max_query_len=3, max_seq_len=60)
        assert out.shape == q.shape and out.dtype == q.dtype


def test_definition_of_attention_against_softmax():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(7, h, 16, generator=g, dtype=torch.float64) for h in (4, 2, 2))
    tables = torch.tensor([[1, 0]], dtype=torch.int32)
    kc, vc = (torch.cat([x[4:], x[:1] * 0, x[:4]]).view(2, 4, 2, 16) for x in (k, v))  # block 1 first
    want = torch.nn.functional.scaled_dot_product_attention(
        q.transpose(0, 1), k.repeat_interleave(2, 1).transpose(0, 1), v.repeat_interleave(2, 1).transpose(0, 1), is_causal=True)
    got, size = oracle.attention(q, kc, vc, tables, [7], [0, 7], 0.25)
    assert torch.allclose(got, want.transpose(0, 1), rtol=1e-12, atol=1e-12) and bool((size >= got.abs() - 1e-12).all())
    got, _ = oracle.attention(q, kc, vc, tables, [7], [0, 7], 0.25, window=1)
    assert torch.allclose(got, v.repeat_interleave(2, 1), rtol=1e-12, atol=1e-12)  # each sees itself
    assert oracle.visible(3, 9, 2, 1).tolist() == [True, False, True, True, False, False, False, False, False]


def test_definition_of_slots_by_hand():
    # 5 cached tokens in block 7; 4 new ones: 3 in block 7, one in a new block; then a fresh sequence.
    got = oracle.slot_mapping([0, 4, 6], [9, 2], [[7, -1], [-1, -1]], 8, 7, [3, 5, 4])
    assert got == ([5, 6, 7, 8, 0, 1, -1], [61, 62, 63, 24, 40, 41, -1], [[7, 3], [5, -1]], 2)


def test_definition_of_norm_and_rotation():
    x = torch.tensor([[[3.0, 4.0, 0.0, 0.0]]])
    table = torch.tensor([[1.0, 1.0, 0.0, 0.0], [0.0, 1.0, 1.0, 0.0]])  # position 1 turns the first pair a quarter
    inv = 1 / math.sqrt(25 / 4)
    got = oracle.norm_rotate(x, torch.ones(4), 0.0, torch.tensor([1]), table, True)
    assert torch.allclose(got[0, 0], torch.tensor([0.0, 4 * inv, 3 * inv, 0.0], dtype=torch.float64))
    got = oracle.norm_rotate(x, torch.ones(4), 0.0, torch.tensor([1]), table, False)
    assert torch.allclose(got[0, 0], torch.tensor([-4 * inv, 3 * inv, 0.0, 0.0], dtype=torch.float64))
