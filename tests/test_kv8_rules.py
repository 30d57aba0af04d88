"""Refusals and sizes of 8-bit storage, of the decode over it and of ragged paged attention (no GPU)."""

import ctypes

import numpy as np
import pytest

from paged8_util import codes_of, e4m3_values, hold8
from sca_amd import hip as H
from sca_amd import host as C

P = 1 << 20  # an aligned address that nothing reads


def kv_shape(nb=4, bs=16, Hkv=2, D=64):
    s = H.KvShape()
    s.num_blocks, s.block_size, s.num_kv_heads, s.head_dim = nb, bs, Hkv, D
    return s


def test_the_oracle_holds_values_as_defined():
    x = np.array([[448.0, 449.0, 0.4375, -3.25], [1.0, 17 / 16, 19 / 16, 2.0 ** -20],
                  [896.0, -900.0, 0.0, 1.0]])
    vals, e = hold8(x, "bf16")
    assert e.tolist() == [127 + 1, 127 - 8, 127 + 2]
    # 449 needs twice the unit; ties go to even codes
    assert vals[0, 1] == 448.0 and vals[1, 1] == 1.0 and vals[1, 2] == 1.25 and vals[1, 3] == 0.0
    assert vals[2, 1] == -896.0
    codes = codes_of(vals, e)
    back = e4m3_values()[codes] * (2.0 ** (e.astype(float) - 127))[:, None]
    assert np.array_equal(back, vals)


def test_config_rules_and_budget():
    base = dict(num_layers=3, num_kv_heads=4, head_dim=96, block_size=16, num_blocks=10)
    same = C.kv_cache_bytes(C.KVCacheConfig(**base, dtype="bf16"))
    held = C.kv_cache_bytes(C.KVCacheConfig(**base, dtype="bf16", storage="e4m3"))
    assert same == 2 * 3 * 10 * 16 * 4 * 192 and held == 2 * 3 * 10 * 16 * 4 * 97
    assert C.max_blocks_for_budget(C.KVCacheConfig(**base, dtype="bf16", storage="e4m3"), held) == 10
    assert C.max_blocks_for_budget(C.KVCacheConfig(**base, dtype="bf16", storage="e4m3"), held - 1) == 9
    for change, text in ((dict(dtype="f32"), "float32"), (dict(block_size=1), "8-bit"),
                         (dict(storage=7), "storage=7"), (dict(storage=-1), "storage=-1")):
        with pytest.raises(C.ScaError, match=text):
            C.kv_cache_bytes(C.KVCacheConfig(**{**base, "dtype": "bf16", "storage": "e4m3", **change}))


def test_data_movement_refusals():
    lib = H.hip_lib()
    layer = H.Kv8Layer(P, P, P, P)

    def append(layer=layer, k=P, v=P, slots=P, n=1, shape=kv_shape(), dtype=H.DTYPE_F16):
        return lib.sca_hip_kv8_append(ctypes.byref(layer) if layer else None, k, v, slots, n,
                                      ctypes.byref(shape) if shape else None, dtype, None)

    def gather(codes=P, exps=P, ids=P, n=1, out=P, shape=kv_shape(), dtype=H.DTYPE_F16):
        return lib.sca_hip_kv8_gather(codes, exps, ids, n, out, ctypes.byref(shape) if shape else None,
                                      dtype, None)

    def reset(layer=layer, ids=P, n=1, shape=kv_shape()):
        return lib.sca_hip_kv8_reset_blocks(ctypes.byref(layer) if layer else None, ids, n,
                                            ctypes.byref(shape) if shape else None, None)

    for call in (append, gather, reset):
        assert call(shape=None) == 2005
        assert call(n=0) == 0
        for bad, code in ((kv_shape(nb=0), 2005), (kv_shape(bs=12), 2005), (kv_shape(bs=1), 2005),
                          (kv_shape(D=48), 2001), (kv_shape(D=224), 2001), (kv_shape(D=288), 2001),
                          (kv_shape(Hkv=70000), 2005), (kv_shape(nb=1 << 28), 2005),
                          (kv_shape(bs=1 << 30), 2005)):
            assert call(shape=bad) == code
    for call in (append, gather):
        assert call(dtype=H.DTYPE_F32) == 2002 and call(dtype=9) == 2002
    assert append(layer=None) == 2005 and append(k=None) == 2005 and append(slots=None) == 2005
    assert append(layer=H.Kv8Layer(P, P, P, None)) == 2005
    assert append(layer=H.Kv8Layer(P + 8, P, P, P)) == 2004
    assert append(layer=H.Kv8Layer(P, P, P + 4, P)) == 2004
    assert append(v=P + 8) == 2004
    assert reset(layer=None) == 2005 and reset(ids=None) == 2005
    assert gather(codes=None) == 2005 and gather(exps=None) == 2005 and gather(out=P + 8) == 2004


def decode_params(**change):
    p = H.Decode8Params()
    b = p.base
    b.q = b.k = b.v = b.out = P
    p.k_exp = p.v_exp = P
    b.batch, b.num_heads, b.num_kv_heads, b.seq_kv, b.head_dim, b.num_splits = 2, 8, 2, 64, 64, 1
    b.q_sb, b.q_sh, b.o_sb, b.o_sh = 512, 64, 512, 64
    b.k_sh = b.v_sh = 64
    b.k_ss = b.v_ss = 128
    b.scale, b.dtype = 0.125, H.DTYPE_F16
    b.page_table, b.block_size, b.max_blocks_per_seq, b.num_kv_blocks = P, 16, 4, 8
    for name, value in change.items():
        setattr(p if name.endswith("_exp") else b, name, value)
    return p


@pytest.mark.parametrize("change,code", [
    (dict(q=None), 2005), (dict(k_exp=None), 2005), (dict(v_exp=None), 2005), (dict(page_table=None), 2005),
    (dict(num_splits=0), 2005), (dict(num_splits=70000), 2005), (dict(num_splits=2), 2008),
    (dict(batch=0), 2005), (dict(batch=70000), 2005), (dict(num_heads=7), 2005), (dict(seq_kv=-1), 2005),
    (dict(dtype=H.DTYPE_F32), 2002), (dict(block_size=4), 2005), (dict(block_size=24), 2005),
    (dict(num_kv_blocks=1 << 28), 2005), (dict(max_blocks_per_seq=0), 2005), (dict(k=P + 8), 2004),
    (dict(k_ss=120), 2004), (dict(v_sh=8), 2004), (dict(q_sh=60), 2004), (dict(slot_waves=2), 2005),
    (dict(batch_order=P + 4), 2004), (dict(head_dim=80), 2001)])
def test_decode_refusals(change, code):
    assert H.hip_lib().sca_hip_decode8_paged(ctypes.byref(decode_params(**change)), None) == code
    assert H.hip_lib().sca_hip_decode8_paged(None, None) == 2005


class Varlen:
    def __init__(self, cu=(0, 3, 4), lens=(20, 9), rows=None, **change):
        self.cu = np.asarray(cu, np.int32)
        self.lens = np.asarray(lens, np.int32)
        self.rows = None if rows is None else np.asarray(rows, np.int32)
        p = self.p = H.PagedVarlenParams()
        p.q = p.k = p.v = p.out = p.page_table = P
        p.cu_seqlens_q, p.kv_lens = self.cu.ctypes.data, self.lens.ctypes.data
        p.table_rows = None if rows is None else self.rows.ctypes.data
        p.num_seqs, p.num_heads, p.num_kv_heads, p.head_dim = len(self.lens), 8, 2, 64
        p.block_size, p.max_blocks_per_seq, p.num_kv_blocks = 16, 4, 8
        p.q_ss = p.o_ss = 512
        p.q_sh = p.o_sh = p.k_sh = p.v_sh = 64
        p.k_ss = p.v_ss = 128
        p.scale, p.causal, p.dtype = 0.125, 1, H.DTYPE_BF16
        for name, value in change.items():
            setattr(p, name, value)


@pytest.mark.parametrize("args,code", [
    (dict(q=None), 2005), (dict(out=None), 2005), (dict(page_table=None), 2005), (dict(k_exp=P), 2005),
    (dict(cu_seqlens_q=None), 2005), (dict(kv_lens=None), 2005), (dict(num_seqs=0), 2005),
    (dict(num_heads=7), 2005), (dict(num_heads=70000), 2005), (dict(head_dim=48), 2001),
    (dict(head_dim=224), 2001), (dict(dtype=H.DTYPE_F32), 2002), (dict(scale=0.0), 2005),
    (dict(scale=float("nan")), 2005), (dict(scale=float("inf")), 2005), (dict(block_size=24), 2005),
    (dict(block_size=0), 2005), (dict(num_kv_blocks=1 << 28), 2005), (dict(max_blocks_per_seq=0), 2005),
    (dict(block_size=4, k_exp=P, v_exp=P), 2005), (dict(k_ss=120, k_exp=P, v_exp=P), 2004),
    (dict(q_ss=500), 2004), (dict(k=P + 8), 2004), (dict(cu=(0, 3, 2)), 2005), (dict(cu=(-1, 3, 4)), 2005),
    (dict(lens=(20, -1)), 2005), (dict(rows=(0, -1)), 2005), (dict(lens=(20, 0x7fffffff)), 2006),
    (dict(cu=(0, 3, 0x7fffff00)), 2006)])
def test_varlen_refusals(args, code):
    v = Varlen(**args)
    assert H.hip_lib().sca_hip_paged_varlen(ctypes.byref(v.p), None, 0, None) == code
    pointers = {"q", "out", "page_table", "k"} | ({"k_exp"} if args == dict(k_exp=P) else set())
    if not set(args) & pointers:
        assert H.hip_lib().sca_hip_paged_varlen_bytes(ctypes.byref(v.p)) == 0


def test_varlen_refuses_null_params_and_unaligned_scratch():
    lib = H.hip_lib()
    assert lib.sca_hip_paged_varlen(None, None, 0, None) == 2005
    assert lib.sca_hip_paged_varlen_bytes(None) == 0
    assert lib.sca_hip_paged_varlen(ctypes.byref(Varlen().p), P + 4, 1 << 20, None) == 2004


def test_varlen_scratch_is_bounded_and_only_where_keys_are_split():
    lib = H.hip_lib()
    few = Varlen(cu=(0, 4), lens=(30000,))
    want = lib.sca_hip_paged_varlen_bytes(ctypes.byref(few.p))
    assert 0 < want <= 64 << 20 and want % (4 * (64 + 2)) == 0
    assert lib.sca_hip_paged_varlen_bytes(ctypes.byref(Varlen(cu=(0, 4), lens=(200,)).p)) == 0
    # many sequences fill the GPU by themselves
    n = 2000
    many = Varlen(cu=np.arange(n + 1), lens=np.full(n, 4000))
    assert lib.sca_hip_paged_varlen_bytes(ctypes.byref(many.p)) == 0
    # long rows: the bound holds
    wide = Varlen(cu=(0, 20000), lens=(400000,), num_heads=64, num_kv_heads=1)
    assert lib.sca_hip_paged_varlen_bytes(ctypes.byref(wide.p)) <= 64 << 20
