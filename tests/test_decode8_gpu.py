"""Decode over 8-bit pages against the formula in 64 bits on the values the codes stand for; bounds in
paged8_util."""

import numpy as np
import pytest
import torch  # (before the library is loaded: both use one HIP runtime)

import sca_amd
from attn_util import DTYPE_ID, decode_params, quantize, to_float
from paged8_util import DIMS, Device, attend64, check, download, hold8, pool, scale_of, sequence
from sca_amd import hip as H
from sca_amd import host as C

pytestmark = pytest.mark.gpu


def run(pl, qb, Hq, splits, slot_waves=0, pass_lens=True, longest_first=True, dev=None):
    dev = dev or Device(pl)
    S, D, Hkv, bs, dtype = len(pl["lens"]), pl["D"], pl["Hkv"], pl["bs"], pl["dtype"]
    dq = H.DeviceBuffer.from_array(qb)
    dl = H.DeviceBuffer.from_array(np.asarray(pl["lens"], np.int32))
    dout = H.DeviceBuffer.from_array(np.full(S * Hq * D, 0x7E7E, np.uint16))
    # scratch full of NaN: what a split leaves out must not be read
    n = sca_amd.hip_lib().sca_hip_decode_partial_elements(S, Hq, splits, D)
    parts = H.DeviceBuffer.from_array(np.full(n, np.nan, np.float32))
    order = H.DeviceBuffer(8 * S)
    p = H.Decode8Params()
    p.base = decode_params(dq, dev.k, dev.v, dout, parts, B=S, Hq=Hq, Hkv=Hkv, Skv=pl["table"].shape[1] * bs,
                           D=D, splits=splits, dtype=dtype, k_strides=(0, D, Hkv * D))
    b = p.base
    b.page_table, b.block_size = dev.table.ptr, bs
    b.max_blocks_per_seq, b.num_kv_blocks = pl["table"].shape[1], pl["nb"]
    b.seq_lens = dl.ptr if pass_lens else None
    b.batch_order = order.ptr if longest_first else None
    b.slot_waves = slot_waves
    p.k_exp, p.v_exp = dev.k_exp.ptr, dev.v_exp.ptr
    H.decode8_paged(p)
    sca_amd.synchronize()
    return download(dout, dtype, (S, Hq, D))


def expect(pl, qd, Hq, lens=None):
    parts = [attend64(qd[s].reshape(1, Hq, pl["D"]), *sequence(pl, s, None if lens is None else lens[s]),
                      False, scale_of(pl["D"])) for s in range(len(pl["lens"]))]
    return [np.concatenate(x) for x in zip(*parts)]


def case(lens, bs, Hq, Hkv, D, dtype, seed, runs, mutate=None, **kw):
    pl = pool(lens, bs, Hkv, D, dtype, seed, True)
    if mutate:
        mutate(pl)
    rng = np.random.default_rng(seed + 1)
    qb, qd = quantize(rng.standard_normal((len(lens), Hq, D)).astype(np.float32), dtype)
    out, _, A, err = expect(pl, qd, Hq)
    for splits, waves in runs:
        tag = f"decode8 {dtype} lens={lens[:4]} bs={bs} Hq={Hq} Hkv={Hkv} D={D} splits={splits} waves={waves}"
        print(tag, flush=True)
        got = run(pl, qb, Hq, splits, waves, **kw)
        check(got, out, A, err, dtype, max(lens), tag)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D", DIMS)
def test_every_head_dim(hip, D, dtype):
    case([1, 31, 33, 500, 0, 64], 16, 8, 2, D, dtype, 1000 + D, [(1, 1), (1, 4), (3, 1), (4, 4)])


@pytest.mark.parametrize("bs", [8, 16, 32, 64])
def test_every_page_size(hip, bs):
    case([257, 5, bs, bs + 1], bs, 8, 8, 128, "bf16", 1100 + bs, [(2, 1), (3, 4)])


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 3), (7, 1), (28, 4), (16, 1), (17, 1), (40, 2), (6, 3)])
def test_groups(hip, Hq, Hkv):
    case([129, 40], 16, Hq, Hkv, 64, "f16", 1200 + Hq, [(1, 1), (2, 4)])
    case([129, 40], 16, Hq, Hkv, 96, "bf16", 1250 + Hq, [(2, 1), (1, 4)])


def test_ragged_batches_ranked_in_the_kernel_and_through_scratch(hip):
    rng = np.random.default_rng(1300)
    lens = rng.integers(0, 90, 300).tolist()
    case(lens, 16, 4, 2, 64, "f16", 1301, [(1, 1), (2, 4)])
    case(lens, 16, 4, 2, 64, "f16", 1302, [(2, 1)], longest_first=False)
    case(rng.integers(1, 2500, 12).tolist(), 16, 16, 4, 128, "bf16", 1303, [(6, 4), (1, 1)])


def test_without_seq_lens_every_mapped_page_counts(hip):
    pl = pool([40], 16, 2, 64, "f16", 1400, True)
    qb, qd = quantize(np.random.default_rng(1401).standard_normal((1, 4, 64)).astype(np.float32), "f16")
    full = pl["table"].shape[1] * 16
    out, _, A, err = expect(pl, qd, 4, [full])
    for splits, waves in ((1, 1), (3, 4)):
        check(run(pl, qb, 4, splits, waves, pass_lens=False), out, A, err, "f16", full, "no lens")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("bs,D", [(8, 64), (16, 128), (64, 96)])
def test_unmapped_pages_and_nan_outside_the_sequences(hip, bs, D, dtype):
    def mutate(pl):
        pl["table"][1, 1] = -1
        pl["table"][1, 2] = pl["nb"] + 7
        used = np.zeros((pl["nb"], bs), bool)
        for s, n in enumerate(pl["lens"]):
            for t in range(n):
                page = pl["table"][s, t // bs]
                if 0 <= page < pl["nb"]:
                    used[page, t % bs] = True
        for name in "kv":
            pl[name][~used] = 0x7F
            pl[name + "_exp"].transpose(0, 2, 1)[~used] = 0xFF
    case([37, 5 * bs + 3, 1, 100], bs, 8, 2, D, dtype, 1500 + bs, [(1, 1), (3, 1), (1, 4), (3, 4)], mutate)


@pytest.mark.parametrize("waves", [1, 4])
def test_a_row_of_unmapped_pages_gives_zeros_and_nan_stays_nan(hip, waves):
    pl = pool([50, 50, 20], 16, 2, 64, "bf16", 1600, True)
    pl["table"][0, :] = -1
    page = pl["table"][2, 0]
    pl["k"][page, 3, 1, 0] = 0x7F  # a NaN key of KV head 1
    qb, qd = quantize(np.ones((3, 4, 64), np.float32), "bf16")
    for splits in (1, 2):
        got = run(pl, qb, 4, splits, waves)
        assert (got[0] == 0).all() and np.isfinite(got[1]).all()
        assert np.isfinite(got[2, :2]).all() and np.isnan(got[2, 2:]).all()
    pl["k"][pl["table"][2, :2]] = 0x7F  # nothing but NaN
    for splits in (1, 2):
        assert np.isnan(run(pl, qb, 4, splits, waves)[2]).all()


@pytest.mark.parametrize("dtype,magnitude", [("f16", 2.0 ** 12), ("f16", 2.0 ** -18), ("bf16", 2.0 ** 60),
                                             ("bf16", 2.0 ** -90)])
def test_values_at_the_ends_of_the_types_range(hip, dtype, magnitude):
    """V far from 1 (K and q scaled against each other so that the scores are ordinary)."""
    pl = pool([200], 16, 2, 128, dtype, 1700, True)
    for name, m in (("k", 2.0 ** (6 if magnitude > 1 else -6)), ("v", magnitude)):
        _, deq = quantize((pl[name + "_val"] * m).astype(np.float32), dtype)
        vals, e = hold8(deq, dtype)
        from paged8_util import codes_of
        pl[name], pl[name + "_exp"], pl[name + "_val"] = codes_of(vals, e), np.ascontiguousarray(e.transpose(0, 2, 1)), vals
    q = np.random.default_rng(1701).standard_normal((1, 4, 128)) * 2.0 ** (-6 if magnitude > 1 else 6)
    qb, qd = quantize(q.astype(np.float32), dtype)
    out, _, A, err = expect(pl, qd, 4)
    for splits, waves in ((1, 1), (2, 4)):
        check(run(pl, qb, 4, splits, waves), out, A, err, dtype, 200, f"magnitude {magnitude}")


def test_many_small_weights_beside_a_dominant_key_count_in_fp16(hip):
    """One key with a score 22 (in e) above 8,000 others whose V it does not share: their weights, below
    fp16's smallest number, still make up their share of the output."""
    L, D = 8192, 64
    pl = pool([L], 16, 1, D, "f16", 1800, True)
    k = np.zeros_like(pl["k_val"])
    v = np.ones_like(pl["v_val"])
    page, off = pl["table"][0, 5], 3
    k[page, off, 0, 0] = 32.0
    v[page, off, 0] = 0.0
    from paged8_util import codes_of
    for name, x in (("k", k), ("v", v)):
        vals, e = hold8(x, "f16")
        pl[name], pl[name + "_exp"], pl[name + "_val"] = codes_of(vals, e), np.ascontiguousarray(e.transpose(0, 2, 1)), vals
    q = np.zeros((1, 1, D), np.float32)
    q[..., 0] = 22.0 / 32.0 * 8.0
    qb, qd = quantize(q, "f16")
    out, _, A, err = expect(pl, qd, 1)
    assert 1e-6 < out[0, 0, 0] < 1e-5
    for splits, waves in ((1, 1), (1, 4), (3, 1)):
        check(run(pl, qb, 1, splits, waves), out, A, err, "f16", 1, "small weights")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D,bs,Hq,Hkv", [(128, 16, 32, 8), (64, 32, 8, 8), (96, 8, 12, 4), (256, 16, 16, 2)])
def test_serving_steps_through_the_host_api(hip, dtype, D, bs, Hq, Hkv):
    """Prompts appended, then steps of one token a sequence: written in 8 bits, attended at once, with
    the cache's plan and with given splits, on a stream of the caller's too."""
    rng = np.random.default_rng(1900 + D)
    lens = [3, 200, 1500]
    cache = C.PagedKVCache(C.KVCacheConfig(num_layers=1, num_kv_heads=Hkv, head_dim=D, block_size=bs,
                                           num_blocks=sum(-(-(n + 2) // bs) for n in lens), max_num_seqs=3,
                                           dtype=dtype, storage="e4m3"))
    vals = {}
    def make(n):
        out = []
        for _ in range(2):
            b, d = quantize(rng.standard_normal((n, Hkv, D)).astype(np.float32), dtype)
            out.append((b, hold8(d, dtype)[0]))
        return out
    for s, n in enumerate(lens):
        (kb, kv), (vb, vv) = make(n)
        cache.append_tokens(s, 0, C.Tensor.from_numpy(kb, dtype), C.Tensor.from_numpy(vb, dtype))
        vals[s] = [kv, vv]
    stream = torch.cuda.Stream()
    for step, (given, st) in enumerate(((0, None), (3, stream.cuda_stream))):
        (kb, kv), (vb, vv) = make(3)
        cache.append_batch([0, 1, 2], 0, C.Tensor.from_numpy(kb, dtype), C.Tensor.from_numpy(vb, dtype), st)
        cache.sync_page_table(st)
        for s in range(3):
            vals[s] = [np.concatenate([vals[s][0], kv[s:s + 1]]), np.concatenate([vals[s][1], vv[s:s + 1]])]
        qb, qd = quantize(rng.standard_normal((3, Hq, 1, D)).astype(np.float32), dtype)
        seq_lens = H.DeviceBuffer.from_array(np.array([cache.seq_length(s) for s in range(3)], np.int32))
        r = C.paged_attention(C.Tensor.from_numpy(qb, dtype), cache,
                              {"seq_lens": seq_lens.ptr, "num_seqs": 3, "block_size": bs},
                              C.AttentionConfig(num_splits=given, stream=st))
        sca_amd.synchronize()
        assert "8-bit" in r.stats["note"]
        got = to_float(r.out.numpy(), dtype).reshape(3, Hq, D).astype(np.float64)
        for s in range(3):
            n = vals[s][0].shape[0]
            out, _, A, err = attend64(qd[s].reshape(1, Hq, D), *vals[s], np.ones(n, bool), False, scale_of(D))
            check(got[s:s + 1], out, A, err, dtype, n, f"step {step} sequence {s}")
    with pytest.raises(C.ScaError, match="8-bit cache"):
        C.paged_attention(C.Tensor.from_numpy(qb, dtype), cache, {"num_seqs": 3, "block_size": 2 * bs})


def test_a_captured_step_replays(hip):
    """A decode captured on one stream replays with what the pages hold then, eager calls between."""
    D, Hkv, Hq, bs, n = 128, 2, 8, 16, 700
    cache = C.PagedKVCache(C.KVCacheConfig(num_kv_heads=Hkv, head_dim=D, block_size=bs, num_blocks=50,
                                           max_num_seqs=1, dtype="bf16", storage="e4m3"))
    gen = torch.Generator(device="cuda").manual_seed(5)
    def wrap(t):
        dims = (C.c_i64 * t.dim())(*t.shape)
        return C.Tensor(C.host_lib().sca_tensor_wrap(t.data_ptr(), dims, t.dim(), C.DTYPES["bf16"], C.GPU), "bf16")
    def rand(*shape):
        return torch.randn(shape, generator=gen, device="cuda").to(torch.bfloat16)
    k, v, q = rand(n, Hkv, D), rand(n, Hkv, D), rand(1, Hq, D)
    cache.append_tokens(0, 0, wrap(k), wrap(v))
    cache.sync_page_table()
    out = torch.zeros(1, Hq, D, dtype=torch.bfloat16, device="cuda")
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    parts = torch.zeros(4 * Hq * (2 + D), dtype=torch.float32, device="cuda")
    p = H.Decode8Params()
    b = p.base
    b.q, b.out = q.data_ptr(), out.data_ptr()
    b.k, b.v = cache.layer_ptrs(0)
    p.k_exp, p.v_exp = cache.layer_exponent_ptrs(0)
    b.partial_m = parts.data_ptr()
    b.partial_l = b.partial_m + 4 * Hq * 4
    b.partial_o = b.partial_l + 4 * Hq * 4
    b.batch, b.num_heads, b.num_kv_heads, b.seq_kv, b.head_dim, b.num_splits = 1, Hq, Hkv, n, D, 4
    b.q_sb, b.q_sh, b.o_sb, b.o_sh = Hq * D, D, Hq * D, D
    b.k_sh, b.k_ss, b.v_sh, b.v_ss = D, Hkv * D, D, Hkv * D
    b.scale, b.dtype = scale_of(D), DTYPE_ID["bf16"]
    b.page_table, b.block_size, b.max_blocks_per_seq, b.num_kv_blocks = cache.page_table_device_ptr, bs, 50, 50
    b.seq_lens = lens.data_ptr()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        H.decode8_paged(p, torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        q.copy_(rand(1, Hq, D))
        lens.fill_(n - 100 * i)
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        out.zero_()
        H.decode8_paged(p, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(replayed, out) and replayed.abs().sum() > 0
