"""Ragged chunks of new tokens over paged KV, 16-bit and 8-bit, against the formula in 64 bits; bounds
in paged8_util."""

import numpy as np
import pytest
import torch  # (before the library is loaded: both use one HIP runtime)

import sca_amd
from attn_util import DTYPE_ID, quantize, to_float
from paged8_util import DIMS, Device, attend64, check, check_lse, codes_of, download, hold8, pool, scale_of, \
    sequence
from sca_amd import hip as H
from sca_amd import host as C

pytestmark = pytest.mark.gpu
STORED = [False, True]


def params(pl, dev, new, Hq, dq, dout, dlse, causal, keep, lens=None, rows=None, first=0, scale=None):
    D, Hkv, bs, dtype = pl["D"], pl["Hkv"], pl["bs"], pl["dtype"]
    cu = np.concatenate([[first], first + np.cumsum(new)]).astype(np.int32)
    kv = np.asarray(pl["lens"] if lens is None else lens, np.int32)
    keep += [cu, kv]
    p = H.PagedVarlenParams()
    p.q, p.out = dq.ptr, dout.ptr
    p.lse = dlse.ptr if dlse else None
    p.k, p.v, p.page_table = dev.k.ptr, dev.v.ptr, dev.table.ptr
    if pl["held8"]:
        p.k_exp, p.v_exp = dev.k_exp.ptr, dev.v_exp.ptr
    p.cu_seqlens_q, p.kv_lens = cu.ctypes.data, kv.ctypes.data
    if rows is not None:
        r = np.asarray(rows, np.int32)
        keep.append(r)
        p.table_rows = r.ctypes.data
    p.num_seqs, p.num_heads, p.num_kv_heads, p.head_dim = len(new), Hq, Hkv, D
    p.block_size, p.max_blocks_per_seq, p.num_kv_blocks = bs, pl["table"].shape[1], pl["nb"]
    p.q_ss = p.o_ss = Hq * D
    p.q_sh = p.o_sh = p.k_sh = p.v_sh = D
    p.k_ss = p.v_ss = Hkv * D
    p.scale = scale or scale_of(D)
    p.causal, p.dtype = int(causal), DTYPE_ID[dtype]
    return p


def run(pl, new, qb, Hq, causal, scratch, lse=True, dev=None, tail=2, **kw):
    """(out, lse) with `tail` rows behind the last sequence, which must stay as they were."""
    dev = dev or Device(pl)
    D, dtype = pl["D"], pl["dtype"]
    total = kw.get("first", 0) + sum(new)
    dq = H.DeviceBuffer.from_array(qb)
    dout = H.DeviceBuffer.from_array(np.full((total + tail) * Hq * D, 0x2A2A, np.uint16))
    dlse = H.DeviceBuffer.from_array(np.full((total + tail) * Hq, 77.0, np.float32)) if lse else None
    keep = []
    p = params(pl, dev, new, Hq, dq, dout, dlse, causal, keep, **kw)
    want = H.paged_varlen_bytes(p) if scratch is True else int(scratch)
    buf = H.DeviceBuffer.from_array(np.full(want // 4 + 1, np.nan, np.float32)) if want else None
    H.paged_varlen(p, buf.ptr if buf else None, want)
    sca_amd.synchronize()
    raw = dout.download(np.uint16).reshape(total + tail, Hq, D)
    assert (raw[total:] == 0x2A2A).all() and (raw[:kw.get("first", 0)] == 0x2A2A).all()
    out = to_float(raw[kw.get("first", 0):total], dtype).astype(np.float64).reshape(sum(new), Hq, D)
    l = None
    if lse:
        l = dlse.download(np.float32).reshape(total + tail, Hq)
        assert (l[total:] == 77.0).all()
        l = l[kw.get("first", 0):total].astype(np.float64)
    return out, l, want


def expect(pl, new, qd, causal, lens=None, rows=None, scale=None):
    parts, at = [], 0
    for s, n in enumerate(new):
        row = s if rows is None else rows[s]
        k, v, ok = sequence(pl, row, (pl["lens"] if lens is None else lens)[s])
        parts.append(attend64(qd[at:at + n], k, v, ok, causal, scale or scale_of(pl["D"])))
        at += n
    return [np.concatenate(x) for x in zip(*parts)]


def case(lens, new, bs, Hq, Hkv, D, dtype, held8, seed, causal=True, scratches=(0, True), mutate=None, std=1.0,
         use_lens=None, **kw):
    pl = pool(lens, bs, Hkv, D, dtype, seed, held8, std=std)
    if mutate:
        mutate(pl)
    rng = np.random.default_rng(seed + 1)
    qb, qd = quantize((rng.standard_normal((kw.get("first", 0) + sum(new), Hq, D)) * std).astype(np.float32), dtype)
    out, lse, A, err = expect(pl, new, qd[kw.get("first", 0):], causal, use_lens, kw.get("rows"))
    dev = Device(pl)
    for scratch in scratches:
        tag = (f"varlen {dtype} held8={held8} lens={list(lens)[:5]} new={list(new)[:5]} bs={bs} Hq={Hq} Hkv={Hkv} "
               f"D={D} causal={causal} scratch={scratch}")
        print(tag, flush=True)
        got, gl, used = run(pl, new, qb, Hq, causal, scratch, dev=dev, lens=use_lens, **kw)
        check(got, out, A, err, dtype, max(list(lens) + [1]), tag)
        check_lse(gl, lse, err, tag)
    return used


@pytest.mark.parametrize("held8", STORED)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D", DIMS)
def test_every_head_dim(hip, D, dtype, held8):
    case([1, 130, 64, 300, 0, 37], [1, 70, 64, 3, 0, 1], 16, 8, 2, D, dtype, held8, 2000 + D)
    case([90, 200], [40, 7], 16, 4, 2, D, dtype, held8, 2050 + D, causal=False)


@pytest.mark.parametrize("held8,bs", [(False, 1), (False, 2), (False, 8), (False, 16), (False, 64), (True, 8),
                                      (True, 16), (True, 32), (True, 64), (False, 128)])
def test_every_page_size(hip, bs, held8):
    case([257, 5, bs, bs + 1], [130, 5, 1, 2], bs, 6, 2, 64, "bf16", held8, 2100 + bs)
    case([257, 5, bs, bs + 1], [130, 5, 1, 2], bs, 2, 2, 192, "f16", held8, 2150 + bs)


@pytest.mark.parametrize("held8", STORED)
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 3), (7, 1), (28, 4), (48, 1), (130, 1), (6, 3), (16, 16)])
def test_groups(hip, Hq, Hkv, held8):
    case([129, 40, 300], [50, 1, 9], 16, Hq, Hkv, 64, "f16", held8, 2200 + Hq)
    case([129, 40], [3, 33], 32, Hq, Hkv, 128, "bf16", held8, 2250 + Hq)


@pytest.mark.parametrize("held8", STORED)
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129])
def test_chunk_lengths_around_tiles(hip, n, held8):
    case([n, n + 1, n + 63, n + 64, n + 65], [n] * 5, 16, 2, 1, 128, "bf16", held8, 2300 + n)
    case([n + 100], [n], 16, 1, 1, 256, "f16", held8, 2350 + n, scratches=(0,))


@pytest.mark.parametrize("held8", STORED)
@pytest.mark.parametrize("D,dtype", [(64, "f16"), (96, "bf16"), (128, "bf16"), (128, "f16"), (256, "bf16")])
def test_keys_are_split_where_rows_are_few(hip, D, dtype, held8):
    used = case([5000, 2300], [3, 1], 16, 4, 2, D, dtype, held8, 2400 + D)
    assert used > 0
    # part of the scratch: fewer splits; a chunk whose first tiles see fewer keys than splits
    pl_bytes = used
    case([5000, 2300], [3, 1], 16, 4, 2, D, dtype, held8, 2400 + D, scratches=(pl_bytes // 3, 64))
    case([2100], [2100], 16, 1, 1, D, dtype, held8, 2450 + D)
    case([3000, 10, 3000], [5, 10, 2], 16, 4, 1, D, dtype, held8, 2470 + D, causal=False)


@pytest.mark.parametrize("held8", STORED)
def test_more_sequences_than_one_launch_lists(hip, held8):
    rng = np.random.default_rng(2500)
    lens = rng.integers(1, 120, 250)
    new = [int(rng.integers(0, n + 1)) if i % 3 else 1 for i, n in enumerate(lens)]
    case(lens.tolist(), new, 16, 4, 2, 64, "bf16", held8, 2501)
    lens = [2500] * 3 + [40] * 120
    case(lens, [1] * len(lens), 16, 2, 1, 32, "f16", held8, 2502)


@pytest.mark.parametrize("held8", STORED)
@pytest.mark.parametrize("D,bs", [(64, 8), (128, 16), (192, 32), (96, 64)])
def test_unmapped_pages_and_nan_outside_the_sequences(hip, D, bs, held8):
    def mutate(pl):
        pl["table"][1, 1] = -1
        pl["table"][1, 3] = pl["nb"] + 7
        used = np.zeros((pl["nb"], bs), bool)
        for s, n in enumerate(pl["lens"]):
            for t in range(n):
                page = pl["table"][s, t // bs]
                if 0 <= page < pl["nb"]:
                    used[page, t % bs] = True
        for name in "kv":
            if held8:
                pl[name][~used] = 0x7F
                pl[name + "_exp"].transpose(0, 2, 1)[~used] = 0xFF
            else:
                pl[name][~used] = 0x7FC0
    case([37, 7 * bs + 3, 1, 1000], [37, 5, 1, 9], bs, 8, 2, D, "bf16", held8, 2600 + bs, mutate=mutate)


@pytest.mark.parametrize("held8", STORED)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_rows_that_see_no_key(hip, D, held8):
    # more new tokens than keys; no keys at all; every page unmapped; a page table that ends early
    def mutate(pl):
        pl["table"][3, :] = -1
    case([5, 0, 70, 50], [9, 4, 70, 3], 16, 4, 2, D, "bf16", held8, 2700, mutate=mutate)
    case([5, 0, 70, 50], [9, 4, 70, 3], 16, 4, 2, D, "f16", held8, 2701, causal=False, mutate=mutate)
    pl = pool([40], 16, 2, D, "f16", 2702, held8)
    far = pl["table"].shape[1] * 16 + 200
    qb, qd = quantize(np.random.default_rng(1).standard_normal((3, 4, D)).astype(np.float32), "f16")
    out, lse, A, err = expect(pl, [3], qd, False, [far])
    got, gl, _ = run(pl, [3], qb, 4, False, 0, lens=[far])
    check(got, out, A, err, "f16", far, "short table")
    check_lse(gl, lse, err, "short table")


@pytest.mark.parametrize("held8", STORED)
@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 192, 256])
def test_tiles_of_rows_before_the_first_key(hip, D, held8):
    """More new tokens than keys by more than a tile of them."""
    case([16, 200, 0], [58, 430, 90], 16, 20, 1, D, "f16", held8, 2750 + D)
    case([3, 40], [300, 129], 16, 2, 2, D, "bf16", held8, 2760 + D)


@pytest.mark.parametrize("held8", STORED)
@pytest.mark.parametrize("D", [64, 128, 192])
def test_nan_keys_reach_their_rows_and_no_others(hip, D, held8):
    pl = pool([600, 600], 16, 2, D, "bf16", 2800, held8)
    page = pl["table"][0, 10]  # keys 160 .. 175
    nan = 0x7F if held8 else 0x7FC0
    pl["k"][page, 4, 1, 0] = nan
    new, Hq = [600, 4], 4
    qb, _ = quantize(np.random.default_rng(2801).standard_normal((604, Hq, D)).astype(np.float32), "bf16")
    for scratch in (0, True):
        out, lse, _ = run(pl, new, qb, Hq, True, scratch)
        bad = np.isnan(out).any(axis=2)
        want = np.zeros((604, Hq), bool)
        want[164:600, 2:] = True
        assert np.array_equal(bad, want) and np.array_equal(np.isnan(lse), want)
        assert np.array_equal(np.isnan(out).all(axis=2), want)
    # keys of nothing but NaN
    pl["k"][:] = nan
    out, lse, _ = run(pl, new, qb, Hq, False, True)
    assert np.isnan(out).all() and np.isnan(lse).all()


@pytest.mark.parametrize("held8", STORED)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_large_scores_and_growing_maxima(hip, dtype, held8):
    """Scores in the hundreds, growing along the keys, so that the running maximum moves often."""
    D, L = 64, 700
    pl = pool([L], 16, 1, D, dtype, 2900, held8)
    ramp = np.zeros_like(pl["k_val"])
    for t in range(L):
        ramp[pl["table"][0, t // 16], t % 16, 0, 0] = 0.1 * t
    k = pl["k_val"] + ramp
    _, deq = quantize(k.astype(np.float32), dtype)
    if held8:
        vals, e = hold8(deq, dtype)
        pl["k"], pl["k_exp"], pl["k_val"] = codes_of(vals, e), np.ascontiguousarray(e.transpose(0, 2, 1)), vals
    else:
        pl["k"], pl["k_val"] = quantize(k.astype(np.float32), dtype)[0], deq.astype(np.float64)
    q = np.random.default_rng(2901).standard_normal((40, 2, D))
    q[..., 0] = 30.0
    q[20:, :, 0] = -30.0
    qb, qd = quantize(q.astype(np.float32), dtype)
    out, lse, A, err = expect(pl, [40], qd, True)
    for scratch in (0, True):
        got, gl, _ = run(pl, [40], qb, 2, True, scratch)
        check(got, out, A, err, dtype, L, f"ramp scratch={scratch}")
        check_lse(gl, lse, err, "ramp")


@pytest.mark.parametrize("D", [32, 64, 128, 160, 192, 256])
def test_unmapped_pages_under_long_chunks(hip, D):
    """Holes at the first page, inside the steady part of the key loop, next to its end, and behind the first
    512 pages; with and without split keys."""
    for n, (L, holes) in enumerate([(400, (0,)), (1500, (0, 1, 17, 18, 50)), (1500, (93,)), (1500, (84,)), (9000, (540,))]):
        def mutate(pl):
            for i, h in enumerate(holes):
                pl["table"][0, h] = -1 if i % 2 == 0 else pl["nb"]
        case([L], [90], 16, 2, 2, D, "f16" if n % 2 else "bf16", False, 3300 + n, mutate=mutate)
        case([L], [90], 16, 1, 1, D, "bf16", False, 3320 + n, mutate=mutate, scratches=(True,), causal=False)


@pytest.mark.parametrize("D", [64, 128, 192, 256])
def test_unmapped_pages_of_eight_tokens_under_long_chunks(hip, D):
    for n, (L, holes) in enumerate([(300, (0,)), (1000, (1, 3, 33, 62, 100)), (1000, (124,)), (6000, (700, 749))]):
        def mutate(pl):
            for i, h in enumerate(holes):
                pl["table"][0, h] = -1 if i % 2 == 0 else pl["nb"]
        case([L], [70], 8, 2, 2, D, "f16" if n % 2 else "bf16", False, 3360 + n, mutate=mutate)
        case([L], [70], 8, 1, 1, D, "bf16", False, 3370 + n, mutate=mutate, scratches=(True,), causal=False)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D", [32, 64, 96])
def test_chunks_and_single_tokens_in_one_step(hip, D, dtype):
    lens = [2600, 1, 0, 3100, 700, 64, 1800, 5000, 65]
    new = [300, 1, 0, 1, 40, 64, 1, 2, 1]
    used = case(lens, new, 16, 8, 2, D, dtype, False, 3400 + D)
    assert used > 0
    case(lens, new, 16, 8, 2, D, dtype, False, 3400 + D, scratches=(used // 2, 4096))
    case(lens, new, 32, 3, 1, D, dtype, False, 3410 + D, causal=False)
    case([900, 900], [1, 200], 16, 16, 1, D, dtype, False, 3420 + D, first=2)


@pytest.mark.parametrize("D", [32, 64])
def test_nan_keys_of_a_single_token_beside_a_chunk(hip, D):
    pl = pool([600, 600, 50], 16, 2, D, "bf16", 3500, False)
    pl["k"][pl["table"][0, 10], 4, 1, 0] = 0x7FC0
    pl["v"][pl["table"][1, 0], 0, 0, 3] = 0x7FC0
    new, Hq = [1, 600, 1], 4
    qb, _ = quantize(np.random.default_rng(3501).standard_normal((602, Hq, D)).astype(np.float32), "bf16")
    for scratch in (0, True):
        out, lse, _ = run(pl, new, qb, Hq, True, scratch)
        want = np.zeros((602, Hq, D), bool)
        want[0, 2:] = True          # a key: every dim of the heads that read it
        want[1:601, :2, 3] = True   # a value: its own dim
        assert np.array_equal(np.isnan(out), want)
        assert np.array_equal(np.isnan(lse), want.all(axis=2))


def test_strides_offsets_rows_of_the_table_and_repeated_sequences(hip):
    case([300, 20, 100], [4, 30, 2], 16, 4, 2, 64, "f16", False, 3000, first=3, rows=[0, 2, 0],
         use_lens=[300, 100, 250])
    # head-major q and out, pages with a wider row
    D, Hq, Hkv, bs, T = 64, 4, 2, 16, 21
    pl = pool([90], bs, Hkv, D, "bf16", 3001, False)
    wide = np.zeros((pl["nb"], bs, Hkv + 1, D), np.uint16)
    wide_v = np.full((pl["nb"], bs, Hkv + 1, D), 0x7FC0, np.uint16)
    wide[:, :, :Hkv], wide_v[:, :, :Hkv] = pl["k"], pl["v"]
    dev = Device(pl)
    dev.k, dev.v = H.DeviceBuffer.from_array(wide), H.DeviceBuffer.from_array(wide_v)
    qb, qd = quantize(np.random.default_rng(3002).standard_normal((Hq, T, D)).astype(np.float32), "bf16")
    dq, dout = H.DeviceBuffer.from_array(qb), H.DeviceBuffer(Hq * T * D * 2)
    keep = []
    p = params(pl, dev, [T], Hq, dq, dout, None, True, keep)
    p.q_ss = p.o_ss = D
    p.q_sh = p.o_sh = T * D
    p.k_ss = p.v_ss = (Hkv + 1) * D
    H.paged_varlen(p)
    sca_amd.synchronize()
    got = download(dout, "bf16", (Hq, T, D)).transpose(1, 0, 2)
    out, _, A, err = expect(pl, [T], qd.transpose(1, 0, 2), True)
    check(got, out, A, err, "bf16", 90, "strided")


@pytest.mark.parametrize("held8", STORED)
def test_a_pool_past_four_gigabytes(hip, held8):
    """Pages whose byte offsets pass 2^32: the last pages of a pool of 4.3 GB of K (and of V)."""
    D, Hkv, bs = 128, 8, 64
    eb = 1 if held8 else 2
    nb = (1 << 32) // (bs * Hkv * D * eb) + 40
    small = pool([500], bs, Hkv, D, "bf16", 3100, held8)
    dev = Device(small)
    bufs = [torch.empty(nb * bs * Hkv * D * eb, dtype=torch.uint8, device="cuda") for _ in range(2)]
    exps = [torch.empty(nb * Hkv * bs, dtype=torch.uint8, device="cuda") for _ in range(2)]
    first = nb - small["nb"]
    for buf, e, name in zip(bufs, exps, "kv"):
        raw = torch.from_numpy(np.ascontiguousarray(small[name]).view(np.uint8).reshape(-1))
        buf[first * bs * Hkv * D * eb:].copy_(raw)
        if held8:
            e[first * Hkv * bs:].copy_(torch.from_numpy(small[name + "_exp"].reshape(-1)))
    class Ptr:
        def __init__(self, t):
            self.ptr = t.data_ptr()
    dev.k, dev.v, dev.k_exp, dev.v_exp = Ptr(bufs[0]), Ptr(bufs[1]), Ptr(exps[0]), Ptr(exps[1])
    table = np.where(small["table"] >= 0, small["table"] + first, -1).astype(np.int32)
    dev.table = H.DeviceBuffer.from_array(table)
    Hq, new = 16, [9]
    qb, qd = quantize(np.random.default_rng(3101).standard_normal((9, Hq, D)).astype(np.float32), "bf16")
    out, lse, A, err = expect(small, new, qd, True)
    big = dict(small, nb=nb)
    torch.cuda.synchronize()
    for scratch in (0, True):
        got, gl, _ = run(big, new, qb, Hq, True, scratch, dev=dev)
        check(got, out, A, err, "bf16", 500, "large pool")
        check_lse(gl, lse, err, "large pool")
    del bufs
    torch.cuda.empty_cache()


# ---- through the host API -----------------------------------------------------------------------------

class Served:
    """A cache and the 64-bit values it holds, grown by appends."""

    def __init__(self, storage, dtype, Hkv, D, bs, seqs, blocks, layers=1):
        self.dtype, self.Hkv, self.D = dtype, Hkv, D
        self.storage = storage
        self.cache = C.PagedKVCache(C.KVCacheConfig(num_layers=layers, num_kv_heads=Hkv, head_dim=D,
                                                    block_size=bs, num_blocks=blocks, max_num_seqs=seqs,
                                                    dtype=dtype, storage=storage))
        self.layers = layers
        self.held = {(s, l): [np.zeros((0, Hkv, D))] * 2 for s in range(seqs) for l in range(layers)}

    def grow(self, rng, s, n, stream=None):
        self.cache.reserve(s, n, stream)
        for l in range(self.layers):
            bits = []
            for i in range(2):
                b, d = quantize(rng.standard_normal((n, self.Hkv, self.D)).astype(np.float32), self.dtype)
                x = hold8(d, self.dtype)[0] if self.storage == "e4m3" else d.astype(np.float64)
                self.held[s, l][i:i + 1] = [np.concatenate([self.held[s, l][i], x])]
                bits.append(C.Tensor.from_numpy(b, self.dtype))
            self.cache.write_layer(l, *bits, stream)

    def expect(self, qd, new, ids, layer=0, causal=True, lens=None):
        parts, at = [], 0
        for i, (s, n) in enumerate(zip(ids, new)):
            k, v = self.held[s, layer]
            L = len(k) if lens is None else lens[i]
            parts.append(attend64(qd[at:at + n], k[:L], v[:L], np.ones(L, bool), causal, scale_of(self.D)))
            at += n
        return [np.concatenate(x) for x in zip(*parts)]


@pytest.mark.parametrize("storage", ["same", "e4m3"])
@pytest.mark.parametrize("dtype,D,bs,Hq,Hkv", [("bf16", 128, 16, 16, 4), ("f16", 64, 8, 4, 4), ("bf16", 96, 32, 6, 2),
                                               ("f16", 256, 16, 8, 1)])
def test_a_conversation_through_the_host_api(hip, storage, dtype, D, bs, Hq, Hkv):
    """Prompts in chunks, then mixed steps (single tokens beside a chunk), drafted tokens, two layers: the
    run that a serving loop makes, each call checked; the last step by decode too."""
    rng = np.random.default_rng(3200 + D)
    sv = Served(storage, dtype, Hkv, D, bs, 3, 200 if bs < 16 else 120, layers=2)
    for ids, new, causal in (([0], [150], True), ([0, 2], [77, 300], True), ([2, 0, 1], [1, 1, 40], True),
                             ([1, 0], [5, 5], True), ([0, 1, 2], [1, 1, 1], False)):
        for s, n in zip(ids, new):
            sv.grow(rng, s, n)
        sv.cache.sync_page_table()
        T = sum(new)
        for layer in range(2):
            qb, qd = quantize(rng.standard_normal((T, Hq, D)).astype(np.float32), dtype)
            q = C.Tensor.from_numpy(qb, dtype)
            cfg = C.AttentionConfig(causal=causal, return_lse=True,
                                    cu_seqlens_q=np.concatenate([[0], np.cumsum(new)]))
            r = C.paged_attention_varlen(q, sv.cache, {"num_seqs": len(ids), "seq_ids": ids, "layer": layer}, cfg)
            sca_amd.synchronize()
            out, lse, A, err = sv.expect(qd, new, ids, layer, causal)
            got = to_float(r.out.numpy(), dtype).reshape(T, Hq, D).astype(np.float64)
            tag = f"{storage} {dtype} ids={ids} new={new} layer={layer}"
            print(tag, flush=True)
            check(got, out, A, err, dtype, 600, tag)
            check_lse(r.lse.numpy().reshape(T, Hq).astype(np.float64), lse, err, tag)
            if new == [1, 1, 1]:
                lens = H.DeviceBuffer.from_array(np.array([sv.cache.seq_length(s) for s in ids], np.int32))
                d = C.paged_attention(C.Tensor.from_numpy(qb.reshape(3, Hq, 1, D), dtype), sv.cache,
                                      {"seq_lens": lens.ptr, "num_seqs": 3, "block_size": bs, "layer": layer})
                sca_amd.synchronize()
                check(to_float(d.out.numpy(), dtype).reshape(T, Hq, D).astype(np.float64), out, A, err, dtype,
                      600, tag + " decode")


@pytest.mark.parametrize("storage", ["same", "e4m3"])
def test_padding_limits_and_two_streams(hip, storage):
    rng = np.random.default_rng(3300)
    dtype, D, Hq, Hkv, bs = "bf16", 128, 8, 2, 16
    sv = Served(storage, dtype, Hkv, D, bs, 2, 400)
    sv.grow(rng, 0, 4000)
    sv.grow(rng, 1, 900)
    sv.cache.sync_page_table()
    new, pad = [6, 0], 5
    qb, qd = quantize(rng.standard_normal((sum(new) + pad, Hq, D)).astype(np.float32), dtype)
    q = C.Tensor.from_numpy(qb, dtype)
    out, lse, A, err = sv.expect(qd[:6], new, [0, 1])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    results = []
    for i in range(4):  # overlapping calls on two streams: their scratch must not mix
        cfg = C.AttentionConfig(causal=True, return_lse=True, cu_seqlens_q=[0, 6, 6],
                                num_splits=1 if i == 3 else 0, stream=streams[i % 2].cuda_stream)
        results.append(C.paged_attention_varlen(q, sv.cache, {"num_seqs": 2}, cfg))
    torch.cuda.synchronize()
    for i, r in enumerate(results):
        assert (r.stats["workspace_bytes"] > 0) == (i != 3)
        got = to_float(r.out.numpy(), dtype).reshape(11, Hq, D).astype(np.float64)
        check(got[:6], out, A, err, dtype, 4000, f"call {i}")
        assert (got[6:] == 0).all()
        l = r.lse.numpy().reshape(11, Hq).astype(np.float64)
        check_lse(l[:6], lse, err, f"call {i}")
        assert (l[6:] == 0).all()
    # shorter kv_lens than the cache's, and no new tokens at all
    r = C.paged_attention_varlen(q, sv.cache, {"num_seqs": 2, "kv_lens": [100, 7], "seq_ids": [1, 0]},
                                 C.AttentionConfig(causal=True, cu_seqlens_q=[0, 4, 11]))
    sca_amd.synchronize()
    out, _, A, err = sv.expect(qd, [4, 7], [1, 0], lens=[100, 7])
    check(to_float(r.out.numpy(), dtype).reshape(11, Hq, D).astype(np.float64), out, A, err, dtype, 100, "kv_lens")
    r = C.paged_attention_varlen(q, sv.cache, {"num_seqs": 1}, C.AttentionConfig(cu_seqlens_q=[0, 0]))
    sca_amd.synchronize()
    assert not r.out.numpy().any()


@pytest.mark.parametrize("storage", ["same", "e4m3"])
def test_a_captured_call_replays_with_its_own_lengths(hip, storage):
    """Two graphs of different calls (by the launcher, a scratch of its own each), replayed in turns with
    eager calls between; the plan travels in the launch."""
    rng = np.random.default_rng(3400)
    dtype, D, Hq, Hkv, bs = "bf16", 64, 8, 2, 16
    sv = Served(storage, dtype, Hkv, D, bs, 2, 400)
    sv.grow(rng, 0, 3000)
    sv.grow(rng, 1, 500)
    sv.cache.sync_page_table()
    sca_amd.synchronize()
    graphs = []
    for new, lens in (([4, 2], [3000, 500]), ([1, 60], [2500, 480])):
        T = sum(new)
        q = torch.randn(T, Hq, D, device="cuda").to(torch.bfloat16)
        out = torch.zeros(T, Hq, D, dtype=torch.bfloat16, device="cuda")
        p = H.PagedVarlenParams()
        cu, kv = np.concatenate([[0], np.cumsum(new)]).astype(np.int32), np.array(lens, np.int32)
        p.q, p.out = q.data_ptr(), out.data_ptr()
        p.k, p.v = sv.cache.layer_ptrs(0)
        if storage == "e4m3":
            p.k_exp, p.v_exp = sv.cache.layer_exponent_ptrs(0)
        p.page_table = sv.cache.page_table_device_ptr
        p.cu_seqlens_q, p.kv_lens = cu.ctypes.data, kv.ctypes.data
        p.num_seqs, p.num_heads, p.num_kv_heads, p.head_dim = 2, Hq, Hkv, D
        p.block_size, p.max_blocks_per_seq, p.num_kv_blocks = bs, 400, 400
        p.q_ss = p.o_ss = Hq * D
        p.q_sh = p.o_sh = p.k_sh = p.v_sh = D
        p.k_ss = p.v_ss = Hkv * D
        p.scale, p.causal, p.dtype = scale_of(D), 1, DTYPE_ID[dtype]
        n = H.paged_varlen_bytes(p)
        assert n > 0
        scratch = torch.full((n // 4 + 4,), float("nan"), device="cuda")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            H.paged_varlen(p, scratch.data_ptr(), n, torch.cuda.current_stream().cuda_stream)
        cu_eager, kv_eager = cu.copy(), kv.copy()
        cu[:] = 0  # the host arrays of a captured call are free again
        kv[:] = 1
        graphs.append((graph, p, q, out, scratch, n, cu, kv, cu_eager, kv_eager))
    for i in range(6):
        graph, p, q, out, scratch, n, cu, kv, cu_eager, kv_eager = graphs[i % 2]
        q.copy_(torch.randn(q.shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        out.zero_()
        p.cu_seqlens_q, p.kv_lens = cu_eager.ctypes.data, kv_eager.ctypes.data
        H.paged_varlen(p, scratch.data_ptr(), n, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(replayed, out) and replayed.abs().sum() > 0


def test_host_api_refusals(hip):
    sv = Served("same", "bf16", 2, 64, 16, 2, 20)
    rng = np.random.default_rng(3500)
    sv.grow(rng, 0, 30)
    sv.cache.sync_page_table()

    def call(shape=(4, 4, 64), dtype="bf16", params=None, cu=(0, 4), device=C.GPU, **cfg):
        q = C.Tensor.empty(shape, dtype, device)
        p = {"num_seqs": 1, **(params or {})}
        return C.paged_attention_varlen(q, sv.cache, p, C.AttentionConfig(
            cu_seqlens_q=None if cu is None else list(cu), **cfg))

    call()
    for kw, code in ((dict(shape=(4, 4, 1, 64)), 2005), (dict(dtype="f32"), 2002), (dict(dtype="f16"), 2002),
                     (dict(shape=(4, 4, 128)), 2005), (dict(shape=(4, 3, 64)), 2005),
                     (dict(shape=(4, 1, 64)), 2005), (dict(cu=None), 2005), (dict(cu=(1, 4)), 2005),
                     (dict(cu=(0, 5)), 2005), (dict(cu=(0, 3, 2), params={"num_seqs": 2}), 2005),
                     (dict(params={"layer": 1}), 2005), (dict(params={"layer": -1}), 2005),
                     (dict(params={"seq_ids": [2]}), 2005), (dict(params={"seq_ids": [-1]}), 2005),
                     (dict(params={"kv_lens": [-1]}), 2005), (dict(params={"num_seqs": 0}, cu=(0,)), 2005),
                     (dict(sliding_window=8), 2009), (dict(softcap=30.0), 2009),
                     (dict(params={"page_table": sv.cache.page_table_device_ptr}), 2005),
                     (dict(device=C.HOST), 2009), (dict(scale=float("inf")), 2005)):
        with pytest.raises(C.ScaError) as e:
            call(**kw)
        assert e.value.code == code, (kw, e.value)
    with pytest.raises(ValueError):
        call(params={"seq_ids": [0, 1]})
    sca_amd.synchronize()
