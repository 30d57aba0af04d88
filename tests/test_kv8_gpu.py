"""8-bit pages: what is written, read back and cleared, against the definition in 64 bits."""

import ctypes

import numpy as np
import pytest

import sca_amd
from attn_util import DTYPE_ID, quantize, to_float
from paged8_util import DIMS, LARGEST, codes_of, e4m3_values, hold8
from sca_amd import hip as H
from sca_amd import host as C

pytestmark = pytest.mark.gpu


def kv_shape(nb, bs, Hkv, D):
    s = H.KvShape()
    s.num_blocks, s.block_size, s.num_kv_heads, s.head_dim = nb, bs, Hkv, D
    return s


def rows_with_everything(rng, tokens, Hkv, D, dtype):
    """Rows of very different magnitude, with zeros, subnormals, values at rounding ties and limits."""
    x = rng.standard_normal((tokens, Hkv, D)) * 2.0 ** rng.integers(-8, 9, (tokens, Hkv, 1))
    big = 2.0 ** (15 if dtype == "f16" else 127)
    tiny = 2.0 ** (-24 if dtype == "f16" else -133)
    x = x.astype(np.float64)
    x[0] = 0.0
    if tokens > 1:
        x[1] = rng.integers(-40, 41, x[1].shape) * tiny            # subnormals
    if tokens > 2:
        x[2] = rng.integers(-36, 37, x[2].shape) / 16.0            # many ties at 5 significant bits
    if tokens > 3:
        x[3] = rng.uniform(-1, 1, x[3].shape) * 1.99 * big         # up to the type's largest
        x[3, :, 0] = 1.99 * big
    if tokens > 4:
        x[4, :, 0], x[4, :, 1] = 448.0, 449.0                      # either side of a scale's border
        x[4, 0, 1] = 447.0
    if tokens > 5:
        x[5, :, ::3] = 0.0
        x[5, :, 1] = LARGEST[dtype]
    return x


def bits_of(x, dtype):
    """The type's bits; the oracle's encoder has no NaN, which are put in here."""
    bits, _ = quantize(np.nan_to_num(x, nan=1.0, posinf=np.inf, neginf=-np.inf).astype(np.float32), dtype)
    bits[np.isnan(x)] = 0x7E00 if dtype == "f16" else 0x7FC0
    return bits


def append(x, v, slots, nb, bs, dtype, fill=0):
    T, Hkv, D = x.shape
    kb, vb = bits_of(x, dtype), bits_of(v, dtype)
    bufs = {n: H.DeviceBuffer.from_array(np.full(nb * bs * Hkv * (D if n in "kv" else 1), fill, np.uint8))
            for n in ("k", "v", "ke", "ve")}
    layer = H.Kv8Layer(bufs["k"].ptr, bufs["v"].ptr, bufs["ke"].ptr, bufs["ve"].ptr)
    dk, dv = H.DeviceBuffer.from_array(kb), H.DeviceBuffer.from_array(vb)
    ds = H.DeviceBuffer.from_array(np.asarray(slots, np.int32))
    shape = kv_shape(nb, bs, Hkv, D)
    H.check(H.hip_lib().sca_hip_kv8_append(ctypes.byref(layer), dk.ptr, dv.ptr, ds.ptr, T,
                                           ctypes.byref(shape), DTYPE_ID[dtype], None))
    sca_amd.synchronize()
    codes = [bufs[n].download(np.uint8).reshape(nb, bs, Hkv, D) for n in ("k", "v")]
    exps = [bufs[n].download(np.uint8).reshape(nb, Hkv, bs).transpose(0, 2, 1) for n in ("ke", "ve")]
    return codes, exps, bufs, (kb, vb)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D", DIMS)
def test_append_holds_the_nearest_values(hip, D, dtype):
    rng = np.random.default_rng(9000 + D)
    for Hkv, bs, T in ((1, 8, 1), (3, 16, 7), (8, 64, 100)):
        nb = -(-T // bs) + 2
        slots = rng.permutation(nb * bs)[:T]
        x = rows_with_everything(rng, T, Hkv, D, dtype)
        v = rows_with_everything(rng, T, Hkv, D, dtype)[::-1].copy()
        print(f"kv8 append {dtype} D={D} Hkv={Hkv} bs={bs} T={T}", flush=True)
        codes, exps, _, bits = append(x, v, slots, nb, bs, dtype, fill=0xA5)
        for got, ge, raw in zip(codes, exps, bits):
            want, we = hold8(to_float(raw, dtype).reshape(x.shape), dtype)
            page, off = slots // bs, slots % bs
            assert np.array_equal(ge[page, off], we)
            g = got[page, off]
            zero = want == 0
            assert np.array_equal(np.where(zero, g & 127, g), codes_of(want, we))
            untouched = np.ones((nb, bs), bool)
            untouched[page, off] = False
            assert (got[untouched] == 0xA5).all() and (ge[untouched] == 0xA5).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_nan_infinity_and_values_past_the_largest(hip, dtype):
    D, bs = 64, 16
    rng = np.random.default_rng(9100)
    x = rng.standard_normal((4, 2, D))
    x[0, 0, 5] = np.nan
    x[1, 1, 7], x[1, 1, 8] = np.inf, -np.inf
    x[2, 0, 9] = LARGEST[dtype] * 1.05
    x[3] = np.nan
    codes, exps, _, bits = append(x, x, [3, 0, 17, 9], 2, bs, dtype)
    deq = to_float(bits[0], dtype).reshape(x.shape).astype(np.float64)
    assert np.isnan(deq[3]).all() and np.isinf(deq[1, 1, 7:9]).all()
    want, we = hold8(deq, dtype)
    for got, ge in zip(codes, exps):
        for t, slot in enumerate([3, 0, 17, 9]):
            g = e4m3_values()[got[slot // bs, slot % bs]]
            e = ge[slot // bs, slot % bs]
            assert np.array_equal(e, we[t])
            vals = g * (2.0 ** (e.astype(np.float64) - 127))[:, None]
            assert np.array_equal(np.isnan(vals), np.isnan(deq[t]))
            np.testing.assert_array_equal(np.nan_to_num(vals), np.nan_to_num(want[t]))
    # a row of NaN alone has no largest magnitude: exponent as for zeros
    assert (exps[0][9 // bs, 9 % bs] == 1).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_read_back_is_exact_for_every_code_and_scale(hip, dtype):
    """Every code with every exponent whose product the type represents; append makes no others."""
    D, bs, Hkv = 64, 16, 1
    nb = 256 * 4 // bs
    codes = np.tile(np.arange(256, dtype=np.uint8).reshape(4, D), (256, 1)).reshape(nb, bs, Hkv, D)
    row_exp = np.repeat(np.arange(256, dtype=np.uint8), 4).reshape(nb, bs, Hkv)
    exps = np.ascontiguousarray(row_exp.transpose(0, 2, 1))
    dc, de = H.DeviceBuffer.from_array(codes), H.DeviceBuffer.from_array(exps)
    ids = H.DeviceBuffer.from_array(np.arange(nb, dtype=np.int32))
    out = H.DeviceBuffer(codes.size * 2)
    shape = kv_shape(nb, bs, Hkv, D)
    H.check(H.hip_lib().sca_hip_kv8_gather(dc.ptr, de.ptr, ids.ptr, nb, out.ptr, ctypes.byref(shape),
                                           DTYPE_ID[dtype], None))
    sca_amd.synchronize()
    got = to_float(out.download(np.uint16), dtype).reshape(codes.shape).astype(np.float64)
    want = e4m3_values()[codes] * (2.0 ** (row_exp.astype(np.float64) - 127))[..., None]
    least = 2.0 ** (-24 if dtype == "f16" else -133)
    with np.errstate(invalid="ignore"):
        fits = (np.abs(want) <= LARGEST[dtype]) & (want / least == np.rint(want / least))
    fits &= (row_exp >= 1)[..., None] & (row_exp <= 247)[..., None]
    assert fits.sum() > 256 * (30 if dtype == "f16" else 200)
    bad = fits & (got != want)
    assert not bad.any(), (codes[bad][:5], row_exp[..., None].repeat(D, -1)[bad][:5], got[bad][:5], want[bad][:5])
    nans = np.isnan(want) & (row_exp >= 1)[..., None] & (row_exp <= 247)[..., None]
    assert np.isnan(got[nans]).all()
    # rows never written: codes and exponent zero
    zero = (codes == 0) & (row_exp == 0)[..., None]
    assert (got[zero] == 0).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D,Hkv,bs", [(32, 1, 8), (96, 5, 32), (128, 8, 16), (256, 2, 64)])
def test_cache_round_trip_through_the_host_api(hip, dtype, D, Hkv, bs):
    """Appends of every kind into an 8-bit cache, two layers, pages read back, a sequence reset."""
    rng = np.random.default_rng(9300 + D)
    lens = [1, bs + 3, 2 * bs]
    cfg = C.KVCacheConfig(num_layers=2, num_kv_heads=Hkv, head_dim=D, block_size=bs, num_blocks=8,
                          max_num_seqs=3, dtype=dtype, storage="e4m3")
    cache = C.PagedKVCache(cfg)
    stats = cache.stats()
    assert stats["bytes"] == C.kv_cache_bytes(cfg) == 2 * 2 * 8 * bs * Hkv * (D + 1)
    data = {}
    for s, n in enumerate(lens):
        for layer in range(2):
            for name in "kv":
                b, d = quantize(rng.standard_normal((n, Hkv, D)).astype(np.float32), dtype)
                data[s, layer, name] = (b, d)
        t = [[C.Tensor.from_numpy(data[s, l, name][0], dtype) for name in "kv"] for l in range(2)]
        if s == 1:  # token by token for a part, with a reservation for all layers
            cache.reserve_batch([1] * n)
        else:
            cache.reserve(s, n)
        for l in range(2):
            cache.write_layer(l, *t[l])
    cache.sync_page_table()
    table = cache.page_table_host()

    def pages(s):
        return table[s, :-(-lens[s] // bs)]

    for s, n in enumerate(lens):
        ids = H.DeviceBuffer.from_array(pages(s).astype(np.int32))
        for layer in range(2):
            for name in "kv":
                got = to_float(cache.gather(name == "k", layer, ids.ptr, len(pages(s))).numpy(), dtype)
                got = got.reshape(-1, Hkv, D)
                want = np.zeros_like(got, dtype=np.float64)
                want[:n], _ = hold8(data[s, layer, name][1], dtype)
                np.testing.assert_array_equal(got.astype(np.float64), want)
    gone = H.DeviceBuffer.from_array(np.array(list(pages(1)) + [-1, 99], np.int32))
    n_gone = len(pages(1)) + 2
    cache.reset_seq(1)
    for layer in range(2):
        for is_key in (True, False):
            assert not cache.gather(is_key, layer, gone.ptr, n_gone).numpy().any()
    ids = H.DeviceBuffer.from_array(pages(2).astype(np.int32))
    got = to_float(cache.gather(True, 1, ids.ptr, len(pages(2))).numpy(), dtype).reshape(-1, Hkv, D)
    want, _ = hold8(data[2, 1, "k"][1], dtype)
    np.testing.assert_array_equal(got[:lens[2]].astype(np.float64), want)


def test_slots_outside_the_pool_are_skipped(hip):
    D, bs, nb = 64, 16, 3
    x = np.random.default_rng(9400).standard_normal((5, 2, D))
    slots = [-1, nb * bs, 5, nb * bs - 1, -7]
    codes, exps, _, _ = append(x, x, slots, nb, bs, "bf16", fill=0x11)
    written = np.zeros((nb, bs), bool)
    written[0, 5] = written[nb - 1, bs - 1] = True
    for c, e in zip(codes, exps):
        assert (c[~written] == 0x11).all() and (e[~written] == 0x11).all()
        assert (e[written] != 0x11).all()
