"""Helpers of the tests of 8-bit pages and of paged attention over several new tokens: the values that
8 bits hold, from the definition in 64 bits; pools with scattered pages; the attention formula in 64
bits; and the bounds that the kernels' outputs have to keep.

Bounds. With u half a step of the output type relative to the value (torch.finfo(t).eps / 2: 2^-11
fp16, 2^-8 bf16), a kernel's output may be off by
  * u |ref|          its own rounding;
  * u A              the rounding of every softmax weight to the type before the product with V, where A
                     is the mean of |v| under the softmax weights;
  * 2 e A            the weights' error before that, once in the numerator and once in the sum: a score
                     is a sum of D products in fp32 (2^-23 (D + 8) of scale * sum |q k|, twice a
                     correctly rounded sum's bound, as the matrix unit may truncate) and the exponential
                     is good to 2^-21 of itself and 2^-22 of its argument;
  * tiny             fp32 sums of V, 2^-20 A; fp16 outputs below 2^-14 are off by up to 2^-25, and fp16
                     weights far below the largest lose bits worth 2^-32 of it each.
The lse (fp32) may be off by e and 2^-22 |lse| + 2^-20.
"""

from __future__ import annotations

import numpy as np

from attn_util import ELEM_BYTES, quantize, to_float
from sca_amd import hip as H

HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}
LARGEST = {"f16": 61440.0, "bf16": 1.875 * 2.0 ** 127}
DIMS = [32, 64, 96, 128, 160, 192, 256]


def e4m3_values() -> np.ndarray:
    """The 256 codes' values (NaN for 0x7f and 0xff)."""
    code = np.arange(256)
    e, f = (code >> 3) & 15, code & 7
    mag = np.where(e == 0, f * 2.0 ** -9, (8 + f) * 2.0 ** (np.maximum(e, 1) - 10.0))
    mag = np.where((code & 127) == 127, np.nan, mag)
    return np.where(code >= 128, -mag, mag)


def hold8(x: np.ndarray, dtype: str):
    """(values, exponent bytes) that 8-bit pages hold for rows x [..., D] of the type's values."""
    x = np.clip(x.astype(np.float64), -LARGEST[dtype], LARGEST[dtype])  # (NaN stays)
    a = np.max(np.where(np.isnan(x), 0.0, np.abs(x)), axis=-1)
    k = np.full(a.shape, -126)
    some = a > 0
    k[some] = np.maximum(-126, np.ceil(np.log2(a[some] / 448.0) - 1e-9).astype(int))
    # (the logarithm only proposes k: the definition decides)
    k = np.where(a > 448.0 * 2.0 ** k.astype(np.float64), k + 1, k)
    lower = (k > -126) & (a <= 448.0 * 2.0 ** (k - 1.0))
    k = np.where(lower, k - 1, k)
    unit = 2.0 ** k.astype(np.float64)[..., None]
    y = x / unit
    _, ey = np.frexp(np.where(np.isnan(y), 0.0, y))
    step = 2.0 ** (np.maximum(ey - 1, -6) - 3.0)
    held = np.rint(y / step) * step
    return held * unit, (k + 127).astype(np.uint8)


def codes_of(values: np.ndarray, exponents: np.ndarray) -> np.ndarray:
    """The code bytes of held values (zero as +0, NaN as 0x7f)."""
    table = e4m3_values()
    positive = table[:127]
    y = values / (2.0 ** (exponents.astype(np.float64) - 127))[..., None]
    mag = np.where(np.isnan(y), 0.0, np.abs(y))
    at = np.searchsorted(positive, mag)
    assert np.array_equal(positive[at], mag)
    out = at.astype(np.uint8)
    out = np.where(y < 0, out | 128, out)
    return np.where(np.isnan(y), 127, out).astype(np.uint8)


def pool(lens, bs, Hkv, D, dtype, seed, held8, slack=3, std=1.0):
    """A pool with every sequence's pages scattered: dict with the table, the storage arrays for the
    device, and per sequence the float64 keys and values it stands for."""
    rng = np.random.default_rng(seed)
    need = [-(-max(n, 0) // bs) for n in lens]
    nb = sum(need) + slack
    perm = rng.permutation(nb).astype(np.int32)
    width = max(max(need), 1) + 2
    table = np.full((len(lens), width), -1, np.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = perm[at:at + n]
        at += n
    out = {"lens": list(lens), "bs": bs, "Hkv": Hkv, "D": D, "dtype": dtype, "table": table, "nb": nb,
           "held8": held8}
    for name in ("k", "v"):
        x = (rng.standard_normal((nb, bs, Hkv, D)) * std * np.exp(0.4 * rng.standard_normal((nb, bs, Hkv, 1))))
        bits, deq = quantize(x.astype(np.float32), dtype)
        if held8:
            vals, exps = hold8(deq, dtype)
            out[name] = codes_of(vals, exps)
            out[name + "_exp"] = np.ascontiguousarray(exps.transpose(0, 2, 1))  # [nb, Hkv, bs]
            out[name + "_val"] = vals
        else:
            out[name] = bits
            out[name + "_val"] = deq.astype(np.float64)
    return out


def sequence(pl, s, length=None):
    """(k [L, Hkv, D], v, mapped [L]) of sequence s; unmapped tokens are zeros."""
    n = pl["lens"][s] if length is None else length
    idx = np.arange(n)
    logical = idx // pl["bs"]
    width = pl["table"].shape[1]
    page = np.where(logical < width, pl["table"][s, np.minimum(logical, width - 1)], -1)
    ok = (page >= 0) & (page < pl["nb"])
    page = np.where(ok, page, 0)
    k = np.where(ok[:, None, None], pl["k_val"][page, idx % pl["bs"]], 0.0)
    v = np.where(ok[:, None, None], pl["v_val"][page, idx % pl["bs"]], 0.0)
    return k, v, ok


def attend64(q, k, v, ok, causal, scale):
    """out [n, Hq, D], lse [n, Hq], the mean A of |v| under the weights [n, Hq, D] and the score error
    e [n, Hq] of the module's bounds."""
    n, Hq, D = q.shape
    L, Hkv, _ = k.shape
    g = Hq // Hkv
    out = np.zeros((n, Hq, D))
    lse = np.full((n, Hq), -np.inf)
    A = np.zeros((n, Hq, D))
    err = np.zeros((n, Hq))
    if n == 0 or L == 0:
        return out, lse, A, err
    vis = np.broadcast_to(ok[None, :], (n, L)).copy()
    if causal:
        vis &= np.arange(L)[None, :] <= np.arange(n)[:, None] + (L - n)
    for h in range(Hq):
        kh, vh, qh = k[:, h // g], v[:, h // g], q[:, h].astype(np.float64)
        s = qh @ kh.T * scale
        size = np.where(vis, np.abs(qh) @ np.abs(kh).T * scale, 0.0).max(axis=1)
        s = np.where(vis, s, -np.inf)
        m = s.max(axis=1)
        seen = np.isfinite(m)
        w = np.exp(s - np.where(seen, m, 0.0)[:, None])
        l = w.sum(axis=1)
        safe = np.where(seen, l, 1.0)
        out[:, h] = np.where(seen[:, None], (w @ vh) / safe[:, None], 0.0)
        A[:, h] = np.where(seen[:, None], (w @ np.abs(vh)) / safe[:, None], 0.0)
        lse[:, h] = np.where(seen, np.where(seen, m, 0.0) + np.log(safe), -np.inf)
        spread = np.where(vis, np.abs(s - np.where(seen, m, 0.0)[:, None]), 0.0)
        spread = np.where(spread > 60, 60, spread).max(axis=1)
        err[:, h] = 2.0 ** -23 * (D + 8) * size + 2.0 ** -21 + 2.0 ** -22 * (spread + size)
    return out, lse, A, err


def check(got, ref, A, err, dtype, keys, tag):
    u = HALF_STEP[dtype]
    vmax = float(np.max(A)) if A.size else 0.0
    limit = 1.01 * u * np.abs(ref) + (1.01 * u + 2 * err[..., None] + 2.0 ** -20) * A + \
        keys * 2.0 ** -32 * vmax + (2.0 ** -25 if dtype == "f16" else 0.0)
    bad = ~(np.abs(got - ref) <= limit)
    assert not bad.any(), (f"{tag}: {int(bad.sum())} values off, worst "
                           f"{np.nanmax(np.abs(got - ref) / np.maximum(limit, 1e-30)):.2f} times the bound")


def check_lse(got, ref, err, tag):
    assert np.array_equal(np.isneginf(got), np.isneginf(ref)), tag
    fine = np.isfinite(ref)
    limit = err + 2.0 ** -22 * np.abs(np.where(fine, ref, 0.0)) + 2.0 ** -20
    off = np.abs(np.where(fine, got, 0.0) - np.where(fine, ref, 0.0))
    assert (off <= limit).all(), tag


class Device:
    """A pool's arrays on the GPU."""

    def __init__(self, pl):
        self.k, self.v = H.DeviceBuffer.from_array(pl["k"]), H.DeviceBuffer.from_array(pl["v"])
        self.k_exp = H.DeviceBuffer.from_array(pl["k_exp"]) if pl["held8"] else None
        self.v_exp = H.DeviceBuffer.from_array(pl["v_exp"]) if pl["held8"] else None
        self.table = H.DeviceBuffer.from_array(pl["table"])


def scale_of(D):
    return float(np.float32(1.0 / np.sqrt(np.float64(D))))


def download(buf, dtype, shape):
    return to_float(buf.download(np.uint16), dtype).reshape(shape).astype(np.float64)


__all__ = ["DIMS", "Device", "ELEM_BYTES", "HALF_STEP", "LARGEST", "attend64", "check", "check_lse",
           "codes_of", "download", "e4m3_values", "hold8", "pool", "scale_of", "sequence"]
