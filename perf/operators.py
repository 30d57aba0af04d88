"""The paged-cache operators in their plain form and as this library's calls.

Three operators, used together by a serving engine that keeps its keys and values in pages:

  store    tokens written into a paged cache that keeps K and V in 8 bits, and their pages read
           back as 16-bit values
  decode   one query token per sequence over such a cache
  chunk    ragged chunks of new tokens (prompts, parts of prompts, drafted tokens, single tokens
           beside them) over the pages of a 16-bit or an 8-bit cache, which hold the new tokens too

What 8 bits hold: of the D values x of one token and KV head, with a = max |x|, k is the least
integer (at least -126) with a <= 448 * 2^k, and x is held as the e4m3 value (4 significant bits,
smallest step 2^-9, ties to even) nearest to x / 2^k. Values beyond the largest e4m3 value times a
power of two that the 16-bit type has (61440 in fp16, 1.875 * 2^127 in bf16) are held as that.
Every product code * 2^k is a number of the 16-bit type.

Attention is softmax(scale * q k^T) v over the keys a query sees, scale = 1 / sqrt(D). In a causal
chunk query i of n sees the first L - n + i + 1 of the sequence's L keys, else all L.

Sizes are those of the repository's benchmark, tests and design notes, or generic.
"""

import math
import os
import random
import sys

import numpy as np
import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_TORCH = {"f16": torch.float16, "bf16": torch.bfloat16}
_LARGEST = {"f16": 61440.0, "bf16": 1.875 * 2.0 ** 127}  # what 8 bits hold at most


# ---- the cases ------------------------------------------------------------------------------------

def _store(name, dtype, seqs, low, high, mix, block, kv_heads, head_dim):
    c = {"kind": "store", "dtype": dtype, "seqs": seqs, "low": low, "high": high, "mix": mix,
         "block": block, "kv_heads": kv_heads, "head_dim": head_dim}
    return {"name": name, **c} if name else c


def _decode(name, dtype, seqs, low, high, mix, block, heads, kv_heads, head_dim):
    c = {"kind": "decode", "dtype": dtype, "seqs": seqs, "low": low, "high": high, "mix": mix,
         "block": block, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim}
    return {"name": name, **c} if name else c


def _chunk(name, dtype, storage, seqs, singles, new_low, new_high, low, high, mix, block, heads,
           kv_heads, head_dim, causal=True, lse=False):
    """`seqs` sequences of new_low .. new_high new tokens and `singles` of one, each behind
    low .. high tokens of context."""
    c = {"kind": "chunk", "dtype": dtype, "storage": storage, "seqs": seqs, "singles": singles,
         "new_low": new_low, "new_high": new_high, "low": low, "high": high, "mix": mix,
         "block": block, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
         "causal": causal, "lse": lse}
    return {"name": name, **c} if name else c


def listed():
    return [
        # One layer's K and V of a batch of prompts.
        _store("store_prompts", "bf16", 4, 1200, 3000, 1, 16, 8, 128),
        # One layer of a serving step: the new token of every sequence. Latency counts.
        _store("store_step", "f16", 64, 1, 1, 2, 16, 8, 128),
        # A long document at an odd head dim and the larger page.
        _store("store_long_d96", "bf16", 1, 30001, 30001, 3, 32, 8, 96),
        # One layer of the benchmark's paged serving step: 64 ragged sequences, 16-token pages.
        _decode("decode_64_ragged", "bf16", 64, 512, 16384, 1, 16, 32, 8, 128),
        # The smallest decode: one sequence.
        _decode("decode_1x1500", "f16", 1, 1500, 1500, 2, 16, 32, 8, 128),
        # A batch at a head dim between the powers of two.
        _decode("decode_16_d96", "bf16", 16, 3000, 5200, 3, 16, 32, 8, 96),
        # Chunked prefill: the last 512 tokens of a long context.
        _chunk("chunk_512", "bf16", "same", 1, 0, 512, 512, 12289, 12289, 1, 16, 32, 8, 128),
        # A few new tokens per conversation over its context (a short turn, or drafted tokens).
        _chunk("few_tokens", "bf16", "same", 8, 0, 6, 6, 4096, 4096, 2, 16, 32, 8, 128),
        # A mixed step: single tokens of running sequences beside chunks of new prompts.
        _chunk("mixed_step", "f16", "same", 3, 40, 300, 1000, 200, 6000, 3, 16, 32, 8, 64),
        # Prompts without context at the widest head, with the log-sum-exp a later merge needs.
        _chunk("prompts_d256_lse", "bf16", "same", 3, 0, 900, 2600, 0, 0, 4, 16, 16, 4, 256,
               lse=True),
        # The largest: long chunks over long 8-bit contexts.
        _chunk("chunk8_2048", "bf16", "e4m3", 4, 0, 2048, 2048, 6000, 14000, 5, 16, 32, 8, 128),
        # A handful of drafted tokens of one sequence over an 8-bit cache. Latency counts.
        _chunk("few8_tokens", "f16", "e4m3", 1, 0, 5, 5, 2300, 2300, 6, 16, 32, 8, 128),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


_HEADS = [(8, 8), (16, 16), (32, 32), (16, 8), (32, 8), (24, 8), (64, 8), (28, 4), (16, 2)]
_MOST_FLOPS = 1.4e12
_MOST_BYTES = 1.0e9


def draw(rng):
    while True:
        heads, kv_heads = rng.choice(_HEADS)
        dtype = rng.choice(["bf16", "f16"])
        # 128 and 64 are the common head dims; the others are supported and in use too.
        head_dim = rng.choice([128, 128, 128, 64, 64, 32, 96, 160, 192, 256])
        block = rng.choice([16, 16, 16, 8, 32, 64])
        mix = rng.randrange(1 << 20)
        kind = rng.choice(["store", "decode", "decode", "prompt", "chunk", "few", "mixed"])
        storage = rng.choice(["same", "e4m3"])
        causal = rng.random() < 0.85
        lse = rng.random() < 0.25
        if kind == "store":
            low = _log_int(rng, 1, 3000)
            c = _store("", dtype, _log_int(rng, 1, 200), low, low * rng.randint(1, 6), mix, block,
                       kv_heads, head_dim)
        elif kind == "decode":
            low = _log_int(rng, 64, 6000)
            c = _decode("", dtype, _log_int(rng, 1, 160), low, low * rng.randint(1, 12), mix, block,
                        heads, kv_heads, head_dim)
        elif kind == "prompt":
            low = _log_int(rng, 20, 4000)
            c = _chunk("", dtype, storage, _log_int(rng, 1, 12), 0, low, low * rng.randint(1, 4), 0,
                       0, mix, block, heads, kv_heads, head_dim, causal, lse)
        elif kind == "chunk":
            low = _log_int(rng, 64, 2048)
            past = _log_int(rng, 300, 20000)
            c = _chunk("", dtype, storage, _log_int(rng, 1, 6), 0, low, low, past,
                       past * rng.randint(1, 3), mix, block, heads, kv_heads, head_dim, causal, lse)
        elif kind == "few":
            past = _log_int(rng, 100, 20000)
            c = _chunk("", dtype, storage, _log_int(rng, 1, 40), 0, 2, rng.randint(2, 40), past,
                       past * rng.randint(1, 4), mix, block, heads, kv_heads, head_dim, causal, lse)
        else:
            past = _log_int(rng, 30, 6000)
            new = _log_int(rng, 50, 1500)
            c = _chunk("", dtype, storage, rng.randint(1, 4), _log_int(rng, 1, 100), new,
                       new * rng.randint(1, 3), past, past * rng.randint(1, 8), mix, block, heads,
                       kv_heads, head_dim, causal, lse)
        w = work(c)
        if w["flops"] <= _MOST_FLOPS and w["bytes"] <= _MOST_BYTES:
            return c


# ---- shapes -----------------------------------------------------------------------------------------

def _lengths(c):
    """(keys, new tokens) of every sequence."""
    rng = random.Random(1000003 * c["mix"] + c["seqs"])
    if c["kind"] != "chunk":
        lens = [rng.randint(c["low"], c["high"]) for _ in range(c["seqs"])]
        return lens, (lens if c["kind"] == "store" else [1] * len(lens))
    new = [rng.randint(c["new_low"], c["new_high"]) for _ in range(c["seqs"])]
    new += [1] * c["singles"]
    rng.shuffle(new)
    return [n + rng.randint(c["low"], c["high"]) for n in new], new


def _pairs(keys, new, causal):
    """Visible (query, key) pairs."""
    return new * (keys - new) + new * (new + 1) // 2 if causal else new * keys


def work(case):
    c = case
    d, hkv = c["head_dim"], c["kv_heads"]
    lens, new = _lengths(c)
    pages = sum(-(-n // c["block"]) for n in lens)
    held8 = 2 * hkv * (d + 1)  # K and V of a token in 8 bits, with their exponents
    if c["kind"] == "store":
        # Tokens in; codes out and in again; whole pages out in 16 bits.
        bytes_ = sum(lens) * (2 * hkv * d * 2 + 2 * held8 + 4) + pages * (c["block"] * 2 * hkv * d * 2 + 4)
        return {"bytes": bytes_, "flops": 6 * 2 * sum(lens) * hkv * d}
    eight = c["kind"] == "decode" or c["storage"] == "e4m3"
    held = held8 if eight else 2 * hkv * d * 2
    bytes_ = sum(lens) * held + 4 * pages + 2 * sum(new) * c["heads"] * d * 2
    if c.get("lse"):
        bytes_ += sum(new) * c["heads"] * 4
    causal = c.get("causal", False)
    pairs = sum(_pairs(n, m, causal) for n, m in zip(lens, new))
    return {"bytes": bytes_, "flops": 4 * c["heads"] * d * pairs}


# ---- inputs -----------------------------------------------------------------------------------------

def _tokens(c, seed):
    """K and V rows [tokens, H_kv, D] of all sequences one after the other, and the queries.

    Keys have a few large channels and both have tokens of different magnitude, as a model's
    projections give them."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    lens, new = _lengths(c)
    d, hkv, t = c["head_dim"], c["kv_heads"], _TORCH[c["dtype"]]
    total = sum(lens)
    channel = 1.0 + 3.0 * (torch.rand((hkv, d), generator=gen, device="cuda") < 0.03)
    k = (normal(total, hkv, d).mul_(channel).mul_(torch.exp(0.3 * normal(total, hkv, 1)))).to(t)
    v = (normal(total, hkv, d).mul_(torch.exp(0.3 * normal(total, hkv, 1)))).to(t)
    if c["kind"] == "store":
        return k, v, None
    return k, v, normal(sum(new), c["heads"], d).to(t)


def _hold8(x, largest):
    """(e4m3 values as float32, exponents) that stand for x [..., D]."""
    x = x.float().clamp(-largest, largest)
    bits = x.abs().amax(-1).view(torch.int32)
    k = (bits >> 23) - 127 - 8 + ((bits & 0x7FFFFF) > 0x600000).int()
    k = k.clamp_min(-126)
    return (x * _power(-k).unsqueeze(-1)).to(torch.float8_e4m3fn), k


def _power(k):
    """2^k in float32, -126 <= k <= 127."""
    return ((k + 127) << 23).view(torch.float32)


def _prepare_plain(c, seed):
    """Pages as a program without this library keeps them: a pool, and every sequence's page list."""
    k, v, q = _tokens(c, seed)
    lens, new = _lengths(c)
    bs, hkv, d = c["block"], c["kv_heads"], c["head_dim"]
    counts = [-(-n // bs) for n in lens]
    perm = torch.from_numpy(np.random.RandomState(c["mix"] % (1 << 31)).permutation(sum(counts))).cuda()
    pages = torch.split(perm, counts)
    offset = torch.cat([torch.arange(n, device="cuda") for n in lens])
    first = torch.repeat_interleave(torch.tensor([sum(counts[:i]) for i in range(len(lens))], device="cuda"),
                                    torch.tensor(lens, device="cuda"))
    slots = perm[first + offset // bs] * bs + offset % bs
    state = {"case": c, "pages": pages, "all_pages": perm, "slots": slots, "q": q, "lens": lens,
             "new": new}
    eight = c["kind"] != "chunk" or c["storage"] == "e4m3"
    for name, x in (("k", k), ("v", v)):
        kept = torch.float8_e4m3fn if eight else x.dtype
        pool = torch.zeros((sum(counts) * bs, hkv, d), dtype=x.dtype, device="cuda").to(kept)
        exps = torch.zeros((sum(counts) * bs, hkv), dtype=torch.int32, device="cuda")
        if c["kind"] == "store":
            state[name + "_new"] = x
        elif eight:
            codes, e = _hold8(x, _LARGEST[c["dtype"]])
            pool.view(torch.uint8)[slots] = codes.view(torch.uint8)
            exps[slots] = e
        else:
            pool[slots] = x
        state[name] = pool
        state[name + "_exp"] = exps
    return state


# ---- the same state in this library's cache ---------------------------------------------------------

def _library():
    path = os.path.join(_ROOT, "scicompute-attention_amd", "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    from sca_amd import host
    return host


def _wrap(host, t, dtype):
    """A borrowed sci::Tensor handle over a torch tensor."""
    dims = (host.c_i64 * t.dim())(*t.shape)
    return host.Tensor(host.host_lib().sca_tensor_wrap(t.data_ptr(), dims, t.dim(),
                                                       host.DTYPES[dtype], host.GPU), dtype)


class _Memory:
    """Device memory as torch sees it; `owner` keeps it alive."""

    def __init__(self, ptr, shape, typestr, owner):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": tuple(shape), "data": (ptr, False), "version": 3,
                                         "typestr": typestr}


def _result(t):
    """A tensor that the library returned."""
    f32 = t.dtype == "f32"
    out = torch.as_tensor(_Memory(t.data_ptr, t.shape, "<f4" if f32 else "<i2", t), device="cuda")
    return out if f32 else out.view(_TORCH[t.dtype])


_PIECE = 1024  # tokens a sequence grows by at a time while the others grow too


def _prepare_own(c, seed):
    host = _library()
    k, v, q = _tokens(c, seed)
    lens, new = _lengths(c)
    n, bs = len(lens), c["block"]
    eight = c["kind"] != "chunk" or c["storage"] == "e4m3"
    cache = host.PagedKVCache(host.KVCacheConfig(
        num_layers=1, num_kv_heads=c["kv_heads"], head_dim=c["head_dim"], block_size=bs,
        num_blocks=sum(-(-m // bs) for m in lens), max_num_seqs=n, dtype=c["dtype"],
        storage="e4m3" if eight else "same"))
    state = {"case": c, "host": host, "cache": cache, "keep": (k, v, q)}
    if c["kind"] == "store":
        # The step's slots, one reservation for every layer of a model.
        cache.reserve_batch(np.repeat(np.arange(n), lens))
        cache.sync_page_table()
        table = cache.page_table_host()
        pages = [table[s, i] for s, m in enumerate(lens) for i in range(-(-m // bs))]
        state["ids"] = torch.tensor(pages, dtype=torch.int32, device="cuda")
        state["k_new"], state["v_new"] = _wrap(host, k, c["dtype"]), _wrap(host, v, c["dtype"])
        torch.cuda.synchronize()
        return state
    # The contexts grow side by side in a shuffled order, so a sequence's pages are scattered.
    start, at = [0] * n, 0
    for s, m in enumerate(lens):
        start[s], at = at, at + m
    pieces = [s for s, m in enumerate(lens) for _ in range(0, m, _PIECE)]
    random.Random(c["mix"]).shuffle(pieces)
    done = [0] * n
    for s in pieces:
        m = min(_PIECE, lens[s] - done[s])
        lo = start[s] + done[s]
        cache.reserve(s, m)
        cache.write_layer(0, _wrap(host, k[lo:lo + m], c["dtype"]),
                          _wrap(host, v[lo:lo + m], c["dtype"]))
        done[s] += m
    cache.sync_page_table()
    if c["kind"] == "decode":
        seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        state["keep"] += (seq_lens,)
        state["q"] = _wrap(host, q.view(n, c["heads"], 1, c["head_dim"]), c["dtype"])
        state["cfg"] = host.AttentionConfig()
        state["params"] = {"seq_lens": seq_lens.data_ptr(), "num_seqs": n, "block_size": bs}
    else:
        cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        state["q"] = _wrap(host, q, c["dtype"])
        state["cfg"] = host.AttentionConfig(causal=c["causal"], return_lse=c["lse"], cu_seqlens_q=cu)
        state["params"] = {"num_seqs": n, "layer": 0}
    torch.cuda.synchronize()
    return state


def prepare(case, seed):
    return (_prepare_own if own else _prepare_plain)(dict(case), seed)


# ---- one pass ---------------------------------------------------------------------------------------

def _run_own(state):
    c, host, cache = state["case"], state["host"], state["cache"]
    if c["kind"] == "store":
        cache.write_layer(0, state["k_new"], state["v_new"])
        ids = state["ids"]
        return {"k": _result(cache.gather(True, 0, ids.data_ptr(), ids.numel())),
                "v": _result(cache.gather(False, 0, ids.data_ptr(), ids.numel()))}
    if c["kind"] == "decode":
        return {"out": _result(host.paged_attention(state["q"], cache, state["params"], state["cfg"]).out)}
    r = host.paged_attention_varlen(state["q"], cache, state["params"], state["cfg"])
    return {"out": _result(r.out), "lse": _result(r.lse) if c["lse"] else None}


_MOST_SCORES = 1 << 28


def _attend(q, k, v, causal, scale):
    """(out [n, H_q, D], lse [n, H_q]) of n queries over L keys [L, H_kv, D], in 32 bits."""
    n, hq, d = q.shape
    length, hkv, _ = k.shape
    group = hq // hkv
    q = q.view(n, hkv, group, d).permute(1, 2, 0, 3).reshape(hkv, group * n, d)
    k = k.permute(1, 2, 0).contiguous()
    v = v.permute(1, 0, 2).contiguous()
    hidden = None
    if causal and n > 1:
        row = torch.arange(n, device=q.device).repeat(group) + (length - n)
        hidden = torch.arange(length, device=q.device)[None, :] > row[:, None]
    step = max(1, min(hkv, _MOST_SCORES // (group * n * length)))
    outs, lses = [], []
    for h in range(0, hkv, step):
        s = torch.matmul(q[h:h + step], k[h:h + step]).mul_(scale)
        if hidden is not None:
            s.masked_fill_(hidden, float("-inf"))
        m = s.amax(-1, keepdim=True)
        s.sub_(m).exp_()
        l = s.sum(-1, keepdim=True)
        outs.append(torch.matmul(s, v[h:h + step]) / l)
        lses.append((m + l.log()).squeeze(-1))
    out = torch.cat(outs).view(hkv, group, n, d).permute(2, 0, 1, 3).reshape(n, hq, d)
    lse = torch.cat(lses).view(hkv, group, n).permute(2, 0, 1).reshape(n, hq)
    return out, lse


def _run_plain(state):
    c = state["case"]
    t, bs = _TORCH[c["dtype"]], c["block"]
    hkv, d = c["kv_heads"], c["head_dim"]
    if c["kind"] == "store":
        out = {}
        for name in ("k", "v"):
            codes, e = _hold8(state[name + "_new"], _LARGEST[c["dtype"]])
            state[name].view(torch.uint8)[state["slots"]] = codes.view(torch.uint8)
            state[name + "_exp"][state["slots"]] = e
            pool = state[name].view(torch.uint8).view(-1, bs, hkv, d)
            held = pool[state["all_pages"]].view(torch.float8_e4m3fn).float()
            exps = state[name + "_exp"].view(-1, bs, hkv)[state["all_pages"]]
            out[name] = (held * _power(exps).unsqueeze(-1)).to(t)
        return out
    eight = c["kind"] == "decode" or c["storage"] == "e4m3"
    causal, scale = c.get("causal", False), 1.0 / math.sqrt(d)
    outs, lses, at = [], [], 0
    for pages, length, n in zip(state["pages"], state["lens"], state["new"]):
        kv = []
        for name in ("k", "v"):
            if eight:
                held = state[name].view(torch.uint8).view(-1, bs, hkv, d)[pages].view(torch.float8_e4m3fn)
                held = held.float().mul_(_power(state[name + "_exp"].view(-1, bs, hkv)[pages]).unsqueeze(-1))
            else:
                held = state[name].view(-1, bs, hkv, d)[pages].float()
            kv.append(held.view(-1, hkv, d)[:length])
        out, lse = _attend(state["q"][at:at + n].float(), *kv, causal, scale)
        outs.append(out)
        lses.append(lse)
        at += n
    out = torch.cat(outs).to(t)
    if c["kind"] == "decode":
        return {"out": out.unsqueeze(2)}
    return {"out": out, "lse": torch.cat(lses) if c["lse"] else None}


def run(state):
    return _run_own(state) if "host" in state else _run_plain(state)


# ---- the same in 64 bits ----------------------------------------------------------------------------

def _held64(x, dtype):
    """The float64 values that 8 bits hold for x [..., D]: the nearest multiple of each value's
    step, from the definition."""
    x = x.double()
    x = torch.minimum(torch.maximum(x, torch.tensor(-_LARGEST[dtype], dtype=torch.float64, device=x.device)),
                      torch.tensor(_LARGEST[dtype], dtype=torch.float64, device=x.device))
    largest = x.abs().amax(-1, keepdim=True)
    part, e = torch.frexp(largest)  # largest = part * 2^e, 1/2 <= part < 1; 448 = 7/8 * 2^9
    k = torch.where(part <= 0.875, e - 9, e - 8)
    k = torch.where((largest == 0) | (k < -126), torch.full_like(k, -126), k)
    unit = torch.exp2(k.double())
    unit = torch.exp2(torch.round(torch.log2(unit)))
    y = x / unit
    _, ey = torch.frexp(y)
    step = torch.exp2(torch.round(torch.clamp(ey - 1, min=-6).double()) - 3)
    return torch.round(y / step) * step * unit


def _exact_attend(q, k, v, causal, scale):
    n, hq, d = q.shape
    length, hkv, _ = k.shape
    group = hq // hkv
    out = torch.empty((n, hq, d), dtype=torch.float64, device=q.device)
    lse = torch.empty((n, hq), dtype=torch.float64, device=q.device)
    keys = torch.arange(length, device=q.device)
    rows = max(1, min(n, (1 << 27) // (group * length)))
    for h in range(hkv):
        kt, vh = k[:, h].t().contiguous(), v[:, h].contiguous()
        for a in range(0, n, rows):
            e = min(n, a + rows)
            mine = q[a:e, h * group:(h + 1) * group].double().reshape(-1, d)
            s = torch.matmul(mine, kt).mul_(scale).view(e - a, group, length)
            if causal:
                last = torch.arange(a, e, device=q.device) + (length - n)
                s.masked_fill_((keys[None, :] > last[:, None])[:, None, :], float("-inf"))
            top = s.amax(-1, keepdim=True)
            w = torch.exp(s - top)
            total = w.sum(-1, keepdim=True)
            o = torch.matmul(w.view(-1, length), vh).view(e - a, group, d)
            out[a:e, h * group:(h + 1) * group] = o / total
            lse[a:e, h * group:(h + 1) * group] = (top + torch.log(total)).squeeze(-1)
    return out, lse


def exact(case, seed):
    c = case
    k, v, q = _tokens(c, seed)
    lens, new = _lengths(c)
    eight = c["kind"] != "chunk" or c["storage"] == "e4m3"
    scale = 1.0 / math.sqrt(c["head_dim"])
    found = {"k": [], "v": [], "out": [], "lse": []}
    at_kv, at_q = 0, 0
    for length, n in zip(lens, new):
        rows = [x[at_kv:at_kv + length] for x in (k, v)]
        rows = [_held64(x, c["dtype"]) if eight else x.double() for x in rows]
        at_kv += length
        if c["kind"] == "store":
            short = -length % c["block"]
            for name, x in zip("kv", rows):
                x = torch.cat([x, x.new_zeros((short, *x.shape[1:]))])
                found[name].append(x.view(-1, c["block"], *x.shape[1:]))
            continue
        o, l = _exact_attend(q[at_q:at_q + n], *rows, c.get("causal", False), scale)
        at_q += n
        found["out"].append(o)
        found["lse"].append(l)
    if c["kind"] == "store":
        return {"k": torch.cat(found["k"]), "v": torch.cat(found["v"])}
    out = torch.cat(found["out"])
    if c["kind"] == "decode":
        return {"out": out.unsqueeze(2)}
    return {"out": out, "lse": torch.cat(found["lse"]) if c["lse"] else None}
