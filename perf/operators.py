"""The operators on other forms of the paged cache, as cases that can be timed and checked.

A layer's cache is one pool of K pages and one of V pages, ``block`` tokens a page, reached through block tables.

* ``store4``   -- a step's rows quantised into 4-bit pages and read back as the bf16 values they stand for;
* ``decode4``  -- one query a sequence over 4-bit pages;            ``prefill4`` -- rows of prompts or chunks over them;
* ``windec``   -- one query a sequence over bf16 pages, with a sliding window and first tokens that stay visible;
* ``winpre``   -- rows of prompts or chunks over bf16 pages, with the same window;
* ``copy``     -- pages copied inside every layer's pools: forks of a sequence, compaction.

A 4-bit page holds, for each KV head, ``block`` rows of 64 bytes (128 e2m1 codes, the even one in the low half of its
byte), then 4 bytes a row: the power of two (biased by 127) of each run of 32 values.  The rows' scales are padded to 16
bytes together.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

BF16, F32, F64, U8 = torch.bfloat16, torch.float32, torch.float64, torch.uint8
HD = 128
TILE = 64  # query rows of one prefill tile in the step's tile list


# ------------------------------------------------------------------------------------------------ the cases
def _decode(name, kind, nq, nkv, block, lens, rows, lo, hi, window=0, sinks=0, pad=0):
    """``rows`` sequences with contexts in [lo, hi] and ``pad`` padding rows with none."""
    return {"name": name, "kind": kind, "nq": nq, "nkv": nkv, "block": block, "lens": lens, "rows": rows, "lo": lo,
            "hi": hi, "window": window, "sinks": sinks, "pad": pad}


def _prefill(name, kind, nq, nkv, block, lens, first=0, chunks=0, lo=1, hi=1, past_lo=0, past_hi=0, window=0, sinks=0,
             rows=0, row_hi=1):
    """A fresh prompt of ``first`` tokens (0: none), ``chunks`` chunks of [lo, hi] tokens behind [past_lo, past_hi] cached
    ones, and ``rows`` single decode rows with up to ``row_hi`` cached tokens."""
    return {"name": name, "kind": kind, "nq": nq, "nkv": nkv, "block": block, "lens": lens, "first": first,
            "chunks": chunks, "lo": lo, "hi": hi, "past_lo": past_lo, "past_hi": past_hi, "window": window,
            "sinks": sinks, "rows": rows, "row_hi": row_hi}


def _copy(name, layers, block_bytes, blocks, pairs, shape):
    return {"name": name, "kind": "copy", "layers": layers, "block_bytes": block_bytes, "blocks": blocks, "pairs": pairs,
            "shape": shape}


def listed():
    return [
        # the rows of a small decode step, one token a sequence: the smallest write there is
        {"name": "store4_step", "kind": "store4", "tokens": 8, "nkv": 8, "block": 16},
        # the rows of a long prompt
        {"name": "store4_prompt", "kind": "store4", "tokens": 16384, "nkv": 8, "block": 256},
        # the ordinary decode step of a small server: 32 sequences of very different lengths
        _decode("decode4_batch", "decode4", 16, 8, 16, 2, 32, 128, 1024),
        # long contexts, what 4-bit pages are for: 0.57 GB of cache in a layer
        _decode("decode4_long", "decode4", 32, 8, 256, 5, 16, 32768, 32768),
        # two chunks of long prompts, odd sizes, behind what is cached already
        _prefill("prefill4_chunks", "prefill4", 16, 8, 16, 4, chunks=2, lo=389, hi=512, past_lo=5000, past_hi=8192),
        # one long prompt
        _prefill("prefill4_prompt", "prefill4", 32, 8, 256, 6, first=8192),
        # a single user far into a conversation, of which a short window is kept
        _decode("windec_single", "windec", 16, 8, 16, 1, 1, 5003, 5003, window=1000, sinks=4),
        # a full server whose contexts are far longer than the window
        _decode("windec_batch", "windec", 32, 8, 16, 7, 64, 700, 20000, window=4096, sinks=4),
        # prompts arriving together, ragged, with an odd window and odd pages
        _prefill("winpre_prompts", "winpre", 16, 8, 48, 3, first=3584, chunks=8, lo=128, hi=512, window=777, sinks=5),
        # one very long prompt
        _prefill("winpre_long", "winpre", 32, 8, 256, 6, first=16384, window=1024, sinks=4),
        # one prompt forked into eight samples: each of the others gets the last, half-filled page in every layer
        _copy("copy_fork", 28, 32768, 64, 7, "fork"),
        # compaction of a pool of 4-bit pages: the pages in use move to the front
        _copy("copy_compact", 28, 8704, 4096, 1500, "compact"),
    ]


def _log_int(rng, lo, hi):
    """A whole number whose logarithm is even over [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["store4", "decode4", "decode4", "prefill4", "windec", "winpre", "copy"])
    nq, nkv = rng.choice([(16, 8), (16, 8), (32, 8), (32, 8), (8, 8), (64, 8), (32, 2)])
    block = rng.choice([16, 16, 32, 48, 256, 24, 7])
    lens = rng.randrange(1 << 30)
    windowed = kind.startswith("win") or rng.random() < 0.3
    window = _log_int(rng, 1, 8192) if windowed else 0
    sinks = rng.choice([0, 1, 4, 4, 64, 130]) if windowed else 0
    if kind == "store4":
        c = {"kind": kind, "tokens": _log_int(rng, 1, 16384), "nkv": nkv, "block": block}
    elif kind in ("decode4", "windec"):
        rows = _log_int(rng, 1, 256)
        hi = _log_int(rng, 1, min(32768, 524288 // rows))
        c = _decode("", kind, nq, nkv, block, lens, rows, max(1, hi // rng.choice([1, 2, 8])), hi, window, sinks,
                    rng.choice([0, 0, 3]))
    elif kind in ("prefill4", "winpre"):
        if rng.random() < 0.5:
            n, hi = rng.choice([0, 0, 1, 5]), _log_int(rng, 17, 700)
            c = _prefill("", kind, nq, nkv, block, lens, first=_log_int(rng, 2, 4096), chunks=n, lo=max(2, hi // 4),
                         hi=hi, window=window, sinks=sinks)
        else:
            past, size = _log_int(rng, 64, 16384), _log_int(rng, 2, 700)
            c = _prefill("", kind, nq, nkv, block, lens, chunks=rng.choice([1, 1, 2, 4]), lo=max(2, size // 2), hi=size,
                         past_lo=past // 2, past_hi=past, window=window, sinks=sinks, rows=rng.choice([0, 0, 9]),
                         row_hi=_log_int(rng, 1, 3000))
    else:
        blocks = _log_int(rng, 8, 4096)
        c = _copy("", _log_int(rng, 1, 28), 16 * _log_int(rng, 32, 2048), blocks, _log_int(rng, 1, max(1, blocks // 3)),
                  rng.choice(["fork", "compact"]))
        while 2 * c["layers"] * c["blocks"] * c["block_bytes"] > 2 << 30:
            c["layers"] = max(1, c["layers"] // 2)
            c["block_bytes"] = max(512, c["block_bytes"] // 32 * 16)
    c.pop("name", None)
    return c


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape, spread=0.0):
    """N(0, 1) rounded to bf16; with ``spread`` each of the last dimension's channels has a size of its own, as keys have."""
    out = torch.empty(shape, dtype=BF16, device="cuda")
    size = torch.exp(spread * torch.randn(shape[-1], generator=gen, device="cuda"))
    flat = out.view(-1, shape[-1])
    for i in range(0, flat.shape[0], 1 << 20):
        part = flat[i:i + (1 << 20)]
        part.copy_(torch.randn(part.shape, generator=gen, device="cuda") * size)
    return out


def _spec(c):
    """[(cached tokens, this step's tokens)] of the step's sequences."""
    r = np.random.default_rng(c["lens"])
    if "pad" in c:
        return [(int(r.integers(c["lo"], c["hi"] + 1)) - 1, 1) for _ in range(c["rows"])]
    spec = [(0, c["first"])] if c["first"] else []
    for _ in range(c["chunks"]):
        n = int(r.integers(c["lo"], c["hi"] + 1))
        spec.append((int(r.integers(c["past_lo"], c["past_hi"] + 1)), n))
    spec += [(int(r.integers(0, c["row_hi"] + 1)), 1) for _ in range(c["rows"])]
    return [spec[i] for i in r.permutation(len(spec))]


def _ints(x):
    return torch.from_numpy(np.ascontiguousarray(x, np.int32)).cuda()


def _page_bytes(block):
    """Bytes one KV head takes in a 4-bit page."""
    return block * 64 + -(-block * 4 // 16) * 16


def _pack4(rows, block):
    """bf16 pages [n, nkv, block, HD] as 4-bit pages [n, nkv * _page_bytes(block)]."""
    n, nkv = rows.shape[:2]
    out = torch.zeros((n, nkv, _page_bytes(block)), dtype=U8, device="cuda")
    step = max(1, (1 << 24) // (nkv * block * HD))
    for i in range(0, n, step):
        codes, scales = _quantise(rows[i:i + step].to(F32))
        m = codes.shape[0]
        out[i:i + step, :, :block * 64] = (codes[..., 0::2] | codes[..., 1::2] << 4).reshape(m, nkv, -1)
        out[i:i + step, :, block * 64:block * 68] = scales.reshape(m, nkv, -1)
    return out.view(n, -1)


def _attention_inputs(c, seed):
    gen, spec = _gen(seed), _spec(c)
    block, nkv = c["block"], c["nkv"]
    need = [-(-(a + b) // block) for a, b in spec]
    ends = np.cumsum([0] + need)
    ids = np.random.default_rng(seed).permutation(int(ends[-1]))
    pad = c.get("pad", 0)
    tables = np.zeros((len(spec) + pad, max(need)), np.int32)
    for i, n in enumerate(need):
        tables[i, :n] = ids[ends[i]:ends[i + 1]]
    shape = (int(ends[-1]), nkv, block, HD)
    kc, vc = _normal(gen, *shape, spread=0.4), _normal(gen, *shape)
    if c["kind"].endswith("4"):
        kc, vc = _pack4(kc, block), _pack4(vc, block)
    q = _normal(gen, sum(b for _, b in spec) + pad, c["nq"], HD)
    ctx = [a + b for a, b in spec] + [0] * pad
    return {"c": c, "spec": spec, "kc": kc, "vc": vc, "q": q, "tables": _ints(tables), "ctx": _ints(ctx), "ctx_list": ctx,
            "out": torch.empty_like(q), "scale": 1 / math.sqrt(HD)}


def _tiles(spec):
    """The step's query tiles as the executor lists them: single rows first, then the lightest first."""
    tiles = []
    for i, (past, n) in enumerate(spec):
        tiles += [(n > 1, past + min(q0 + TILE, n), i, q0) for q0 in range(0, n, TILE)]
    tiles.sort(key=lambda t: t[:2])
    return [t[2] for t in tiles], [t[3] for t in tiles]


def _inputs(c, seed):
    gen = _gen(seed)
    if c["kind"] == "store4":
        T, nkv, block = c["tokens"], c["nkv"], c["block"]
        blocks = -(-T // block) + 2
        slots = np.random.default_rng(seed).permutation(blocks)[:, None] * block + np.arange(block)[None, :]
        shape = (blocks, nkv * _page_bytes(block))
        k, v = _normal(gen, T, nkv, HD, spread=0.4), _normal(gen, T, nkv, HD)
        return {"c": c, "k": k, "v": v, "slots": _ints(slots.reshape(-1)[:T]), "k2": torch.empty_like(k),
                "v2": torch.empty_like(v), "kc": torch.zeros(shape, dtype=U8, device="cuda"),
                "vc": torch.zeros(shape, dtype=U8, device="cuda")}
    if c["kind"] == "copy":
        r = np.random.default_rng(seed)
        n, blocks = c["pairs"], c["blocks"]
        if c["shape"] == "fork":  # few pages, each copied to several free ones
            ids = r.permutation(blocks)
            sources = max(1, n // 7)
            src, dst = ids[np.arange(n) % sources], ids[sources:sources + n]
        else:  # the used pages behind the first ones in use go to the free ones before them
            used = np.sort(r.permutation(blocks)[:2 * n])
            free = np.setdiff1d(np.arange(blocks), used)
            n = min(n, len(free))
            src, dst = used[::-1][:n], free[:n]
        pools = [torch.randint(0, 256, (blocks, c["block_bytes"]), dtype=U8, generator=gen, device="cuda")
                 for _ in range(2 * c["layers"])]
        return {"c": c, "pools": pools, "src": np.ascontiguousarray(src, np.int32),
                "dst": np.ascontiguousarray(dst, np.int32)}
    s = _attention_inputs(c, seed)
    if c["kind"] in ("prefill4", "winpre"):
        tile_seq, tile_q0 = _tiles(s["spec"])
        s.update(cu_q=_ints(np.cumsum([0] + [n for _, n in s["spec"]])), tile_seq=_ints(tile_seq), tile_q0=_ints(tile_q0))
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        _prepare_own(s)
    elif case["kind"] == "copy":
        s["src_dev"], s["dst_dev"] = (_ints(s[n]).long() for n in ("src", "dst"))
    return s


def run(state):
    return (_RUN_OWN if own else _RUN)[state["c"]["kind"]](state)


# ------------------------------------------------------------------------------------------------ plain forms
def _quantise(x):
    """f32 [..., HD] -> codes [..., HD] (0..15) and scale bytes [..., HD / 32]."""
    b = x.view(*x.shape[:-1], HD // 32, 32)
    amax = b.abs().amax(-1)
    low = torch.frexp(amax)[1] - 3  # amax / 2^low lies in [4, 8)
    e = low + (amax > 7 * torch.exp2(low.to(F32))).to(torch.int32)
    e = torch.where(amax > 0, e.clamp(-127, 125), -127)
    y = torch.ldexp(b.abs(), -e[..., None])
    code = ((y > 0.25).to(U8) + (y >= 0.75).to(U8) + (y > 1.25).to(U8) + (y >= 1.75).to(U8) + (y > 2.5).to(U8)
            + (y >= 3.5).to(U8) + (y > 5).to(U8))
    code = code | (torch.signbit(b).to(U8) << 3)
    bad = ~torch.isfinite(amax)
    scale = torch.where(bad, 255, e + 127).to(U8)
    return torch.where(bad[..., None], 0, code).view(x.shape), scale


def _values(codes, scales):
    """What bytes of codes [..., 64] and scales [..., 4] stand for: f32 [..., HD]."""
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=F32, device="cuda")
    grid = torch.cat([grid, -grid])
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()
    e = torch.exp2(scales.to(F32) - 127)
    e = torch.where(scales == 255, math.nan, e)
    return grid[c] * e.repeat_interleave(32, -1)


def _rows(pool, c, blocks, offsets):
    """Cache rows as f32: [..., nkv, HD] for index tensors of one shape."""
    nkv, block = c["nkv"], c["block"]
    if pool.dtype == BF16:
        return pool[blocks, :, offsets].to(F32)
    p = pool.view(pool.shape[0], nkv, -1)
    codes = p[:, :, :block * 64].unflatten(-1, (block, 64))
    scales = p[:, :, block * 64:block * 68].unflatten(-1, (block, 4))
    return _values(codes[blocks, :, offsets], scales[blocks, :, offsets])


def _run_store4(s):
    c, slots = s["c"], s["slots"].long()
    nkv, block = c["nkv"], c["block"]
    b, o = slots // block, slots % block
    for rows, pool, back in ((s["k"], s["kc"], s["k2"]), (s["v"], s["vc"], s["v2"])):
        codes, scales = _quantise(rows.to(F32))
        p = pool.view(pool.shape[0], nkv, -1)
        p[:, :, :block * 64].unflatten(-1, (block, 64))[b, :, o] = codes[..., 0::2] | codes[..., 1::2] << 4
        p[:, :, block * 64:block * 68].unflatten(-1, (block, 4))[b, :, o] = scales
        back.copy_(_rows(pool, c, b, o))
    return {"k": s["k2"], "v": s["v2"]}


def _run_decode(s):
    c, out = s["c"], s["out"]
    nq, nkv, block, window, sinks = c["nq"], c["nkv"], c["block"], c["window"], c["sinks"]
    G = nq // nkv
    longest = max(s["ctx_list"])
    keep = min(longest, window + sinks) if window else longest
    step = max(1, (1 << 27) // (keep * nkv * HD))
    for i in range(0, len(s["ctx_list"]), step):
        ctx = s["ctx"][i:i + step].long()
        at = torch.arange(keep, device="cuda")[None, :].expand(len(ctx), -1)
        if window:  # the sinks, then the window
            lo = torch.clamp(ctx - window, min=0)[:, None]
            first = torch.minimum(lo, torch.tensor(sinks, device="cuda"))
            at = torch.where(at < first, at, at - first + lo)
        seen = at < ctx[:, None]
        at = torch.where(seen, at, 0)
        b = torch.gather(s["tables"][i:i + step].long(), 1, at // block)
        k, v = (_rows(s[n], c, b, at % block).transpose(1, 2) for n in ("kc", "vc"))
        q = s["q"][i:i + step].to(F32).view(-1, nkv, G, HD)
        x = torch.matmul(q, k.transpose(-1, -2)) * s["scale"]
        x = x.masked_fill(~seen[:, None, None, :], -math.inf)
        top = x.amax(-1, keepdim=True)
        p = torch.exp(x - torch.where(top == -math.inf, 0, top))
        o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
        out[i:i + step] = torch.where(ctx[:, None, None, None] > 0, o, 0).view(-1, nq, HD)
    return out


def _run_prefill(s):
    c, out = s["c"], s["out"]
    nq, nkv, block, window, sinks = c["nq"], c["nkv"], c["block"], c["window"], c["sinks"]
    G, t = nq // nkv, 0
    for i, (past, n) in enumerate(s["spec"]):
        for q0 in range(0, n, 512):
            m = min(512, n - q0)
            end = past + q0 + m
            lo = max(0, past + q0 - window + 1) if window else 0
            at = torch.arange(lo, end, device="cuda")
            if lo and sinks:
                at = torch.cat([torch.arange(min(sinks, lo), device="cuda"), at])
            b = s["tables"][i].long()[at // block]
            k, v = (_rows(s[name], c, b, at % block).transpose(0, 1) for name in ("kc", "vc"))
            pos = past + q0 + torch.arange(m, device="cuda")
            seen = at[None, :] <= pos[:, None]
            if window:
                seen &= (at[None, :] > pos[:, None] - window) | (at[None, :] < sinks)
            q = s["q"][t + q0:t + q0 + m].to(F32).view(m, nkv, G, HD).permute(1, 2, 0, 3).reshape(nkv, G * m, HD)
            x = torch.matmul(q, k.transpose(-1, -2)).view(nkv, G, m, -1) * s["scale"]
            x = x.masked_fill_(~seen, -math.inf)
            p = torch.exp(x - x.amax(-1, keepdim=True))
            o = torch.matmul(p.view(nkv, G * m, -1), v).view(nkv, G, m, HD) / p.sum(-1, keepdim=True)
            out[t + q0:t + q0 + m] = o.permute(2, 0, 1, 3).reshape(m, nq, HD)
        t += n
    return out


def _run_copy(s):
    for p in s["pools"]:
        p[s["dst_dev"]] = p[s["src_dev"]]
    return s["pools"]


_RUN = {"store4": _run_store4, "decode4": _run_decode, "windec": _run_decode, "prefill4": _run_prefill,
        "winpre": _run_prefill, "copy": _run_copy}


# ------------------------------------------------------------------------------------------------ the framework's calls
def _prepare_own(s):
    from llmgen_amd import attention as A
    from llmgen_amd import cache

    A.init_device()
    s["L"] = cache.lib()
    if s["c"]["kind"] == "copy":
        s["list"] = cache.BlockCopies(s["pools"])
    elif s["c"]["kind"] != "store4":
        s["work"] = cache.attn_work()
        s["single"] = sum(n == 1 for _, n in s["spec"])


def _p(t):
    return t.data_ptr()


def _own_store4(s):
    c, L = s["c"], s["L"]
    T, nkv, block = c["tokens"], c["nkv"], c["block"]
    L.hip_store_kv4(_p(s["k"]), _p(s["v"]), _p(s["slots"]), _p(s["kc"]), _p(s["vc"]), T, nkv, HD, block)
    L.hip_load_kv4(_p(s["k2"]), _p(s["v2"]), _p(s["slots"]), _p(s["kc"]), _p(s["vc"]), T, nkv, HD, block)
    return {"k": s["k2"], "v": s["v2"]}


def _own_decode(s):
    c, L, work = s["c"], s["L"], s["work"]
    call = L.hip_attn_decode_kv4 if c["kind"] == "decode4" else L.hip_attn_decode_window
    call(_p(s["out"]), _p(s["q"]), _p(s["kc"]), _p(s["vc"]), _p(s["tables"]), _p(s["ctx"]), s["q"].shape[0], c["nq"],
         c["nkv"], HD, s["tables"].shape[1], c["block"], s["scale"], c["window"], c["sinks"], c["hi"], _p(work),
         work.numel())
    return s["out"]


def _own_prefill(s):
    c, L, work = s["c"], s["L"], s["work"]
    call = L.hip_attn_prefill_kv4 if c["kind"] == "prefill4" else L.hip_attn_prefill_window
    call(_p(s["out"]), _p(s["q"]), _p(s["kc"]), _p(s["vc"]), _p(s["tables"]), _p(s["ctx"]), _p(s["cu_q"]),
         _p(s["tile_seq"]), _p(s["tile_q0"]), s["tile_seq"].numel(), c["nq"], c["nkv"], HD, s["tables"].shape[1],
         c["block"], s["scale"], c["window"], c["sinks"], s["single"], _p(work), work.numel())
    return s["out"]


def _own_copy(s):
    s["list"].run(s["src"], s["dst"])
    return s["pools"]


_RUN_OWN = {"store4": _own_store4, "decode4": _own_decode, "windec": _own_decode, "prefill4": _own_prefill,
            "winpre": _own_prefill, "copy": _own_copy}


# ------------------------------------------------------------------------------------------------ work
def work(case):
    c, kind = case, case["kind"]
    if kind == "store4":
        n = 2 * c["tokens"] * c["nkv"]  # rows of K and V: read, written as pages, read back, written as rows
        return {"bytes": n * (256 + 68 + 68 + 256) + 8 * c["tokens"], "flops": 0}
    if kind == "copy":
        n = min(c["pairs"], c["blocks"] - 2 * c["pairs"]) if c["shape"] == "compact" else c["pairs"]
        return {"bytes": 2 * c["layers"] * 2 * n * c["block_bytes"], "flops": 0}
    window, sinks = c["window"], c["sinks"]
    row = 2 * c["nkv"] * (68 if kind.endswith("4") else 256)
    keys = pairs = tokens = 0
    for past, n in _spec(c):
        tokens += n
        lo = max(0, past - window + 1) if window else 0  # the first row's window begins here
        keys += past + n - lo + min(sinks, lo)
        pos = np.arange(past, past + n)
        seen = pos + 1
        if window:
            seen = np.minimum(pos + 1, window) + np.minimum(sinks, np.maximum(0, pos + 1 - window))
        pairs += int(seen.sum())
    return {"bytes": keys * row + 2 * 2 * HD * c["nq"] * tokens, "flops": 4 * HD * c["nq"] * pairs}


# ------------------------------------------------------------------------------------------------ 64-bit results
def exact(case, seed):
    return _EXACT[case["kind"]](case, _inputs(case, seed))


def _exact_store4(c, s):
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=F64, device="cuda")
    steps = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=F64, device="cuda")
    out = {}
    for name in ("k", "v"):
        x = s[name].to(F64).reshape(-1, 32)
        top = x.abs().amax(1, keepdim=True)
        power = torch.floor(torch.log2(top.clamp(min=2.0 ** -200))) - 2
        power = torch.where(top > 7 * torch.exp2(power), power + 1, power).clamp(-127, 125)
        y = x.abs() / torch.exp2(power)
        # a value on a border goes to the even code: up at the borders of odd index, down at the others
        up, down = torch.bucketize(y, borders, right=True), torch.bucketize(y, borders, right=False)
        code = torch.where(down % 2 == 1, up, down)
        out[name] = (steps[code] * torch.exp2(power) * torch.sign(x)).view(s[name].shape)
    return out


def _sequence64(pool, c, table, h, n):
    """Rows of KV head h of one sequence's first n tokens, in 64 bits."""
    block = c["block"]
    pages = table[:-(-n // block)].long()
    if pool.dtype == BF16:
        return pool[pages, h].reshape(-1, HD)[:n].to(F64)
    raw = pool.view(pool.shape[0], c["nkv"], -1)[pages, h]
    codes = raw[:, :block * 64].reshape(-1, 64)[:n]
    power = raw[:, block * 64:block * 68].reshape(-1, 4)[:n].to(F64) - 127
    nib = torch.empty((n, HD), dtype=F64, device="cuda")
    nib[:, 0::2], nib[:, 1::2] = (codes % 16).to(F64), torch.div(codes, 16, rounding_mode="floor").to(F64)
    sign, m = torch.where(nib >= 8, -1.0, 1.0), nib % 8
    e = torch.floor(m / 2)  # two bits of exponent, one of mantissa
    mag = torch.where(e == 0, (m % 2) / 2, (1 + (m % 2) / 2) * torch.exp2(e - 1))
    return sign * mag * torch.exp2(power).repeat_interleave(32, 1)


def _exact_attention(c, s):
    nq, nkv, window, sinks = c["nq"], c["nkv"], c["window"], c["sinks"]
    G, t = nq // nkv, 0
    out = torch.zeros(s["q"].shape, dtype=F64, device="cuda")
    for i, (past, n) in enumerate(s["spec"]):
        for h in range(nkv):
            k, v = (_sequence64(s[name], c, s["tables"][i], h, past + n) for name in ("kc", "vc"))
            kt = k.t().contiguous()
            for q0 in range(0, n, 2048):
                m = min(2048, n - q0)
                end = past + q0 + m
                pos = (past + q0 + torch.arange(m, device="cuda"))[:, None]
                at = torch.arange(end, device="cuda")[None, :]
                hidden = at > pos
                if window:
                    hidden |= (pos - at >= window) & (at >= sinks)
                for head in range(h * G, (h + 1) * G):
                    x = s["q"][t + q0:t + q0 + m, head].to(F64) @ kt[:, :end] * s["scale"]
                    out[t + q0:t + q0 + m, head] = torch.softmax(x.masked_fill_(hidden, -math.inf), -1) @ v[:end]
        t += n
    return out


def _exact_copy(c, s):
    before = [p.clone() for p in s["pools"]]
    for p, b in zip(s["pools"], before):
        for a, d in zip(s["src"].tolist(), s["dst"].tolist()) if c["pairs"] < 64 else ():
            p[d] = b[a]
        if c["pairs"] >= 64:
            p.index_copy_(0, _ints(s["dst"]).long(), b.index_select(0, _ints(s["src"]).long()))
    return s["pools"]


_EXACT = {"store4": _exact_store4, "decode4": _exact_attention, "windec": _exact_attention,
          "prefill4": _exact_attention, "winpre": _exact_attention, "copy": _exact_copy}
