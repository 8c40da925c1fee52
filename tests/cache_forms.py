"""Shared by the tests of the cache's other forms: 4-bit pages by their definition, a step over paged pools whose unseen
places hold infinities and NaN, and attention in 64 bits with the tolerance its roundings allow."""
from __future__ import annotations

import math

import numpy as np
import torch

HD = 128
GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
TILE = 64


# ---------------------------------------------------------------------------------------------- 4-bit pages
def bf16_values(bits: np.ndarray) -> np.ndarray:
    with np.errstate(invalid="ignore"):
        return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def quantise(x: np.ndarray):
    """Rows [..., 128] of float64 (bf16 values) -> codes [..., 128], scale bytes [..., 4], by the definition."""
    b = x.reshape(-1, 32)
    codes, scales = np.zeros(b.shape, np.uint8), np.zeros(len(b), np.uint8)
    for i, run in enumerate(b):
        if not np.isfinite(run).all():
            scales[i] = 255
            continue
        amax = np.abs(run).max()
        e = -127
        if amax > 0:
            e = math.frexp(amax)[1] - 3  # floor(log2 amax) - 2
            if amax > 7 * 2.0 ** e:
                e += 1
            e = min(max(e, -127), 125)
        y = np.abs(run) / 2.0 ** e
        d = np.abs(y[:, None] - GRID[None, :])
        near = d.min(1, keepdims=True)
        for j in range(32):  # nearest, ties to the even index
            at = np.flatnonzero(d[j] == near[j])
            code = at[0] if len(at) == 1 or at[0] % 2 == 0 else at[1]
            codes[i, j] = code | (8 if np.signbit(run[j]) else 0)
        scales[i] = e + 127
    return codes.reshape(x.shape), scales.reshape(*x.shape[:-1], 4)


def dequantise(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    v = GRID[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    p = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return v * np.repeat(p, 32, -1)


def head_bytes(block: int) -> int:
    return block * 64 + -(-block * 4 // 16) * 16


def page_views(pool: torch.Tensor, nkv: int, block: int):
    """(codes [n, nkv, block, 64], scales [n, nkv, block, 4]) of a pool of 4-bit pages, on the CPU."""
    p = pool.cpu().numpy().reshape(pool.shape[0], nkv, head_bytes(block))
    return (p[:, :, :block * 64].reshape(-1, nkv, block, 64), p[:, :, block * 64:block * 68].reshape(-1, nkv, block, 4))


def page_values(pool: torch.Tensor, nkv: int, block: int) -> np.ndarray:
    """float64 [n, nkv, block, 128] of either kind of pool."""
    if pool.dtype == torch.bfloat16:
        return pool.double().cpu().numpy()
    codes, scales = page_views(pool, nkv, block)
    nib = np.empty((*codes.shape[:-1], HD), np.uint8)
    nib[..., 0::2], nib[..., 1::2] = codes & 15, codes >> 4
    return dequantise(nib, scales)


# ---------------------------------------------------------------------------------------------- a step
def seen_by(pos: int, n: int, window: int, sinks: int) -> np.ndarray:
    """Which of keys 0..n-1 a row at position pos sees."""
    k = np.arange(n)
    s = k <= pos
    return s & ((k > pos - window) | (k < sinks)) if window else s


class Step:
    """A step of sequences (ctx, q_len) over pools of bf16 or 4-bit pages.  Places that no row of a sequence sees hold
    infinities and NaN; table entries of pages without a seen place name a page full of them."""

    def __init__(self, spec, nq, nkv, block, kv4=False, window=0, sinks=0, seed=0, poison=True, max_blocks=None):
        self.spec, self.nq, self.nkv, self.block = spec, nq, nkv, block
        self.kv4, self.window, self.sinks = kv4, window, sinks
        rng = np.random.default_rng(seed)
        need = [max(0, -(-c // block)) for c, _ in spec]
        self.max_blocks = max_blocks or max(max(need), 1)
        n = sum(need) + 1
        ids = rng.permutation(n)
        self.bad = int(ids[0])
        self.tables = np.full((len(spec), self.max_blocks), self.bad, np.int32)
        at = 1
        shape = (n, nkv, block, HD)
        size = np.exp(0.4 * rng.standard_normal(HD))
        k = (rng.standard_normal(shape) * size).astype(np.float32)
        v = rng.standard_normal(shape).astype(np.float32)
        unseen = np.ones((n, block), bool)
        for i, (ctx, q_len) in enumerate(spec):
            if ctx >= q_len and ctx > 0:
                seen = np.zeros(need[i] * block, bool)
                for pos in range(ctx - q_len, ctx):
                    seen[:ctx] |= seen_by(pos, ctx, window, sinks)
                for j in range(need[i]):
                    page = seen[j * block:(j + 1) * block]
                    unseen[ids[at + j]] = ~page
                    if page.any():
                        self.tables[i, j] = ids[at + j]
            at += need[i]
        self.k = torch.from_numpy(k).to(torch.bfloat16)
        self.v = torch.from_numpy(v).to(torch.bfloat16)
        if poison:
            b, o = np.nonzero(unseen)
            self.k[b, :, o] = float("nan")
            self.v[b, :, o] = float("inf")
            self.v[b[::2], :, o[::2]] = float("nan")
        self.rows = sum(q for _, q in spec)
        self.q = torch.from_numpy(rng.standard_normal((self.rows, nq, HD)).astype(np.float32)).to(torch.bfloat16)
        self.scale = 1 / math.sqrt(HD)

    def upload(self):
        dev = "cuda"
        self.kc, self.vc = self.k.to(dev), self.v.to(dev)
        if self.kv4:
            self.kc, self.vc = pack(self.kc), pack(self.vc)
        self.qd = self.q.to(dev)
        up = lambda x: torch.from_numpy(np.ascontiguousarray(x, np.int32)).to(dev)  # noqa: E731
        self.bt = up(self.tables)
        self.ctx = up([c for c, _ in self.spec])
        self.cu_q = up(np.cumsum([0] + [q for _, q in self.spec]))
        tiles = [(q > 1, min(q0 + TILE, q) - q + c, i, q0) for i, (c, q) in enumerate(self.spec) for q0 in range(0, q, TILE)]
        tiles.sort(key=lambda t: t[:2])
        self.tile_seq, self.tile_q0 = up([t[2] for t in tiles]), up([t[3] for t in tiles])
        self.n_tiles = len(tiles)
        self.out = torch.full((self.rows + 2, self.nq, HD), 7.0, dtype=torch.bfloat16, device=dev)  # two rows behind
        return self

    def decode(self, work=None, max_ctx=None):
        from llmgen_amd._lib import lib

        L, p = lib(), lambda t: t.data_ptr()
        call = L.hip_attn_decode_kv4 if self.kv4 else L.hip_attn_decode_window
        call(p(self.out), p(self.qd), p(self.kc), p(self.vc), p(self.bt), p(self.ctx), len(self.spec), self.nq, self.nkv, HD,
             self.max_blocks, self.block, self.scale, self.window, self.sinks,
             max(c for c, _ in self.spec) if max_ctx is None else max_ctx, None if work is None else p(work),
             0 if work is None else work.numel())
        return self.out

    def prefill(self, work=None, single=-1):
        from llmgen_amd._lib import lib

        L, p = lib(), lambda t: t.data_ptr()
        call = L.hip_attn_prefill_kv4 if self.kv4 else L.hip_attn_prefill_window
        call(p(self.out), p(self.qd), p(self.kc), p(self.vc), p(self.bt), p(self.ctx), p(self.cu_q), p(self.tile_seq),
             p(self.tile_q0), self.n_tiles, self.nq, self.nkv, HD, self.max_blocks, self.block, self.scale, self.window,
             self.sinks, single, None if work is None else p(work), 0 if work is None else work.numel())
        return self.out

    def reference(self):
        """(out, tolerance), float64 [rows, nq, HD].

        A result is a quotient of f32 sums, rounded once to bf16: half a step, 2^-8 |o|.  Its numerator's probabilities
        are rounded to bf16 as well: 2^-8 of the sum of p |v| over the denominator, a.  A score of f32 products and sums
        over 128 values is off by at most 2^-24 * 130 * |scale| sum |q k|, which moves a probability by as much,
        relatively, in numerator and denominator; 2^-16 a covers exp2 (a step of f32 on an exponent of up to 2^5), the
        sums over keys and the merges of partial results."""
        kv = [page_values(t, self.nkv, self.block) for t in (self.kc, self.vc)]
        q = self.q.double().numpy()
        out, tol = np.zeros(q.shape), np.zeros(q.shape)
        G, t = self.nq // self.nkv, 0
        for i, (ctx, q_len) in enumerate(self.spec):
            if ctx >= q_len and ctx > 0:
                pages = self.tables[i][:-(-ctx // self.block)]
                k, v = (x[pages].transpose(1, 0, 2, 3).reshape(self.nkv, -1, HD)[:, :ctx] for x in kv)
                for j in range(q_len):
                    seen = np.flatnonzero(seen_by(ctx - q_len + j, ctx, self.window, self.sinks))
                    for h in range(self.nq):
                        ks, vs, qr = k[h // G, seen], v[h // G, seen], q[t + j, h]
                        with np.errstate(invalid="ignore"):
                            s = self.scale * (ks @ qr)
                            p = np.exp(s - s.max())
                            p /= p.sum()
                            e = 2.0 ** -24 * 130 * self.scale * (np.abs(ks) @ np.abs(qr)).max()
                            out[t + j, h] = p @ vs
                            a = p @ np.abs(vs)
                            tol[t + j, h] = 2.0 ** -8 * np.abs(out[t + j, h]) + (2.0 ** -8 + 2 * e + 2.0 ** -16) * a * 1.01
            t += q_len
        return out, tol

    def check(self, what=""):
        torch.cuda.synchronize()
        from llmgen_amd._lib import lib

        assert lib().hip_last_error() == 0, what
        got = self.out.double().cpu().numpy()
        assert (got[self.rows:] == 7).all(), f"{what}: rows behind the last sequence were written"
        ref, tol = self.reference()
        compare(got[:self.rows], ref, tol, what)


def compare(got, ref, tol, what=""):
    same = (got == ref) | (np.isnan(got) & np.isnan(ref))
    with np.errstate(invalid="ignore"):
        bad = ~(same | (np.isfinite(ref) & (np.abs(got - ref) <= tol)))
    if bad.any():
        i = np.argwhere(bad)[0]
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} values outside, first at {i.tolist()}: got {got[tuple(i)]}, "
                             f"want {ref[tuple(i)]}, tolerance {tol[tuple(i)]}")


def pack(rows: torch.Tensor) -> torch.Tensor:
    """Pools [n, nkv, block, 128] bf16 as 4-bit pages (the definition, on the CPU), on the rows' device."""
    n, nkv, block, _ = rows.shape
    codes, scales = quantise_fast(rows.double().cpu().numpy())
    out = np.zeros((n, nkv, head_bytes(block)), np.uint8)
    out[:, :, :block * 64] = (codes[..., 0::2] | codes[..., 1::2] << 4).reshape(n, nkv, -1)
    out[:, :, block * 64:block * 68] = scales.reshape(n, nkv, -1)
    return torch.from_numpy(out.reshape(n, -1)).to(rows.device)


def quantise_fast(x: np.ndarray):
    """:func:`quantise` for whole arrays (a test holds the two against each other)."""
    b = x.reshape(*x.shape[:-1], 4, 32)
    with np.errstate(invalid="ignore"):
        amax = np.abs(b).max(-1)
        fine = np.isfinite(b).all(-1)
        top = np.where(fine, amax, 1.0)
        e = np.frexp(top)[1] - 3
        e = e + (top > 7 * np.exp2(e.astype(np.float64)))
        e = np.where(top > 0, np.clip(e, -127, 125), -127)
        y = np.abs(np.where(fine[..., None], b, 0.0)) / np.exp2(e.astype(np.float64))[..., None]
    c = sum((y > t if i % 2 == 0 else y >= t).astype(np.uint8) for i, t in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5)))
    c = c | (np.signbit(b).astype(np.uint8) << 3)
    return np.where(fine[..., None], c, 0).astype(np.uint8).reshape(x.shape), np.where(fine, e + 127, 255).astype(np.uint8)
