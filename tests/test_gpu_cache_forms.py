"""GPU: 4-bit pages, sliding windows with sinks and page copies against 64-bit results from their definitions.

Places that a row does not see hold infinities and NaN in all of these steps (pages behind the context's end, between the
sinks and the window, whole pages there), and two rows behind the last sequence must stay as they are.  Tolerances are
derived in cache_forms.Step.reference."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from cache_forms import HD, Step, bf16_values, compare, dequantise, page_values, page_views, quantise_fast
from llmgen_amd import attention as A
from llmgen_amd import cache, host
from llmgen_amd import step as S
from llmgen_amd._lib import lib

pytestmark = pytest.mark.gpu


def _say(*a):
    print("[gpu-test]", *a, flush=True)


def _check_error():
    torch.cuda.synchronize()
    assert lib().hip_last_error() == 0


def p(t):
    return t.data_ptr()


# ------------------------------------------------------------------------------------------ rows into 4-bit pages
def _bits(kind, n, rng):
    if kind == "all":  # every bf16 there is, infinities and NaN among them
        return np.concatenate([rng.permutation(1 << 16), rng.integers(0, 1 << 16, n - (1 << 16))]).astype(np.uint16)
    size = {"normal": 0, "wide": 20, "tiny": -85, "huge": 86}[kind]
    x = rng.standard_normal(n) * np.exp(size * (rng.random(n) if kind == "wide" else 1.0))
    x[rng.random(n) < 0.05] = 0
    with np.errstate(over="ignore"):
        return (np.clip(x, -3.3e38, 3.3e38).astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)


@pytest.mark.parametrize("kind", ["normal", "wide", "tiny", "huge", "all"])
@pytest.mark.parametrize("T, nkv, block", [(1, 1, 1), (3, 8, 16), (130, 4, 7), (300, 8, 256)])
def test_store_and_load(gpu, kind, T, nkv, block):
    if kind == "all" and T * nkv * HD < 1 << 16:
        T = (1 << 16) // (nkv * HD) + 1
    _say("store4", kind, T, nkv, block)
    rng = np.random.default_rng(T * nkv + block)
    k, v = (_bits(kind, T * nkv * HD, rng).reshape(T, nkv, HD) for _ in range(2))
    blocks = -(-T // block) + 2
    slots = rng.permutation(blocks * block)[:T].astype(np.int32)
    slots[rng.random(T) < 0.2] = -1
    up = lambda x: torch.from_numpy(x.view(np.int16) if x.dtype == np.uint16 else x).cuda()  # noqa: E731
    kd, vd, sd = up(k), up(v), up(slots)
    kc, vc = (torch.full((blocks, lib().hip_kv4_block_bytes(nkv, HD, block)), 0xA5, dtype=torch.uint8, device="cuda")
              for _ in range(2))
    lib().hip_store_kv4(p(kd), p(vd), p(sd), p(kc), p(vc), T, nkv, HD, block)
    k2, v2 = torch.full_like(kd, 77), torch.full_like(vd, 77)
    lib().hip_load_kv4(p(k2), p(v2), p(sd), p(kc), p(vc), T, nkv, HD, block)
    _check_error()
    for src, pool, back in ((k, kc, k2), (v, vc, v2)):
        codes, scales = quantise_fast(bf16_values(src))
        want = np.full(tuple(pool.shape), 0xA5, np.uint8).reshape(blocks, nkv, -1)
        for t, s in enumerate(slots):
            if s >= 0:
                b, o = divmod(int(s), block)
                want[b, :, o * 64:o * 64 + 64] = codes[t, :, 0::2] | codes[t, :, 1::2] << 4
                want[b, :, block * 64 + o * 4:block * 64 + o * 4 + 4] = scales[t]
        assert np.array_equal(pool.cpu().numpy(), want.reshape(blocks, -1))
        got = back.cpu().numpy()
        assert (got[slots < 0] == 77).all()
        values, stored = bf16_values(got.view(np.uint16)), slots >= 0
        np.testing.assert_array_equal(values[stored], dequantise(codes, scales)[stored])


# ------------------------------------------------------------------------------------------ one query a sequence
WINDOWS = [(0, 0), (1, 0), (1, 1), (7, 4), (64, 0), (100, 33), (1000, 300)]


@pytest.mark.parametrize("kv4", [False, True], ids=["bf16", "kv4"])
@pytest.mark.parametrize("block", [16, 32, 48, 256, 7, 1])
@pytest.mark.parametrize("window, sinks", WINDOWS)
def test_decode(gpu, kv4, block, window, sinks):
    _say("decode", kv4, block, window, sinks)
    spec = [(c, 1) for c in (1, 2, 15, 16, 17, 33, 64, 65, 100, 257, 400)] + [(0, 1), (0, 1)]
    s = Step(spec, 8, 4, block, kv4, window, sinks, seed=block + window).upload()
    s.decode(cache.attn_work())
    s.check("split")
    s.out.fill_(7)
    s.decode(None)  # no scratch: one workgroup a (sequence, head)
    s.check("whole")


@pytest.mark.parametrize("kv4", [False, True], ids=["bf16", "kv4"])
@pytest.mark.parametrize("nq, nkv", [(1, 1), (3, 3), (8, 4), (8, 2), (16, 2), (16, 1), (32, 2)])
@pytest.mark.parametrize("window, sinks", [(0, 0), (70, 5)])
def test_decode_heads(gpu, kv4, nq, nkv, window, sinks):
    _say("decode heads", kv4, nq, nkv, window)
    s = Step([(300, 1), (5, 1), (0, 1), (77, 1)], nq, nkv, 16, kv4, window, sinks, seed=nq).upload()
    s.decode(cache.attn_work())
    s.check()


@pytest.mark.parametrize("kv4", [False, True], ids=["bf16", "kv4"])
@pytest.mark.parametrize("block", [16, 256, 24, 7])
@pytest.mark.parametrize("window, sinks", [(0, 0), (3000, 130), (5000, 4)])
def test_decode_long(gpu, kv4, block, window, sinks):
    _say("decode long", kv4, block, window, sinks)
    s = Step([(6001, 1), (40, 1), (5003, 1)], 4, 2, block, kv4, window, sinks, seed=5).upload()
    work = cache.attn_work()
    s.decode(work)
    s.check("split")
    first = s.out.clone()
    for _ in range(3):  # the scratch's counters are back at 0, and the order of the merge is fixed
        s.out.fill_(7)
        s.decode(work)
        assert torch.equal(s.out, first)
    # the longest context was not foreseen; then only a little scratch
    for kw in (dict(work=work, max_ctx=100), dict(work=work, max_ctx=0), dict(work=work[:65536 + 4 * 130 * 4 * 3 * 2])):
        s.out.fill_(7)
        s.decode(**kw)
        s.check(str(kw.get("max_ctx")))


def test_decode_many_sequences(gpu):
    """More (sequence, head) pairs than the scratch has counters: no split."""
    for kv4 in (False, True):
        _say("decode many", kv4)
        s = Step([(1 + i % 40, 1) for i in range(2100)], 8, 8, 16, kv4, 20, 3, seed=1).upload()
        s.decode(cache.attn_work())
        s.check()


@pytest.mark.parametrize("kv4", [False, True], ids=["bf16", "kv4"])
def test_visible_infinities_reach_their_row_only(gpu, kv4):
    _say("visible special", kv4)
    s = Step([(50, 1), (50, 1), (50, 1)], 4, 2, 16, kv4, 30, 4, seed=9)
    page, off = s.tables[1][45 // 16], 45 % 16
    s.v[page, 0, off, 3] = float("nan")
    s.k[s.tables[2][1], 1, 10, 5] = float("nan")
    s.upload()
    s.decode(cache.attn_work())
    torch.cuda.synchronize()
    got = s.out.double().cpu().numpy()
    ref, tol = s.reference()
    nan = np.isnan(ref)
    assert nan.any() and not nan[0].any()
    compare(got[:3], ref, tol)


# ------------------------------------------------------------------------------------------ prompts and chunks
@pytest.mark.parametrize("kv4", [False, True], ids=["bf16", "kv4"])
@pytest.mark.parametrize("block", [16, 64, 48, 256, 6, 7])
@pytest.mark.parametrize("window, sinks", WINDOWS + [(63, 65), (200, 64)])
def test_prefill(gpu, kv4, block, window, sinks):
    _say("prefill", kv4, block, window, sinks)
    spec = [(70, 70), (1, 1), (33, 33), (200, 65), (300, 2), (0, 1), (150, 1), (3, 5), (129, 64)]
    s = Step(spec, 4, 2, block, kv4, window, sinks, seed=block).upload()
    for work in (cache.attn_work(), None):
        for single in (-1, 3, 0):
            s.out.fill_(7)
            s.prefill(work, single)
            if single == -1 or work is not None:
                s.check(f"single {single} work {work is not None}")


@pytest.mark.parametrize("kv4", [False, True], ids=["bf16", "kv4"])
@pytest.mark.parametrize("nq, nkv", [(1, 1), (3, 3), (4, 2), (4, 1), (8, 1), (16, 1), (32, 2)])
@pytest.mark.parametrize("window, sinks", [(0, 0), (50, 5)])
def test_prefill_heads(gpu, kv4, nq, nkv, window, sinks):
    _say("prefill heads", kv4, nq, nkv, window)
    s = Step([(90, 66), (40, 1), (10, 10)], nq, nkv, 16, kv4, window, sinks, seed=nq).upload()
    for work in (cache.attn_work(), None):
        s.out.fill_(7)
        s.prefill(work)
        s.check()


@pytest.mark.parametrize("kv4", [False, True], ids=["bf16", "kv4"])
@pytest.mark.parametrize("nq, nkv", [(2, 2), (4, 2)])
@pytest.mark.parametrize("window, sinks", [(0, 0), (900, 130), (64, 1)])
def test_prefill_chunk_behind_long_context(gpu, kv4, nq, nkv, window, sinks):
    """Few units of many key tiles: split over workgroups and merged."""
    _say("prefill chunk", kv4, nq, window)
    s = Step([(2000, 37), (1500, 70)], nq, nkv, 16, kv4, window, sinks, seed=3).upload()
    work = cache.attn_work()
    s.prefill(work, 0)
    s.check()
    first = s.out.clone()
    for _ in range(3):
        s.out.fill_(7)
        s.prefill(work, 0)
        assert torch.equal(s.out, first)


@pytest.mark.parametrize("kv4", [False, True], ids=["bf16", "kv4"])
@pytest.mark.parametrize("nq, nkv", [(1, 1), (4, 1)])
def test_prefill_pieces_merged_twice(gpu, kv4, nq, nkv):
    """Key tiles for 16 pieces of a unit, 9 of others, 40 of one, and values that rows see or not in some of them."""
    _say("prefill pieces", kv4, nq)
    s = Step([(5000, 37), (2200, 66), (20500, 3)], nq, nkv, 16, kv4, 0, 0, seed=4)
    for seq, key, what, dim in ((0, 4970, "v", 3), (0, 1000, "v", 100), (1, 2150, "v", 64), (1, 2170, "k", 1),
                                (2, 20498, "v", 9), (2, 3, "v", 8)):
        x = s.v if what == "v" else s.k
        x[s.tables[seq][key // 16], 0, key % 16, dim] = float("inf")
    s.upload()
    work = cache.attn_work()
    s.prefill(work, 0)
    torch.cuda.synchronize()
    first = s.out.clone()
    got = s.out.double().cpu().numpy()[:s.rows]
    ref, tol = s.reference()
    special = ~np.isfinite(ref)
    assert special.any() and not special.all()
    compare(got, ref, tol)
    s.prefill(work, 0)
    assert torch.equal(s.out.view(torch.int16), first.view(torch.int16))
    assert not work[:65536].any()


@pytest.mark.parametrize("kv4", [False, True], ids=["bf16", "kv4"])
@pytest.mark.parametrize("nq, nkv, block", [(2, 2, 16), (4, 2, 48), (16, 1, 7)])
@pytest.mark.parametrize("window, sinks", [(0, 0), (2000, 5)])
def test_prefill_single_rows_of_long_contexts(gpu, kv4, nq, nkv, block, window, sinks):
    """Single rows whose keys are split over workgroups, behind sequences without rows: more of these than tiles."""
    _say("prefill long rows", kv4, nq, block, window)
    spec = [(0, 0)] * 30 + [(3000, 1), (90, 70), (2500, 1), (5, 0), (17, 1), (0, 1), (2049, 1)]
    s = Step(spec, nq, nkv, block, kv4, window, sinks, seed=nq, max_blocks=-(-9000 // block)).upload()
    work = cache.attn_work()
    for single in (5, -1, 1):  # the count, unknown, a wrong one
        s.out.fill_(7)
        s.prefill(work, single)
        s.check(f"single {single}")
        first = s.out.clone()
        s.prefill(work, single)
        assert torch.equal(s.out, first)
    assert not work[: 4 * nkv * len(spec)].any()  # left ready


@pytest.mark.parametrize("G", [1, 2, 4, 8])
@pytest.mark.parametrize("kv4", [False, True], ids=["bf16", "kv4"])
def test_prefill_many_units(gpu, kv4, G):
    """More units than the chip holds at once: the widest workgroups."""
    _say("prefill many", kv4, G)
    s = Step([(65 + i, 65 + i) for i in range(26)], 8 * G, 8, 16, kv4, 40, 3, seed=2)
    s.upload().prefill(cache.attn_work(), 0)
    # heads and sequences alike: a part of them is enough
    torch.cuda.synchronize()
    got = s.out.double().cpu().numpy()
    full, cut = s.spec, 2
    s.spec = full[:cut]
    s.rows = sum(q for _, q in s.spec)
    ref, tol = (x[:s.rows] for x in s.reference())
    compare(got[:s.rows], ref, tol)
    s.spec = full
    assert (got[sum(q for _, q in full):] == 7).all() and np.isfinite(got).all()


@pytest.mark.parametrize("kv4", [False, True], ids=["bf16", "kv4"])
@pytest.mark.parametrize("window, sinks", [(0, 0), (30, 5), (64, 70)])
@pytest.mark.parametrize("work", [True, False], ids=["split", "whole"])
def test_prefill_infinities_between_rows(gpu, kv4, window, sinks, work):
    """Infinities and NaN in keys and values that some rows of a tile see and others do not."""
    _say("prefill special", kv4, window, work)
    s = Step([(150, 140), (400, 80)], 4, 2, 16, kv4, window, sinks, seed=11)
    for seq, key, what, dim in ((0, 60, "v", 3), (0, 61, "v", 40), (0, 62, "v", 40), (0, 99, "k", 7), (0, 2, "v", 100),
                                (1, 330, "v", 64), (1, 345, "k", 1), (1, 380, "v", 5)):
        page, off = s.tables[seq][key // 16], key % 16
        x = s.v if what == "v" else s.k
        x[page, key % 2, off, dim] = [float("nan"), float("inf"), -float("inf")][key % 3]
    s.upload().prefill(cache.attn_work() if work else None, 0)
    torch.cuda.synchronize()
    got = s.out.double().cpu().numpy()[:s.rows]
    ref, tol = s.reference()
    special = ~np.isfinite(ref)
    assert special.any() and not special.all()
    compare(got, ref, tol)


# ------------------------------------------------------------------------------------------ the fused write
@pytest.mark.parametrize("T, nq, nkv, block", [(1, 1, 1, 16), (5, 16, 8, 16), (300, 32, 8, 256), (33, 3, 3, 7), (64, 8, 1, 48)])
def test_fused_norm_rope_and_4_bit_write(gpu, T, nq, nkv, block):
    """One launch leaves the bytes of the five it replaces, at extreme values too; q may be its own output."""
    from llmgen_amd.qwen3 import rope_tables

    _say("fused write", T, nq, nkv, block)
    L, gen = lib(), torch.Generator(device="cuda").manual_seed(T)
    rand = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    size = torch.exp(4 * rand(T, 1, 1))
    q, k, v = ((rand(T, n, HD) * size).to(torch.bfloat16) for n in (nq, nkv, nkv))
    v[0, 0, :32] = 0
    v[0, 0, 33], v[-1, -1, 127], k[-1, 0, 5] = float("inf"), float("nan"), float("nan")
    v[0, 0, 64:96] *= 2.0 ** -126
    qw, kw = (1 + 0.1 * rand(HD) for _ in range(2))
    cos, sin = (torch.from_numpy(np.asarray(t, np.float32)).cuda() for t in rope_tables(512, HD, 1e6))
    pos = torch.randint(0, 512, (T,), generator=gen, device="cuda", dtype=torch.int32)
    blocks = -(-T // block) + 2
    slots = torch.randperm(blocks * block, generator=gen, device="cuda")[:T].to(torch.int32)
    slots[1::7] = -1
    pools = [torch.full((blocks, L.hip_kv4_block_bytes(nkv, HD, block)), 17, dtype=torch.uint8, device="cuda") for _ in range(6)]
    qu, ku = q.clone(), k.clone()
    for x, w, n in ((qu, qw, nq), (ku, kw, nkv)):
        L.hip_rmsnorm(p(x), p(x), p(w), T * n, HD, 1e-6)
        L.hip_rope(p(x), p(x), p(cos), p(sin), p(pos), T, n, HD)
    L.hip_store_kv4(p(ku), p(v), p(slots), p(pools[0]), p(pools[1]), T, nkv, HD, block)
    qf, qi = torch.empty_like(q), q.clone()
    for i, (src, dst) in enumerate(((q, qf), (qi, qi))):
        L.hip_qk_norm_rope_store_kv4(p(dst), p(pools[2 + 2 * i]), p(pools[3 + 2 * i]), p(src), p(k), p(v), p(qw), p(kw), 1e-6,
                                     p(cos), p(sin), p(pos), p(slots), T, nq, nkv, HD, block)
    torch.cuda.synchronize()
    _check_error()
    for got in (qf, qi):
        assert torch.equal(got.view(torch.int16), qu.view(torch.int16))
    for i in (2, 4):
        assert torch.equal(pools[i], pools[0]) and torch.equal(pools[i + 1], pools[1])
    assert (pools[0] != 17).any()


# ------------------------------------------------------------------------------------------ copies
@pytest.mark.parametrize("shape, dtype", [((9, 16), torch.uint8), ((40, 3, 1088), torch.uint8), ((12, 2, 16, 128), torch.bfloat16),
                                          ((5, 16400), torch.uint8), ((700, 48), torch.uint8)])
@pytest.mark.parametrize("n_pools", [1, 3, 70])
def test_copy_blocks(gpu, shape, dtype, n_pools):
    _say("copy", shape, n_pools)
    rng = np.random.default_rng(shape[0])
    pools = [torch.randint(0, 256, shape, dtype=torch.uint8, device="cuda").to(dtype) for _ in range(n_pools)]
    before = [x.clone() for x in pools]
    ids = rng.permutation(shape[0])
    n = shape[0] // 2
    src, dst = ids[rng.integers(0, n, n)], ids[n:2 * n]
    src[0], dst[0] = ids[-1], ids[-1] if shape[0] % 2 else src[0]  # a pair that does nothing
    if src[0] != dst[0]:
        src, dst = src[1:], dst[1:]
    copies = cache.BlockCopies(pools)
    copies.run(src, dst)
    copies.run([], [])
    _check_error()
    for x, b in zip(pools, before):
        want = b.clone()
        for a, d in zip(src, dst):
            want[d] = b[a]
        assert torch.equal(x, want)
    copies.run([0, 1], [2, 2])  # refused: nothing moves
    torch.cuda.synchronize()
    assert lib().hip_last_error() != 0
    assert torch.equal(pools[0][2], want[2] if n_pools == 1 else pools[0][2])


def test_block_copies_refuses_other_pools(gpu):
    a = torch.zeros(4, 64, dtype=torch.uint8, device="cuda")
    for other in (torch.zeros(5, 64, dtype=torch.uint8, device="cuda"), torch.zeros(4, 48, dtype=torch.uint8, device="cuda"),
                  torch.zeros(64, 4, dtype=torch.uint8, device="cuda").t(), torch.zeros(4, 65, dtype=torch.uint8, device="cuda")):
        with pytest.raises(ValueError):
            cache.BlockCopies([a, other])
    for src, dst in (([1], [2, 3]), ([0.5], [1]), ([1 << 32], [1]), (np.array([1 << 32]), [1]), ([[0]], [[1]])):
        with pytest.raises(ValueError):
            cache.BlockCopies([a]).run(src, dst)


# ------------------------------------------------------------------------------------------ graphs and streams
@pytest.mark.parametrize("kv4", [False, True], ids=["bf16", "kv4"])
def test_captured_steps_replay(gpu, kv4):
    """A captured sequence of a row write, decode, prefill and a page copy, replayed with other work in between."""
    _say("graph", kv4)
    L = lib()
    d = Step([(3000, 1), (17, 1)], 4, 2, 16, kv4, 0 if kv4 else 2500, 4, seed=1).upload()
    f = Step([(1500, 40), (30, 1)], 4, 2, 16, kv4, 700, 4, seed=2).upload()
    work = torch.empty(L.hip_attn_work_bytes(), dtype=torch.uint8, device="cuda")
    L.hip_attn_work_init(p(work), work.numel())
    copies = cache.BlockCopies([d.kc, d.vc])
    spare = d.bad  # a page no row sees
    k = torch.randn(1, 2, HD, device="cuda").to(torch.bfloat16)
    slot = torch.tensor([int(d.tables[0][2999 // 16]) * 16 + 2999 % 16], dtype=torch.int32, device="cuda")

    def step():
        if kv4:
            L.hip_store_kv4(p(k), p(k), p(slot), p(d.kc), p(d.vc), 1, 2, HD, 16)
        else:
            L.hip_store_kv(p(k), p(k), p(slot), p(d.kc), p(d.vc), 1, 2, HD, 16)
        d.decode(work)
        f.prefill(work)
        copies.run([int(d.tables[1][0])], [spare])

    step()
    torch.cuda.synchronize()
    assert L.hip_graph_begin() == 0
    step()
    graph = L.hip_graph_end()
    assert graph
    try:
        for i in range(4):
            k.copy_(torch.randn(1, 2, HD, device="cuda"))
            d.qd.copy_(torch.randn_like(d.qd.float()))
            step()
            torch.cuda.synchronize()
            eager = d.out.clone(), f.out.clone(), d.kc.clone()
            d.out.fill_(7)
            f.out.fill_(7)
            d.kc[spare].zero_()
            torch.cuda.synchronize()
            L.hip_graph_launch(graph)
            for got, want in zip((d.out, f.out, d.kc), eager):
                assert torch.equal(got.view(torch.uint8), want.view(torch.uint8)), i
    finally:
        torch.cuda.synchronize()
        L.hip_graph_destroy(graph)
    _check_error()


def test_scratch_is_ready_for_any_stream(gpu):
    """Memory that torch's stream still writes when it becomes a scratch is clear for calls on another stream."""
    _say("scratch ready")
    side = torch.cuda.Stream()
    for _ in range(3):
        dirty = torch.empty(lib().hip_attn_work_bytes(), dtype=torch.uint8, device="cuda")
        for _ in range(20):
            dirty.fill_(255)
        del dirty
        work = cache.attn_work()
        with torch.cuda.stream(side):
            seen = work.clone()
        side.synchronize()
        assert not seen.any()


def test_two_streams_with_a_scratch_each(gpu):
    _say("two streams")
    L, main = lib(), lib().hip_get_stream()
    steps = [Step([(4000 + 7 * i, 1), (900, 1)], 8, 4, 16, i == 0, 0, 0, seed=i).upload() for i in range(2)]
    works = [cache.attn_work() for _ in steps]
    alone = []
    for s, w in zip(steps, works):
        alone.append(s.decode(w).clone())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    try:
        for i in range(6):
            for s, w, st in zip(steps, works, streams):
                L.hip_set_stream(st.cuda_stream)
                s.decode(w)
    finally:
        L.hip_set_stream(main)
    torch.cuda.synchronize()
    for s, want in zip(steps, alone):
        assert torch.equal(s.out, want)
        s.check()


# ------------------------------------------------------------------------------------------ together, as they are used
def _bind(entries, nq, nkv, block, mb, max_len):
    ws = A.Workspace.allocate(nq, HD, len(entries), max_len, A.meta_bytes(entries, mb))
    A.bind_step(entries, ws, nq, nkv, HD, block, mb, max_len)
    return ws


def _attend(mgr, x, entries, nq, nkv, block, mb, max_len):
    """One attention node over the step's rows x = (q, k, v)."""
    ws = _bind(entries, nq, nkv, block, mb, max_len)
    out = torch.full_like(x[0], 7)
    A.g_attn_mgr = mgr
    A.PagedAttentionImpl.execute(0, A.AttnNode(out, list(x), layer_id=0))
    torch.cuda.synchronize()
    del ws
    return out


@pytest.mark.parametrize("kv4, window, sinks", [(True, 0, 0), (True, 60, 4), (False, 60, 4), (False, 0, 0)])
def test_prompt_forks_and_compaction(gpu, kv4, window, sinks):
    """A prompt in two chunks, forked into three samples that each write into a page of their own, decoded in one step,
    two given back, the rest compacted and decoded again: the attention node, the block manager and the page copies."""
    _say("together", kv4, window)
    nq, nkv, block, mb, max_len = 8, 4, 16, 16, 256
    gen = torch.Generator(device="cuda").manual_seed(3)
    rows = lambda n: [torch.randn(n, h, HD, generator=gen, device="cuda").to(torch.bfloat16) for h in (nq, nkv, nkv)]  # noqa: E731
    blocks = host.Blocks(40)
    mgr = A.PagedAttentionManager()
    layer = mgr.reserve_layer(0, 40, nkv, block, HD, kv4=kv4, window=window, sinks=sinks, work=cache.attn_work())
    copies = cache.BlockCopies([layer.k, layer.v])
    blocks.alloc(5)  # somebody else's pages
    table = blocks.alloc(7)
    history = [[], []]  # the sequence's own k, v rows

    def expect(out, q, kv, first):
        """Each row of q against the rows its sequence holds, through the definition of the pages."""
        s = Step([(len(kv[0]), len(q))], nq, nkv, block, kv4, window, sinks)
        pages = -(-len(kv[0]) // block)
        for name, x in (("kc", kv[0]), ("vc", kv[1])):
            t = torch.zeros(pages * block, nkv, HD, dtype=torch.bfloat16)
            t[:len(x)] = x
            t = t.view(pages, block, nkv, HD).transpose(1, 2).contiguous()
            setattr(s, name, t)
        if kv4:
            from cache_forms import pack
            s.kc, s.vc = pack(s.kc), pack(s.vc)
        s.tables = np.arange(pages, dtype=np.int32)[None]
        s.q = q.cpu()
        ref, tol = s.reference()
        compare(out.double().cpu().numpy(), ref, tol, first)

    for a, n in ((0, 70), (70, 35)):
        x = rows(n)
        out = _attend(mgr, x, [S.Entry(a, n, table)], nq, nkv, block, mb, max_len)
        history = [torch.cat([h, y.cpu()]) if len(h) else y.cpu() for h, y in zip(history, x[1:])]
        expect(out, x[0], history, f"chunk at {a}")
    tables = [table, blocks.fork(table), blocks.fork(table)]
    x = rows(3)
    pairs = [blocks.writable(t, 105 // block) for t in tables]
    assert [pr is None for pr in pairs] == [False, False, True]
    src, dst = zip(*[pr for pr in pairs if pr])
    copies.run(src, dst)
    out = _attend(mgr, x, [S.Entry(105, 1, t) for t in tables], nq, nkv, block, mb, max_len)
    own = []
    for i in range(3):
        own.append([torch.cat([h, y[i:i + 1].cpu()]) for h, y in zip(history, x[1:])])
        expect(out[i:i + 1], x[0][i:i + 1], own[i], f"sample {i}")
    blocks.free(tables[0])
    blocks.free(range(5))
    blocks.free(tables[1])
    rest = [tables[2]]
    src, dst = blocks.compact(rest)
    assert len(src) and max(rest[0]) == 6
    copies.run(src, dst)
    x = rows(1)
    assert blocks.writable(rest[0], 106 // block) is None
    out = _attend(mgr, x, [S.Entry(106, 1, rest[0])], nq, nkv, block, mb, max_len)
    expect(out, x[0], [torch.cat([h, y.cpu()]) for h, y in zip(own[2], x[1:])], "after compaction")
    _check_error()


@pytest.mark.parametrize("kv4, window, sinks", [(True, 0, 0), (True, 40, 4), (False, 40, 4)])
def test_model_with_another_form(gpu, kv4, window, sinks):
    """The Qwen3 forward over such a cache: the fused and the unfused layers agree bit for bit, and a layer's pages hold
    what the definition says of the rows that a bf16 cache holds."""
    from llmgen_amd.qwen3 import Qwen3, Qwen3Config, random_weights

    _say("model", kv4, window)
    kw = dict(vocab=512, hidden=256, n_layers=2, n_head=4, n_kv_head=2, ffn=512, max_model_len=256)
    cfg = Qwen3Config(**kw, kv4=kv4, window=window, sinks=sinks)
    weights = random_weights(cfg, seed=1)
    table = list(range(10))
    ids = [int(i) for i in np.random.default_rng(0).integers(0, 512, 101)]
    logits = []
    for fused in (True, False):
        m = Qwen3(cfg, weights, num_blocks=12)
        m.forward([S.Entry(0, 100, table)], ids[:100], fused_qk=fused)
        logits.append(m.last_logits.clone())
        m.forward([S.Entry(100, 1, table)], ids[100:], fused_qk=fused)
        logits.append(m.last_logits.clone())
    assert torch.equal(logits[0], logits[2]) and torch.equal(logits[1], logits[3])
    assert torch.isfinite(logits[1].view(torch.bfloat16)).all()
    plain = Qwen3(Qwen3Config(**kw), weights, num_blocks=12)
    plain.forward([S.Entry(0, 100, table)], ids[:100])
    # the first layer's rows do not depend on attention
    for pool, other in ((m.kv[0].k, plain.kv[0].k), (m.kv[0].v, plain.kv[0].v)):
        rows = other[:6].double().cpu().numpy()
        got = page_values(pool, 2, 16)[:6]
        if kv4:
            rows = dequantise(*quantise_fast(rows))
        np.testing.assert_array_equal(got, rows)
    m.copy_blocks([0], [11])
    torch.cuda.synchronize()
    assert all(torch.equal(x[0], x[11]) for kv in m.kv for x in (kv.k, kv.v))
    if kv4:
        assert page_views(m.kv[0].k, 2, 16)[0].shape == (12, 2, 16, 64)
    _check_error()


@pytest.mark.parametrize("kv4, window, sinks", [(True, 0, 0), (True, 90, 4), (False, 90, 4)])
def test_decode_graph_buckets_of_another_form(gpu, kv4, window, sinks):
    """The executor's decode graph buckets over layers of such a form, against the eager attention node, with changing
    batches and pages that the window has passed given back."""
    _say("buckets", kv4, window)
    nq, nkv, block, max_len = 8, 4, 16, 512
    mb = max_len // block
    work = cache.attn_work()
    layers = [[], []]
    mgr = A.PagedAttentionManager()
    gen = torch.Generator(device="cuda").manual_seed(5)
    for i in range(2):
        st = mgr.reserve_layer(i, 100, nkv, block, HD, kv4=kv4, window=window, sinks=sinks, work=work)
        fill = [torch.randn(100 * block, nkv, HD, generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2)]
        slots = torch.arange(100 * block, dtype=torch.int32, device="cuda")
        store = lib().hip_store_kv4 if kv4 else lib().hip_store_kv
        store(p(fill[0]), p(fill[1]), p(slots), p(st.k), p(st.v), 100 * block, nkv, HD, block)
        layers[0].append(st.k)
        layers[1].append(st.v)
    graphs = host.Graphs(*layers, nq, nkv, HD, block, max_len, 4, form=st.form, work=work)
    try:
        rng = np.random.default_rng(0)
        for n in (1, 3, 4, 2):
            blocks = host.Blocks(100)
            lens = [int(x) for x in rng.integers(1, max_len, n)]
            tables = [blocks.alloc(-(-c // block)) for c in lens]
            if window:  # pages between the sinks and the window: given back, their entries are not read
                for c, t in zip(lens, tables):
                    for j in range(-(-sinks // block), max(0, c - window) // block):
                        blocks.free([t[j]])
                        t[j] = 0
            x = [torch.randn(n, h, HD, generator=gen, device="cuda").to(torch.bfloat16) for h in (nq, nkv, nkv)]
            entries = [S.Entry(c - 1, 1, t) for c, t in zip(lens, tables)]
            out = torch.full_like(x[0], 7)
            seqs = [host.Sequence_([0] * c, t) for c, t in zip(lens, tables)]
            graphs.step(seqs, [(i, c - 1, 1) for i, c in enumerate(lens)], *x, out)
            torch.cuda.synchronize()
            ws = _bind(entries, nq, nkv, block, mb, max_len)
            eager = torch.full_like(x[0], 7)
            A.g_attn_mgr = mgr
            A.PagedAttentionImpl.execute(0, A.AttnNode(eager, x, layer_id=1))  # the bucket's last layer wrote out
            torch.cuda.synchronize()
            del ws
            # buckets are padded to another batch, so the keys may be split otherwise: the last bit of bf16 may differ
            a, b = out.double().cpu().numpy(), eager.double().cpu().numpy()
            assert np.isfinite(a).all() and (np.abs(a - b) <= 2.0 ** -7 * np.abs(b) + 2.0 ** -8).all()
            _check_error()
    finally:
        graphs.destroy()


def test_large_values_behind_growing_scores(gpu):
    """Values of the largest size that cannot overflow (2^96), with scores that grow along the context: sums against an
    early reference stay finite."""
    for kv4 in (False, True):
        _say("large values", kv4)
        s = Step([(700, 1), (500, 90), (90, 90)], 4, 2, 16, kv4, 0, 0, seed=4, poison=False)
        grow = torch.linspace(0, 3, s.k.shape[0] * 16).view(-1, 1, 16, 1)
        order = torch.argsort(torch.from_numpy(np.concatenate([s.tables[i][:-(-c // 16)] for i, (c, _) in enumerate(s.spec)]
                                                              + [[s.bad]])))
        s.k = (s.k.float() * grow[order]).to(torch.bfloat16)
        s.v = (s.v.float().clamp(-1, 1) * 2.0 ** 96).to(torch.bfloat16)
        s.upload()
        s.prefill(cache.attn_work())
        s.check("prefill")
        d = Step([(700, 1)], 4, 2, 16, kv4, 0, 0, seed=4, poison=False)
        d.k, d.v, d.tables = s.k, s.v, s.tables[:1]
        d.max_blocks = s.max_blocks
        d.upload().decode(cache.attn_work())
        d.check("decode")
