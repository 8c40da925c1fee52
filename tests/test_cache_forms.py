"""CPU: the block manager, what the cache's other entry points refuse, and the tests' own definition of 4-bit pages."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from cache_forms import bf16_values, dequantise, head_bytes, quantise, quantise_fast
from llmgen_amd import attention as A
from llmgen_amd import cache, host
from llmgen_amd._lib import lib


# ------------------------------------------------------------------------------------------ the definition
def test_definition_of_4_bit_rows():
    rng = np.random.default_rng(0)
    bits = rng.integers(0, 1 << 16, (300, 128)).astype(np.uint16)  # every kind of value, infinities and NaN among them
    bits[:200] = (rng.standard_normal((200, 128)) * np.exp(rng.standard_normal((200, 1)) * 8)).astype(np.float32).view(
        np.uint32) >> 16
    bits[200:230] &= 0x80ff  # subnormal and zero
    x = bf16_values(bits)
    a, b = quantise(x), quantise_fast(x)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
    back = dequantise(*a)
    runs, got = x.reshape(-1, 32), back.reshape(-1, 32)
    fine = np.isfinite(runs).all(1)
    assert np.isnan(got[~fine]).all() and (~fine).any()
    # no value is off by more than half the last step of its run's grid, but for runs at the end of the range
    e = a[1].reshape(-1).astype(float) - 127
    inside = fine & (a[1].reshape(-1) < 252)
    assert (np.abs(got - runs)[inside] <= 2.0 ** e[inside, None]).all()
    # values of the grid come back as they are
    again = quantise(np.where(np.isfinite(back), back, 0.0))
    assert np.array_equal(dequantise(*again), np.where(np.isfinite(back), back, 0.0))


def test_page_size():
    L = lib()
    for nkv, block in ((8, 16), (1, 1), (3, 7), (2, 256)):
        assert L.hip_kv4_block_bytes(nkv, 128, block) == nkv * head_bytes(block)
    for bad in ((0, 128, 16), (8, 64, 16), (8, 128, 0), (-1, 128, 16)):
        assert L.hip_kv4_block_bytes(*bad) == 0
    with pytest.raises(ValueError):
        cache.kv4_pool(4, 8, 16, hd=64, device="cpu")
    assert cache.kv4_pool(4, 8, 16, device="cpu").shape == (4, 8 * 1088)


# ------------------------------------------------------------------------------------------ refusals
P = 1 << 20  # an aligned address that no refused call reads


def _refused(capfd, call, *args):
    lib().hip_last_error()
    call(*args)
    assert lib().hip_last_error() != 0
    assert lib().hip_last_error() != 1  # the read cleared it (hipErrorInvalidValue)
    assert "[llmgen-hip]" in capfd.readouterr().err


DECODE = dict(out=P, q=P, kc=P, vc=P, bt=P, ctx=P, S=1, nq=16, nkv=8, hd=128, mb=4, bs=16, scale=0.1, window=8, sinks=4,
              max_ctx=64, work=P, nbytes=1 << 20)
PREFILL = dict(out=P, q=P, kc=P, vc=P, bt=P, ctx=P, cu_q=P, ts=P, tq=P, n_tiles=1, nq=16, nkv=8, hd=128, mb=4, bs=16,
               scale=0.1, window=8, sinks=4, single=-1, work=P, nbytes=1 << 20)
BAD = [dict(out=None), dict(q=None), dict(kc=None), dict(vc=None), dict(bt=None), dict(ctx=None), dict(q=P + 2),
       dict(kc=P + 8), dict(work=P + 4), dict(hd=64), dict(hd=256), dict(nkv=0), dict(nq=0), dict(nq=12), dict(nq=24),
       dict(nq=256), dict(bs=0), dict(mb=0), dict(mb=1 << 26), dict(scale=0.0), dict(scale=-1.0),
       dict(scale=float("nan")), dict(scale=float("inf")), dict(window=-1), dict(sinks=-1)]


@pytest.mark.parametrize("bad", BAD, ids=str)
@pytest.mark.parametrize("name", ["window", "kv4"])
def test_attention_refuses(capfd, name, bad):
    _refused(capfd, getattr(lib(), f"hip_attn_decode_{name}"), *{**DECODE, **bad}.values())
    _refused(capfd, getattr(lib(), f"hip_attn_prefill_{name}"), *{**PREFILL, **bad}.values())


@pytest.mark.parametrize("bad", [dict(cu_q=None), dict(ts=None), dict(tq=None)], ids=str)
@pytest.mark.parametrize("name", ["window", "kv4"])
def test_prefill_refuses(capfd, name, bad):
    _refused(capfd, getattr(lib(), f"hip_attn_prefill_{name}"), *{**PREFILL, **bad}.values())


def test_nothing_to_do_is_not_an_error(capfd):
    lib().hip_last_error()
    for n in (0, -3):
        lib().hip_attn_decode_kv4(*{**DECODE, "S": n, "hd": 1}.values())
        lib().hip_attn_decode_window(*{**DECODE, "S": n, "out": None}.values())
        lib().hip_attn_prefill_kv4(*{**PREFILL, "n_tiles": n, "hd": 1}.values())
        lib().hip_attn_prefill_window(*{**PREFILL, "n_tiles": n, "hd": 1}.values())
        lib().hip_store_kv4(None, None, None, None, None, n, 8, 128, 16)
        lib().hip_load_kv4(None, None, None, None, None, n, 8, 128, 16)
        lib().hip_copy_blocks(None, 1, 16, 4, None, None, n)
    assert "[llmgen-hip]" not in capfd.readouterr().err


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(slots=None), dict(kc=None), dict(vc=None), dict(k=P + 2),
                                 dict(vc=P + 4), dict(hd=64), dict(nkv=0), dict(bs=0), dict(T=1 << 30, nkv=1 << 10)], ids=str)
def test_rows_refuse(capfd, bad):
    args = {**dict(k=P, v=P, slots=P, kc=P, vc=P, T=1, nkv=8, hd=128, bs=16), **bad}
    _refused(capfd, lib().hip_store_kv4, *args.values())
    _refused(capfd, lib().hip_load_kv4, *args.values())


@pytest.mark.parametrize("src, dst", [([0], [4]), ([4], [0]), ([-1], [0]), ([0], [-1]), ([0, 1], [2, 2]), ([0, 2], [2, 3]),
                                      ([1, 0], [0, 2]), ([0, 0], [3, 3])])
def test_copies_refuse_pages(capfd, src, dst):
    pools = (ctypes.c_void_p * 1)(P)
    _refused(capfd, lib().hip_copy_blocks, pools, 1, 64, 4, (ctypes.c_int32 * len(src))(*src),
             (ctypes.c_int32 * len(dst))(*dst), len(src))


@pytest.mark.parametrize("pool, nbytes, blocks", [(None, 64, 4), (P + 8, 64, 4), (P, 0, 4), (P, 24, 4), (P, 64, 0), (P, (1 << 28) + 16, 4)])
def test_copies_refuse_pools(capfd, pool, nbytes, blocks):
    one = (ctypes.c_int32 * 1)
    _refused(capfd, lib().hip_copy_blocks, (ctypes.c_void_p * 1)(pool), 1, nbytes, blocks, one(0), one(1), 1)


@pytest.mark.parametrize("bad", [dict(hd=64), dict(nq=0), dict(nkv=-1), dict(bs=0), dict(kc=P + 8), dict(vc=P + 4), dict(q=P + 2),
                                 dict(out=P + 8)], ids=str)
def test_fused_write_refuses(capfd, bad):
    args = {**dict(out=P, kc=P, vc=P, q=P, k=P, v=P, qw=P, kw=P, eps=1e-6, cos=P, sin=P, pos=P, slots=P, T=1, nq=16, nkv=8, hd=128,
                   bs=16), **bad}
    lib().hip_qk_norm_rope_store_kv4(*args.values())
    assert "hip_qk_norm_rope_store_kv4" in capfd.readouterr().err
    lib().hip_qk_norm_rope_store_kv4(*{**args, "T": 0}.values())
    assert not capfd.readouterr().err


def test_work_init_refuses(capfd):
    _refused(capfd, lib().hip_attn_work_init, None, 1 << 20)
    _refused(capfd, lib().hip_attn_work_init, P + 4, 1 << 20)


def test_block_copies_checks_pools():
    with pytest.raises(ValueError):
        cache.BlockCopies([])
    with pytest.raises(ValueError):  # host memory
        cache.BlockCopies([torch.zeros(4, 64)])


def test_block_copies_takes_whole_numbers():
    ids = cache.BlockCopies._ids
    for good in ([3, 1], (3, 1), np.array([3, 1]), np.array([3, 1], np.uint8), np.array([3, 9, 1], np.int32)[::2], torch.tensor([3, 1])):
        a = ids(good)
        assert a.dtype == np.int32 and a.flags.c_contiguous and a.tolist() == [3, 1]
    assert ids([]).tolist() == []
    for bad in ([0.5], [1 << 32], [-(1 << 31) - 1], np.array([1 << 31]), np.array([1.0]), ["1"]):
        with pytest.raises(ValueError):
            ids(bad)


def test_layer_scratch_is_checked():
    with pytest.raises(ValueError):
        A.PagedAttentionManager().reserve_layer(0, 4, 8, 16, 128, device="cpu", window=4, work=torch.zeros(64)[::2])


def test_forms_are_checked():
    with pytest.raises(ValueError):
        A.PagedAttentionManager().reserve_layer(0, 4, 8, 16, 128, device="cpu", window=-1)
    st = A.PagedAttentionManager().reserve_layer(0, 4, 8, 16, 128, device="cpu", kv4=True, window=7, sinks=2)
    assert st.k.dtype == torch.uint8 and (st.form.kv4, st.form.window, st.form.sinks) == (1, 7, 2)
    st = A.PagedAttentionManager().reserve_layer(0, 4, 8, 16, 128, device="cpu")
    assert st.form is None and st.k.shape == (4, 8, 16, 128)
    step = host.StepState()
    form = host.CacheForm(1, -1, 0, None, 0)
    assert host.L().llmgen_paged_attention_form(ctypes.byref(step), ctypes.byref(form), P, P, P, P, P, P, 1) == -1
    form = host.CacheForm(1, 0, 0, None, 0)
    assert host.L().llmgen_paged_attention_form(ctypes.byref(step), ctypes.byref(form), P, P, None, P, P, P, 1) == -1
    assert host.L().llmgen_paged_attention_form(None, ctypes.byref(form), P, P, P, P, P, P, 1) == -1


# ------------------------------------------------------------------------------------------ the block manager
def test_blocks_alloc_and_free():
    b = host.Blocks(5)
    t = b.alloc(3)
    assert t == [0, 1, 2] and b.free_count == 2
    with pytest.raises(host.OutOfBlocks):
        b.alloc(3)
    assert b.free_count == 2 and b.alloc(0) == []
    b.free([1])
    assert b.alloc(1) == [1]  # the lowest free page
    b.free([-1, 0, -1, 2])
    assert b.free_count == 4 and b.ref(1) == 1 and b.ref(0) == 0
    for bad in ([0], [7], [1, 1], [1, 3]):
        with pytest.raises(ValueError):
            b.free(bad)
        assert b.ref(1) == 1 and b.free_count == 4
    assert b.ref(-1) == -1 and b.ref(5) == -1
    with pytest.raises(ValueError):
        host.Blocks(0)
    with pytest.raises(ValueError):
        b.alloc(-1)
    b.destroy()
    b.destroy()


def test_blocks_fork_and_write():
    b = host.Blocks(6)
    t = b.alloc(2)
    u, w = b.fork(t), b.fork(t)
    assert b.free_count == 4 and b.ref(0) == 3
    assert b.writable(u, 1) == (1, 2) and u == [0, 2] and b.ref(1) == 2 and b.ref(2) == 1
    assert b.writable(u, 1) is None
    b.free(w)
    assert b.writable(t, 1) is None and b.ref(0) == 2  # the last holder writes in place
    with pytest.raises(ValueError):
        b.fork([0, 5])
    assert b.ref(0) == 2
    with pytest.raises(ValueError):
        b.writable(t, 2)
    with pytest.raises(ValueError):
        b.writable([-1], 0)
    b.alloc(b.free_count)
    with pytest.raises(host.OutOfBlocks):
        b.writable(t, 0)
    assert t == [0, 1] and b.ref(0) == 2
    assert b.fork([-1, 0]) == [-1, 0] and b.ref(0) == 3


@pytest.mark.parametrize("seed", range(6))
def test_blocks_compact(seed):
    rng = np.random.default_rng(seed)
    n = int(rng.integers(1, 60))
    b = host.Blocks(n)
    tables = []
    while b.free_count and rng.random() < 0.9:
        tables.append(b.alloc(int(rng.integers(1, b.free_count + 1)) if rng.random() < 0.3 else 1))
    for t in tables[::3]:
        tables.append(b.fork(t))
    keep = []
    for t in tables:
        if rng.random() < 0.5:
            b.free(t)
        else:
            keep.append([-1] + t)
    before, used = [list(t) for t in keep], n - b.free_count
    content = np.arange(n)  # what each page holds
    src, dst = b.compact(keep)
    assert len(set(dst.tolist())) == len(dst) and not set(src.tolist()) & set(dst.tolist())
    after = content.copy()
    after[dst] = content[src]
    for old, new in zip(before, keep):
        assert new[0] == -1 and after[new[1:]].tolist() == content[old[1:]].tolist()
        assert all(0 <= x < used for x in new[1:])
    assert b.free_count == n - used and all((b.ref(i) > 0) == (i < used) for i in range(n))
    assert b.compact(keep)[0].size == 0
    for t in keep:
        b.free(t)
    assert b.free_count == n


def test_compact_that_does_not_fit_changes_nothing():
    b = host.Blocks(8)
    t = b.alloc(8)
    b.free(t[:4])
    buf = (ctypes.c_int32 * 8)()
    assert host.L().llmgen_blocks_compact(b.h, buf, buf, 3) == -1
    assert [b.ref(i) for i in range(8)] == [0, 0, 0, 0, 1, 1, 1, 1]
    a, c = b.compact([t])
    assert a.size == 4 and sorted(c.tolist()) == [0, 1, 2, 3]
