"""Refusals of the packed-batch operators that need no GPU: the C-ABI's
argument checks return before any CUDA call, the module's tensor checks before
any kernel.  The pointers below are never read."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

import capi

P, I, I64 = C.c_void_p, C.c_int, C.c_int64
SOME = 0x1000  # a 16-byte aligned address that no call may touch

INVALID, UNSUPPORTED = -1, -3


def sections(*values):
    return (C.c_int32 * max(1, len(values)))(*values)


def attention(q=SOME, k=SOME, v=SOME, cu=SOME, out=SOME, qs=512, dtype=0, seqs=1, tokens=8, H=4, KVH=2, D=128,
              longest=8, ws=0, ws_bytes=0):
    return capi.lib().memopt_packed_attention(P(q), I64(qs), P(k), I64(256), P(v), I64(256), I(dtype), P(cu), I(seqs),
                                              I64(tokens), I(longest), I(H), I(KVH), I(D), I(0), I(1), P(out), P(ws),
                                              C.c_size_t(ws_bytes), P(0))


def workspace_size(seqs=1, tokens=8, longest=8, H=4, KVH=2, D=128, window=0, causal=1):
    f = capi.lib().memopt_packed_attention_workspace_size
    f.restype = C.c_size_t
    return f(I(seqs), I64(tokens), I(longest), I(H), I(KVH), I(D), I(window), I(causal))


@pytest.mark.parametrize("change,status", [
    (dict(q=0), INVALID), (dict(k=0), INVALID), (dict(v=0), INVALID), (dict(cu=0), INVALID), (dict(out=0), INVALID),
    (dict(q=SOME + 2), INVALID), (dict(out=SOME + 8), INVALID), (dict(qs=516), INVALID), (dict(seqs=-1), INVALID),
    (dict(tokens=-1), INVALID), (dict(H=0), INVALID), (dict(KVH=0), INVALID), (dict(H=5, KVH=2), INVALID),
    (dict(dtype=2), UNSUPPORTED), (dict(D=96), UNSUPPORTED), (dict(D=256), UNSUPPORTED),
    (dict(tokens=2 ** 31), UNSUPPORTED)])
def test_packed_attention_refuses(change, status):
    assert attention(**change) == status
    assert capi.lib().memopt_last_error().decode().startswith("packed_attention:")


def test_packed_attention_workspace():
    """One long prompt of few heads is split along its keys: the workspace is asked for and checked."""
    need = workspace_size(tokens=4000, longest=4000, H=4, KVH=1)
    assert 0 < need <= 256 << 20
    assert workspace_size(tokens=4000, longest=4000, H=64, KVH=64) == 0  # items enough
    assert workspace_size(tokens=100, longest=100) == 0                  # too short
    for bad in (dict(seqs=0), dict(tokens=0), dict(seqs=-1), dict(tokens=-5), dict(H=0), dict(KVH=0), dict(H=5),
                dict(D=96)):
        assert workspace_size(**{**dict(tokens=4000, longest=4000), **bad}) == 0
    long = dict(tokens=4000, longest=4000, H=4, KVH=1)
    assert attention(**long) == -6
    assert attention(**long, ws=SOME, ws_bytes=need - 1) == -6
    assert attention(**long, ws=0, ws_bytes=need) == -6
    assert attention(**long, ws=SOME + 8, ws_bytes=need) == INVALID


@pytest.mark.parametrize("H,KVH", [(1, 1), (4, 1), (32, 8), (5, 5), (128, 1)])
def test_packed_attention_workspace_is_bounded(H, KVH):
    for tokens in (1, 700, 5000, 131072, 2 ** 31 - 1):
        for seqs in (1, 2, 33, 2 ** 20, 2 ** 31 - 1):
            for longest in (0, 1, 5000, 2 ** 31 - 1):
                for window in (0, 1, 4096, 2 ** 31 - 1):
                    for causal in (0, 1):
                        for D in (64, 128):
                            assert workspace_size(seqs, tokens, longest, H, KVH, D, window, causal) <= 256 << 20


def test_packed_attention_of_nothing():
    assert attention(tokens=0, q=0, k=0, v=0, out=0) == 0
    assert attention(seqs=0) == 0


def rotary(q=SOME, k=SOME, v=SOME, qs=512, dtype=0, T=8, H=4, KVH=2, D=128, pos=SOME, axes=1, sec=(64,), freq=SOME,
           pairs=64, qo=SOME, ko=SOME, slots=SOME, kc=SOME, vc=SOME, NB=4, BS=16):
    return capi.lib().memopt_rotary_write_cache(
        P(q), I64(qs), P(k), I64(256), P(v), I64(256), I(dtype), I64(T), I(H), I(KVH), I(D), P(pos), I(axes),
        sections(*sec), P(freq), I(pairs), I(0), P(qo), P(ko), P(slots), P(kc), P(vc), I64(NB), I(BS), P(0))


@pytest.mark.parametrize("change,status", [
    (dict(q=0), INVALID), (dict(k=0), INVALID), (dict(v=0), INVALID), (dict(pos=0), INVALID), (dict(freq=0), INVALID),
    (dict(qo=0), INVALID), (dict(ko=0), INVALID), (dict(kc=0), INVALID), (dict(vc=0), INVALID), (dict(BS=0), INVALID),
    (dict(NB=-1), INVALID), (dict(q=SOME + 4), INVALID), (dict(qs=510), INVALID), (dict(T=-1), INVALID),
    (dict(H=-1), INVALID), (dict(H=0, KVH=0), INVALID), (dict(sec=(63,)), INVALID), (dict(axes=2, sec=(65, -1)), INVALID),
    (dict(axes=2, sec=(40, 40)), INVALID), (dict(axes=0), UNSUPPORTED), (dict(axes=5, sec=(64, 0, 0, 0, 0)), UNSUPPORTED),
    (dict(pairs=60, sec=(60,)), UNSUPPORTED), (dict(pairs=0, sec=(0,)), UNSUPPORTED), (dict(D=64), UNSUPPORTED),
    (dict(D=256), UNSUPPORTED), (dict(dtype=7), UNSUPPORTED)])
def test_rotary_refuses(change, status):
    assert rotary(**change) == status
    assert capi.lib().memopt_last_error().decode().startswith("rotary:")


def test_rotary_of_nothing():
    assert rotary(T=0, q=0, k=0, v=0) == 0


def reserve(tables=SOME, lens=SOME, R=4, MB=8, ring=SOME, NB=32, state=SOME, rows=SOME, new=SOME, B=2, BS=16,
            most=64, cu=SOME, slots=SOME, pos=SOME, bt=SOME, bl=SOME):
    return capi.lib().memopt_reserve_slots(P(tables), P(lens), I(R), I(MB), P(ring), I(NB), P(state), P(rows), P(new),
                                           I(B), I(BS), I64(most), P(cu), P(slots), P(pos), P(bt), P(bl), P(0))


def truncate(tables=SOME, lens=SOME, R=4, MB=8, ring=SOME, NB=32, state=SOME, rows=SOME, keep=SOME, B=2, BS=16):
    return capi.lib().memopt_truncate_rows(P(tables), P(lens), I(R), I(MB), P(ring), I(NB), P(state), P(rows), P(keep),
                                           I(B), I(BS), P(0))


COMMON = [(dict(tables=0), INVALID), (dict(lens=0), INVALID), (dict(ring=0), INVALID), (dict(state=0), INVALID),
          (dict(rows=0), INVALID), (dict(R=0), INVALID), (dict(MB=0), INVALID), (dict(NB=0), INVALID),
          (dict(BS=0), INVALID), (dict(B=-1), INVALID), (dict(B=8193), UNSUPPORTED), (dict(R=2 ** 18 + 1), UNSUPPORTED),
          (dict(NB=2 ** 27), UNSUPPORTED), (dict(MB=2 ** 27), UNSUPPORTED)]


@pytest.mark.parametrize("change,status", COMMON + [
    (dict(new=0), INVALID), (dict(cu=0), INVALID), (dict(slots=0), INVALID), (dict(pos=0), INVALID),
    (dict(bt=0), INVALID), (dict(bl=0), INVALID), (dict(slots=SOME + 4), INVALID), (dict(pos=SOME + 8), INVALID),
    (dict(most=-1), INVALID), (dict(most=2 ** 31), UNSUPPORTED)])
def test_reserve_refuses(change, status):
    assert reserve(**change) == status
    assert capi.lib().memopt_last_error().decode().startswith("reserve_slots:")


@pytest.mark.parametrize("change,status", COMMON)
def test_truncate_refuses(change, status):
    assert truncate(**change) == status
    assert capi.lib().memopt_last_error().decode().startswith("truncate_rows:")


def test_truncate_of_nothing():
    assert truncate(B=0, rows=0, keep=0) == 0


def test_module_refuses_cpu_tensors():
    import memopt_C

    q = torch.zeros(4, 2, 64, dtype=torch.float16)
    i = torch.zeros(4, dtype=torch.int32)
    f = torch.ones(32, dtype=torch.float64)
    pool = torch.zeros(1, 16, 2, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        memopt_C.packed_attention(q, q, q, i, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        memopt_C.apply_rotary(q, q, i, f, [32])
    with pytest.raises(RuntimeError, match="CUDA"):
        memopt_C.rotary_write_cache(q, q, q, i, f, [32], i, pool, pool)
    with pytest.raises(RuntimeError, match="CUDA"):
        memopt_C.reserve_slots(i.reshape(2, 2), i[:2], i, i, i[:1], i[:1], 16, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        memopt_C.truncate_rows(i.reshape(2, 2), i[:2], i, i, i[:1], None, 16)


def test_python_classes_refuse_bad_arguments():
    from memopt import DevicePageTable, RotaryPositions

    for bad in ((0, 16, 1, 1), (1, 0, 1, 1), (1, 16, 0, 1), (1, 16, 1, 0)):
        with pytest.raises(ValueError):
            DevicePageTable(*bad, device="cpu")
    for kw in (dict(rotary_dim=24), dict(rotary_dim=256), dict(rotary_dim=0), dict(sections=[32, 31]),
               dict(sections=[]), dict(sections=[80, -16]), dict(sections=[60, 1, 1, 1, 1]),
               dict(inv_freq=torch.ones(63))):
        with pytest.raises(ValueError):
            RotaryPositions(128, device="cpu", **kw)
    table = DevicePageTable(8, 16, 2, 64, device="cpu")
    with pytest.raises(ValueError):
        table.reserve([0], torch.tensor([3]))
