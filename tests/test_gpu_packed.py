"""Packed-batch operators on the GPU against plain implementations in 64 bits:
attention over packed prompts, rotary positions with the cache write, device
page tables, and the three together as a cache uses them."""
from __future__ import annotations

import math
import random
from collections import deque

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


def C():
    import memopt_C

    return memopt_C


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


# ---- attention over packed prompts -------------------------------------------
def attention_ref(q, k, v, lens, window, causal):
    """(out, sum of p |v|, max |v|) per element, fp64; sequences in order."""
    T, H, D = q.shape
    G = H // k.shape[1]
    out = torch.zeros(T, H, D, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    lo = 0
    for n in lens:
        if n:
            i = torch.arange(n, device=q.device)
            end = i + 1 if causal else torch.full_like(i, n)
            start = (end - window).clamp(min=0) if window > 0 else torch.zeros_like(end)
            hide = (i[None] >= end[:, None]) | (i[None] < start[:, None])
            kk = k[lo:lo + n].double().repeat_interleave(G, 1)
            vv = v[lo:lo + n].double().repeat_interleave(G, 1)
            s = torch.einsum("qhd,khd->hqk", q[lo:lo + n].double(), kk) / math.sqrt(D)
            p = torch.softmax(s.masked_fill(hide[None], float("-inf")), -1)
            out[lo:lo + n] = torch.einsum("hqk,khd->qhd", p, vv)
            mag[lo:lo + n] = torch.einsum("hqk,khd->qhd", p, vv.abs())
        lo += n
    return out, mag


def attention_tol(out, mag, v, n, dtype):
    """u = half a step of the type.  The final rounding is u |out|.  A weight p
    is rounded to the type before P.V and the row sum may add rounded or exact
    weights: 2 u sum p |v|.  Scores are fp32 sums of D products with |s| < 64
    here, 2^-14 on a weight covers them and the exponential.  fp16 weights
    below 2^-14 are subnormal: an absolute 2^-25 each, n of them."""
    u = half_step(dtype)
    tol = u * out.abs() + (2 * u + 2.0 ** -14) * mag + 1e-7
    if dtype == torch.float16:
        tol = tol + n * 2.0 ** -25 * v.abs().max().double()
    return tol


def make_qkv(lens, H, KVH, D, dtype, seed=0, tail=0, fused=False, spread=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    T = sum(lens) + tail
    if fused:
        x = torch.randn(T, H + 2 * KVH, D, generator=g, device=DEV)
        x[:, :H] *= spread
        x = x.to(dtype)
        return x[:, :H], x[:, H:H + KVH], x[:, H + KVH:]
    q = (spread * torch.randn(T, H, D, generator=g, device=DEV)).to(dtype)
    k = torch.randn(T, KVH, D, generator=g, device=DEV).to(dtype)
    v = torch.randn(T, KVH, D, generator=g, device=DEV).to(dtype)
    return q, k, v


def cu_of(lens):
    return torch.tensor([0] + lens, device=DEV).cumsum(0).to(torch.int32)


def check_attention(lens, H, KVH, D, dtype, causal=True, window=-1, fused=False, seed=0, spread=2.0, tail=0,
                    max_seqlen=None):
    q, k, v = make_qkv(lens, H, KVH, D, dtype, seed, tail, fused, spread)
    out = C().packed_attention(q, k, v, cu_of(lens), max(lens) if max_seqlen is None else max_seqlen, window, causal)
    T = sum(lens)
    ref, mag = attention_ref(q[:T], k[:T], v[:T], lens, window, causal)
    err = (out[:T].double() - ref).abs()
    bad = err > attention_tol(ref, mag, v, max(lens), dtype)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {err.max().item():.3g}"


LENGTHS = [[1], [5], [64], [127, 128, 129], [255, 1, 0, 257], [0, 0, 33], [300, 2, 61, 0, 16, 128, 400], [1000],
           [63, 65, 191, 193, 32, 31], [2049, 7]]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens", LENGTHS, ids=str)
def test_attention_lengths(lens, causal):
    check_attention(lens, 4, 2, 128, torch.float16, causal)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,KVH", [(1, 1), (3, 3), (8, 1), (5, 1), (12, 4), (6, 2), (32, 1), (7, 7), (24, 2)])
def test_attention_heads(H, KVH, D, dtype):
    check_attention([150, 1, 77, 300], H, KVH, D, dtype, fused=True, seed=3)


@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 128, 200, 511, 5000])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_window(window, causal):
    check_attention([700, 90, 1, 333], 4, 2, 64, torch.bfloat16, causal, window, seed=5)
    check_attention([700, 90, 1, 333], 4, 4, 128, torch.float16, causal, window, seed=6)


# Long prompts and many heads: the kernel's form with two query tiles an item.
TWO_TILES = [1500, 777, 1, 1300]


@pytest.mark.parametrize("causal,window", [(True, -1), (False, -1), (True, 100), (True, 1000), (False, 300), (True, 1)])
@pytest.mark.parametrize("H,KVH,D,dtype", [(20, 20, 128, torch.float16), (24, 6, 128, torch.bfloat16),
                                           (20, 20, 64, torch.bfloat16), (24, 6, 64, torch.float16),
                                           (40, 8, 128, torch.float16), (64, 4, 64, torch.bfloat16)])
def test_attention_two_tiles(H, KVH, D, dtype, causal, window):
    check_attention(TWO_TILES, H, KVH, D, dtype, causal, window, fused=True, seed=H + D)


@pytest.mark.parametrize("H,KVH,D", [(20, 20, 64), (24, 6, 128)])
def test_attention_two_tiles_hidden_tokens(H, KVH, D):
    """Non-finite values in the two-tile form: rows that do not see them keep
    their result, also where they lie behind a sequence's end."""
    q, k, v = make_qkv(TWO_TILES, H, KVH, D, torch.float16, seed=21, tail=33)
    T = sum(TWO_TILES)
    at = [700, 1500 + 776, T - 1]  # inside a sequence, last of one, last of all
    ref, mag = attention_ref(q[:T], k[:T], v[:T], TWO_TILES, -1, True)
    tol = attention_tol(ref, mag, v, 1500, torch.float16)
    v[at], v[T:] = float("nan"), float("inf")
    out = C().packed_attention(q, k, v, cu_of(TWO_TILES), 1500)
    sees = torch.zeros(T, dtype=torch.bool, device=DEV)
    sees[700:1500], sees[2276], sees[T - 1] = True, True, True
    assert torch.isnan(out[:T][sees].float()).all()
    assert ((out[:T].double() - ref).abs() <= tol)[~sees].all()


def test_attention_scores_of_minus_infinity():
    """A score of -inf weighs nothing; a row with no other score is NaN, as its
    softmax is."""
    n, H, D = 150, 2, 64
    q, k, v = make_qkv([n], H, H, D, torch.float16, seed=22)
    q[:, :, 0] = 1.0
    k[:70, 0, 0] = -float("inf")  # head 0: the first 70 keys
    out = C().packed_attention(q, k, v, cu_of([n]), n)
    assert torch.isnan(out[:70, 0].float()).all()
    kk = k.clone()
    kk[:70, 0, 0] = 0.0
    ref, mag = attention_ref(q, kk, v, [n], -1, True)
    assert ((out.double() - ref).abs() <= attention_tol(ref, mag, v, n, torch.float16))[:, 1].all()
    i = torch.arange(n, device=DEV)
    s = (q[:, 0].double() @ kk[:, 0].double().T / math.sqrt(D))
    s = s.masked_fill((i[None] > i[:, None]) | (i[None] < 70), float("-inf"))
    p = torch.softmax(s, -1)[70:]
    want, size = p @ v[:, 0].double(), p @ v[:, 0].double().abs()
    assert ((out[70:, 0].double() - want).abs() <= attention_tol(want, size, v, n, torch.float16)).all()


def test_attention_long_and_peaked():
    check_attention([5000, 3], 2, 1, 128, torch.float16, seed=7)
    check_attention([3001], 2, 2, 64, torch.bfloat16, seed=8, spread=4.0)  # |s| < 64: q.k/8 of 64 products


def test_attention_rising_scores():
    """Every key scores above all earlier ones: the running maximum moves in each block."""
    n, D = 1500, 128
    q = torch.zeros(n, 1, D, device=DEV, dtype=torch.float16)
    k = torch.zeros_like(q)
    q[:, 0, 0] = 8.0
    k[:, 0, 0] = torch.linspace(-40.0, 40.0, n, device=DEV).half()
    v = torch.randn(n, 1, D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).half()
    for order in (torch.arange(n, device=DEV), torch.arange(n - 1, -1, -1, device=DEV)):
        kk, vv = k[order].contiguous(), v[order].contiguous()
        out = C().packed_attention(q, kk, vv, cu_of([n]), n)
        ref, mag = attention_ref(q, kk, vv, [n], -1, True)
        assert ((out.double() - ref).abs() <= attention_tol(ref, mag, v, n, torch.float16)).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_attention_hidden_tokens_never_reach_a_row(dtype, value):
    """Non-finite keys and values of other sequences, of later tokens and of
    tokens before the window leave the rows that do not see them unchanged."""
    lens, H, KVH, D = [130, 200, 50], 4, 2, 128
    q, k, v = make_qkv(lens, H, KVH, D, dtype, seed=11, tail=40)
    cu = cu_of(lens)
    at = 130 + 120  # a token of the second sequence
    for window in (-1, 40):
        ref, mag = attention_ref(q[:380], k[:380], v[:380], lens, window, True)
        for which in (k, v):
            x = which.clone()
            x[at], x[380:] = value, value  # and the rows behind the last sequence
            kk, vv = (x, v) if which is k else (k, x)
            out = C().packed_attention(q, kk, vv, cu, 200, window, True)
            last = 330 if window < 0 else at + window
            clean = torch.ones(380, dtype=torch.bool, device=DEV)
            clean[at:last] = False
            tol = attention_tol(ref, mag, v, 200, dtype)
            assert ((out[:380].double() - ref).abs() <= tol)[clean].all()
            if which is v:  # the rows that see the value carry it
                assert not torch.isfinite(out[at:last].float()).any()
            elif math.isnan(value):
                assert torch.isnan(out[at:last].float()).all()


def test_attention_leaves_rows_behind_the_last_sequence():
    lens = [100, 29]
    q, k, v = make_qkv(lens, 4, 2, 128, torch.float16, tail=70)
    out = torch.full_like(q, 7.0)
    got = C().packed_attention(q, k, v, cu_of(lens), 100, -1, True, out)
    assert got.data_ptr() == out.data_ptr()
    assert (out[129:] == 7.0).all() and (out[:129] != 7.0).any()
    # sequences need not begin at the first row either
    out.fill_(7.0)
    C().packed_attention(q, k, v, cu_of(lens) + 40, 100, -1, True, out)
    assert (out[:40] == 7.0).all() and (out[169:] == 7.0).all()
    again = C().packed_attention(q[40:169].contiguous(), k[40:169].contiguous(), v[40:169].contiguous(), cu_of(lens),
                                 100)
    assert torch.equal(out[40:169], again)


@pytest.mark.parametrize("hint", [0, 1, 64, 100000])
def test_attention_length_hint_changes_nothing(hint):
    check_attention([300, 70, 513], 4, 2, 128, torch.float16, max_seqlen=hint)


def test_attention_lengths_out_of_range_stay_inside():
    """cu_seqlens is device data that the host cannot check: decreasing or too
    large values must not reach outside the tensors."""
    q, k, v = make_qkv([200], 2, 2, 64, torch.float16)
    out = torch.zeros_like(q)
    C().packed_attention(q, k, v, torch.tensor([0, 120, 60, 500], dtype=torch.int32, device=DEV), 200, -1, True, out)
    torch.cuda.synchronize()
    ref = C().packed_attention(q, k, v, torch.tensor([0, 120], dtype=torch.int32, device=DEV), 200)
    assert torch.equal(out[:60], ref[:60])


# Few rows with many keys: items are split along the keys and joined.
def splits(lens, H, KVH, D, window=-1, causal=True, hint=None):
    import capi

    f = capi.lib().memopt_packed_attention_workspace_size
    f.restype = capi.SZ
    return f(capi.I(len(lens)), capi.I64(sum(lens)), capi.I(max(lens) if hint is None else hint), capi.I(H), capi.I(KVH),
             capi.I(D), capi.I(max(0, window)), capi.I(int(causal)))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,H,KVH,D", [
    ([4000], 4, 1, 128), ([2049], 1, 1, 64), ([2411, 800, 95], 4, 4, 64), ([3, 0, 2300, 1, 129, 0, 640], 2, 2, 128),
    ([1900] + [1] * 40, 4, 2, 64), ([3177, 176], 5, 1, 64), ([5000, 3], 2, 1, 128), ([3301], 8, 1, 64)], ids=str)
def test_attention_split(lens, H, KVH, D, dtype):
    assert splits(lens, H, KVH, D) > 0
    check_attention(lens, H, KVH, D, dtype, fused=True, seed=31, tail=9)


@pytest.mark.parametrize("lens,H,KVH,D,causal,window", [
    ([1200], 4, 4, 128, False, -1), ([2500, 1, 300], 4, 1, 64, False, -1), ([1500], 2, 2, 128, False, 1300),
    ([3000], 2, 1, 64, True, 2000), ([2600, 0, 77], 1, 1, 128, True, 1801), ([4100, 64], 2, 1, 128, True, 1665)], ids=str)
def test_attention_split_windows_and_all_keys(lens, H, KVH, D, causal, window):
    assert splits(lens, H, KVH, D, window, causal) > 0
    check_attention(lens, H, KVH, D, torch.float16, causal, window, seed=32)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,H,KVH,D,window", [
    ([2500, 5, 7, 0, 20, 1], 16, 4, 128, -1), ([5000], 8, 4, 64, -1), ([2700], 16, 4, 128, 2300),
    ([2600, 2599], 8, 4, 64, -1), ([2500], 32, 8, 64, -1)], ids=str)
def test_attention_tiles_past_a_round_are_split(lens, H, KVH, D, window, dtype):
    """Not causal, a little more than one or two items for every slot: the last tiles are split, the others whole."""
    assert splits(lens, H, KVH, D, window, False) > 0
    check_attention(lens, H, KVH, D, dtype, False, window, seed=35, tail=7)
    shorter = [max(0, n - 700) for n in lens] + [700 * sum(n > 700 for n in lens)]
    check_attention(shorter, H, KVH, D, dtype, False, window, seed=36, max_seqlen=max(lens))


@pytest.mark.parametrize("hint", [900, 2600, 6000, 2 ** 31 - 1])
def test_attention_split_with_another_length_hint(hint):
    """The hint and the true lengths give different pieces: more, fewer or empty ones."""
    for lens in ([2600], [1300, 1300], [2, 2500, 98], [40] * 65):
        check_attention(lens, 2, 1, 128, torch.float16, max_seqlen=hint, seed=33)


def test_attention_split_non_finite():
    lens, H, KVH, D = [2500, 300], 2, 2, 64
    assert splits(lens, H, KVH, D) > 0
    q, k, v = make_qkv(lens, H, KVH, D, torch.float16, seed=34, tail=33)
    T = sum(lens)
    ref, mag = attention_ref(q[:T], k[:T], v[:T], lens, -1, True)
    tol = attention_tol(ref, mag, v, 2500, torch.float16)
    for value in (float("nan"), float("inf"), -float("inf")):
        for which in (0, 1):
            kk, vv = k.clone(), v.clone()
            (kk, vv)[which][[1700, T - 1]], (kk, vv)[which][T:] = value, value
            out = C().packed_attention(q, kk, vv, cu_of(lens), 2500)
            sees = torch.zeros(T, dtype=torch.bool, device=DEV)
            sees[1700:2500], sees[T - 1] = True, True
            assert ((out[:T].double() - ref).abs() <= tol)[~sees].all()
            if which == 1:
                assert not torch.isfinite(out[:T][sees].float()).any()
    # One dim of one value: the others keep their result.
    vv = v.clone()
    vv[1700, 0, 5] = float("nan")
    out = C().packed_attention(q, k, vv, cu_of(lens), 2500)[:T]
    hit = torch.zeros(T, H, D, dtype=torch.bool, device=DEV)
    hit[1700:2500, 0, 5] = True
    assert torch.isnan(out[hit].float()).all()
    assert ((out.double() - ref).abs() <= tol)[~hit].all()


def test_attention_split_rising_and_hidden_scores():
    """Pieces whose maxima lie far apart, and rows that see nothing in a piece's masked part."""
    n, D = 2500, 128
    q = torch.zeros(n, 1, D, device=DEV, dtype=torch.float16)
    k = torch.zeros_like(q)
    q[:, 0, 0] = 8.0
    k[:, 0, 0] = torch.linspace(-40.0, 40.0, n, device=DEV).half()
    v = torch.randn(n, 1, D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2)).half()
    for order in (torch.arange(n, device=DEV), torch.arange(n - 1, -1, -1, device=DEV)):
        for window in (-1, 1500):
            assert splits([n], 1, 1, D, window) > 0
            kk, vv = k[order].contiguous(), v[order].contiguous()
            out = C().packed_attention(q, kk, vv, cu_of([n]), n, window)
            ref, mag = attention_ref(q, kk, vv, [n], window, True)
            assert ((out.double() - ref).abs() <= attention_tol(ref, mag, v, n, torch.float16)).all()


def test_attention_split_same_bits_and_leaves_the_rest():
    lens = [2222, 0, 5]
    q, k, v = make_qkv(lens, 4, 2, 128, torch.bfloat16, fused=True, tail=60)
    cu, out = cu_of(lens), torch.full((2287, 4, 128), 3.0, dtype=torch.bfloat16, device=DEV)
    C().packed_attention(q, k, v, cu, 2222, -1, True, out)
    assert (out[2227:] == 3.0).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    both = []
    for _ in range(4):  # two streams at once, each with its own workspace
        both.append(C().packed_attention(q, k, v, cu, 2222))
        with torch.cuda.stream(side):
            both.append(C().packed_attention(q, k, v, cu, 2222))
    torch.cuda.synchronize()
    assert all(torch.equal(o[:2227], out[:2227]) for o in both)


def test_attention_split_in_graphs_with_new_lengths():
    q, k, v = make_qkv([2600], 2, 1, 128, torch.float16)
    cu = cu_of([2600, 0, 0])
    outs, graphs = [torch.zeros_like(q) for _ in range(2)], [torch.cuda.CUDAGraph() for _ in range(2)]
    C().packed_attention(q, k, v, cu, 2600)  # warm-up
    for out, graph in zip(outs, graphs):
        with torch.cuda.graph(graph):
            C().packed_attention(q, k, v, cu, 2600, -1, True, out)
    for lens in ([2600, 0, 0], [0, 2599, 1], [700, 1000, 900], [1, 1, 1], [0, 0, 0]):
        cu.copy_(cu_of(lens))
        T = sum(lens)
        ref, mag = attention_ref(q[:T], k[:T], v[:T], lens, -1, True)
        for out, graph in zip(outs, graphs):
            out.zero_()
            graph.replay()
        for out in outs:
            if T:
                assert ((out[:T].double() - ref).abs() <= attention_tol(ref, mag, v, max(lens), torch.float16)).all()
            assert (out[T:] == 0).all()


def test_attention_split_lengths_out_of_range_stay_inside():
    q, k, v = make_qkv([2600], 2, 2, 64, torch.float16)
    for cu in ([0, 2000, 600, 5000], [-5, 2600, 0, 2600], [2600, 2600, 3, 2600], [0, 2 ** 31 - 1, -2 ** 31, 7]):
        C().packed_attention(q, k, v, torch.tensor(cu, dtype=torch.int32, device=DEV), 2600)
    torch.cuda.synchronize()
    check_attention([2600], 2, 2, 64, torch.float16)


def test_attention_many_sequences():
    rng = random.Random(0)
    lens = [rng.choice([0, 1, 2, 3, 7, 20, 33]) for _ in range(1500)]
    check_attention(lens, 2, 1, 64, torch.float16, seed=13)


def test_attention_same_bits_again_and_on_another_stream():
    lens = [500, 3, 130]
    q, k, v = make_qkv(lens, 8, 2, 128, torch.bfloat16, fused=True)
    cu = cu_of(lens)
    ref = C().packed_attention(q, k, v, cu, 500)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [C().packed_attention(q, k, v, cu, 500) for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(o, ref) for o in outs)


def test_attention_in_a_graph_with_new_lengths():
    q, k, v = make_qkv([600], 4, 4, 128, torch.float16)
    cu = cu_of([100, 200, 300])
    out = torch.zeros_like(q)
    C().packed_attention(q, k, v, cu, 600, -1, True, out)  # warm-up
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        C().packed_attention(q, k, v, cu, 600, -1, True, out)
    for lens in ([100, 200, 300], [0, 599, 1], [600, 0, 0], [1, 1, 1]):
        cu.copy_(cu_of(lens))
        out.zero_()
        graph.replay()
        T = sum(lens)
        ref, mag = attention_ref(q[:T], k[:T], v[:T], lens, -1, True)
        assert ((out[:T].double() - ref).abs() <= attention_tol(ref, mag, v, max(lens), torch.float16)).all()
        assert (out[T:] == 0).all()


# ---- rotary positions ----------------------------------------------------------
def rotary_ref(x, pos, freq, sections, interleaved):
    """(turned, |x| + |y| of the pair) in fp64."""
    P = freq.numel()
    axis = torch.repeat_interleave(torch.arange(len(sections), device=DEV), torch.tensor(sections, device=DEV))
    a = (pos.double().reshape(len(sections), -1)[axis].T * freq[None])[:, None]  # [T, 1, P]
    y, m = x.double().clone(), x.double().abs()
    one = torch.arange(P, device=DEV) * (2 if interleaved else 1)
    two = one + 1 if interleaved else one + P
    u, w = x.double()[..., one], x.double()[..., two]
    y[..., one], y[..., two] = u * a.cos() - w * a.sin(), u * a.sin() + w * a.cos()
    m[..., one] = m[..., two] = u.abs() + w.abs()
    return y, m


def rotary_close(got, ref, mag):
    """Half a step of the type, plus fp32 arithmetic: the angle is off by at
    most pi 2^-24, cos and sin by 2 ulp and two products and a sum round:
    below 2^-20 of |x| + |y|; fp16 subnormals 2^-25."""
    tol = half_step(got.dtype) * ref.abs() + 2.0 ** -20 * mag + 2.0 ** -25
    return bool(((got.double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,H,KVH,D,P,sections,interleaved", [
    (1, 32, 8, 128, 64, [64], False), (1, 1, 1, 64, 32, [32], True), (33, 32, 8, 128, 64, [16, 24, 24], False),
    (700, 5, 1, 64, 24, [10, 14], True), (257, 3, 3, 128, 8, [8], False), (64, 40, 8, 128, 48, [1, 0, 40, 7], True),
    (5000, 8, 2, 64, 32, [32], False), (19, 7, 7, 64, 16, [3, 13], False)])
def test_rotary(T, H, KVH, D, P, sections, interleaved, dtype):
    g = torch.Generator(device=DEV).manual_seed(T)
    x = torch.randn(T, H + 2 * KVH, D, generator=g, device=DEV).to(dtype)
    q, k, v = x[:, :H], x[:, H:H + KVH], x[:, H + KVH:]
    pos = torch.randint(-(1 << 20), 1 << 24, (len(sections), T), generator=g, device=DEV, dtype=torch.int32)
    pos[:, 0] = torch.tensor([0, 2 ** 31 - 1, -2 ** 31, 131071][:len(sections)], dtype=torch.int32, device=DEV)
    freq = 500000.0 ** (-torch.arange(P, device=DEV, dtype=torch.float64) / P)
    q2, k2 = C().apply_rotary(q, k, pos, freq, sections, interleaved)
    assert rotary_close(q2, *rotary_ref(q, pos, freq, sections, interleaved))
    assert rotary_close(k2, *rotary_ref(k, pos, freq, sections, interleaved))
    assert torch.equal(q2[..., 2 * P:], q[..., 2 * P:])  # the rest of the head passes through
    # the same with the cache write: shuffled slots, some tokens without one
    BS = 16
    NB = T // BS + 4
    kc = torch.full((NB, BS, KVH, D), 3.0, dtype=torch.float16, device=DEV)
    vc = kc.clone()
    slots = torch.randperm(NB * BS, generator=g, device=DEV)[:T].to(torch.int32)
    if T > 4:
        slots[2], slots[3], slots[4] = -1, NB * BS, 2 ** 31 - 1
    q3, k3 = C().rotary_write_cache(q, k, v, pos, freq, sections, slots, kc, vc, interleaved)
    assert torch.equal(q3, q2) and torch.equal(k3, k2)
    ok = (slots >= 0) & (slots < NB * BS)
    at = slots[ok].long()
    ref, mag = rotary_ref(k, pos, freq, sections, interleaved)
    assert rotary_close(kc.view(-1, KVH, D)[at], ref[ok], mag[ok])
    assert torch.equal(vc.view(-1, KVH, D)[at], v[ok].half())
    rest = torch.ones(NB * BS, dtype=torch.bool, device=DEV)
    rest[at] = False
    assert (kc.view(-1, KVH, D)[rest] == 3.0).all() and (vc.view(-1, KVH, D)[rest] == 3.0).all()


def test_rotary_relative_positions():
    """Turned by p and by p + s, a pair's inner product depends on s alone."""
    D, P = 128, 64
    freq = 10000.0 ** (-torch.arange(P, device=DEV, dtype=torch.float64) / P)
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(1, 1, D, generator=g, device=DEV).half().expand(64, 1, D).contiguous()
    y = torch.randn(1, 1, D, generator=g, device=DEV).half().expand(64, 1, D).contiguous()
    pos = torch.arange(64, device=DEV, dtype=torch.int32) * 65521
    a, _ = C().apply_rotary(x, x, pos, freq, [P])
    b, _ = C().apply_rotary(y, y, pos + 17, freq, [P])
    dots = (a.double() * b.double()).sum(-1)
    # two fp16 roundings of each of D products
    assert (dots - dots[0]).abs().max() <= 4 * 2.0 ** -11 * (a.double() * b.double()).abs().sum(-1).max()


# ---- device page tables -----------------------------------------------------------
class Host:
    """The same bookkeeping on the host: a FIFO of pages and a list per row."""

    def __init__(self, NB, BS, R, MB):
        self.NB, self.BS, self.R, self.MB = NB, BS, R, MB
        self.free = deque(range(NB))
        self.pages = [[] for _ in range(R)]
        self.lens = [0] * R

    def need(self, tokens):
        return -(-tokens // self.BS)

    def refusal(self, rows, new, cap):
        if len(set(rows)) < len(rows) or any(not 0 <= r < self.R for r in rows):
            return 4
        if any(n < 0 for n in new) or sum(new) > cap:
            return 8
        if any(self.need(self.lens[r] + n) > self.MB for r, n in zip(rows, new)):
            return 2
        if sum(self.need(self.lens[r] + n) - len(self.pages[r]) for r, n in zip(rows, new)) > len(self.free):
            return 1
        return 0

    def reserve(self, rows, new):
        slots, pos = [], []
        for r, n in zip(rows, new):
            while len(self.pages[r]) < self.need(self.lens[r] + n):
                self.pages[r].append(self.free.popleft())
            for t in range(self.lens[r], self.lens[r] + n):
                slots.append(self.pages[r][t // self.BS] * self.BS + t % self.BS)
                pos.append(t)
            self.lens[r] += n
        return slots, pos

    def truncate(self, rows, keep):
        for r, n in zip(rows, keep):
            m = self.need(n)
            self.free.extend(self.pages[r][m:])
            self.pages[r] = self.pages[r][:m]
            self.lens[r] = n

    def same(self, table):
        head, count, status, ticket = table.pool_state.tolist()
        assert (status, ticket) == (0, 0)
        ring = table.free_pages.tolist()
        assert [ring[(head + i) % self.NB] for i in range(count)] == list(self.free)
        assert table.context_lens.tolist() == self.lens
        assert table.block_tables.tolist() == [p + [-1] * (self.MB - len(p)) for p in self.pages]


@pytest.mark.parametrize("NB,BS,R,width,batch,most", [(64, 16, 8, 7, 5, 40), (5000, 16, 300, 300, 280, 300),
                                                     (900, 32, 3, 300, 2, 6000), (40, 1, 9, 11, 4, 3),
                                                     (20000, 16, 1200, 40, 1100, 60)])
def test_page_table_against_the_host(NB, BS, R, width, batch, most):
    from memopt import DevicePageTable

    rng = random.Random(NB)
    host, table = Host(NB, BS, R, width), DevicePageTable(NB, BS, R, width * BS)
    refused = 0
    for step in range(30):
        rows = rng.sample(range(R), rng.randint(0, batch))
        new = [rng.choice([0, 1, 1, rng.randint(0, most)]) for _ in rows]
        cap = sum(new) + rng.choice([0, 0, 1, 70])
        why = host.refusal(rows, new, cap)
        got = table.reserve(rows, new, cap)
        if why:
            refused += 1
            assert table.pool_state[2].item() == why
            with pytest.raises(MemoryError if why == 1 else RuntimeError):
                table.check()
            assert (got.slot_mapping == -1).all() and (got.cu_seqlens == 0).all()
            slots, pos, new = [], [], [0] * len(rows)
        else:
            slots, pos = host.reserve(rows, new)
            assert got.cu_seqlens.tolist() == [sum(new[:i]) for i in range(len(new) + 1)]
        pad = cap - len(slots)
        assert got.slot_mapping.tolist() == slots + [-1] * pad
        assert got.positions.tolist() == pos + [0] * pad
        assert got.context_lens.tolist() == [host.lens[r] for r in rows]
        assert got.block_tables.tolist() == [host.pages[r] + [-1] * (width - len(host.pages[r])) for r in rows]
        host.same(table)
        rows = rng.sample(range(R), rng.randint(0, R // 2))
        keep = [rng.choice([0, host.lens[r], rng.randint(0, host.lens[r])]) for r in rows]
        if rng.random() < 0.3:
            keep = [0] * len(rows)
            table.truncate(rows)
        else:
            table.truncate(rows, keep)
        host.truncate(rows, keep)
        host.same(table)
    assert refused < 30


def test_page_table_takes_pages_as_the_host_table_does():
    from memopt import DevicePageTable, PageTable

    free = deque(range(50))
    host = PageTable(16, lambda: free.popleft() if free else -1, free.append)
    table = DevicePageTable(50, 16, 4, 400)
    ids = [host.add_sequence() for _ in range(4)]
    for new in ([30, 1, 0, 16], [2, 15, 1, 1], [100, 17, 33, 0]):
        want = [s for i, n in zip(ids, new) for s in host.reserve(i, n)]
        assert table.reserve(range(4), new).slot_mapping.tolist() == want
    assert table.block_tables.tolist() == host.block_table(ids, 25)
    table.check()


def test_page_table_refusals_change_nothing():
    from memopt import DevicePageTable

    table = DevicePageTable(10, 16, 4, 96)  # six pages a row
    table.reserve([0, 2], [20, 90])
    before = [t.clone() for t in (table.block_tables, table.context_lens, table.free_pages, table.pool_state[:2])]
    calls = [(lambda: table.reserve([1, 1], [1, 1]), 4), (lambda: table.reserve([4], [1]), 4),
             (lambda: table.reserve([-1], [1]), 4), (lambda: table.reserve([0], [-3], 5), 8),
             (lambda: table.reserve([0, 1], [9, 9], 17), 8), (lambda: table.reserve([2], [7]), 2),
             (lambda: table.reserve([1, 3], [17, 1]), 1), (lambda: table.truncate([0, 0]), 4),
             (lambda: table.truncate([0], [21]), 8), (lambda: table.truncate([0], [-1]), 8),
             (lambda: table.truncate([7]), 4),
             (lambda: table.reserve([0, 1], [2 ** 31 - 1, 2 ** 31 - 1], 64), 2 + 8)]
    for call, why in calls:
        call()
        assert table.pool_state[2].item() & why
        with pytest.raises((MemoryError, RuntimeError)):
            table.check()
        after = [table.block_tables, table.context_lens, table.free_pages, table.pool_state[:2]]
        assert all(torch.equal(a, b) for a, b in zip(before, after))
    table.reserve([1], [1])
    table.check()


def test_page_table_with_damaged_state():
    """Values that no call writes (a foreign page in the ring or a row, a length
    past the table) are reported and never become a slot."""
    from memopt import DevicePageTable

    table = DevicePageTable(10, 16, 3, 96)
    table.free_pages[1] = 4711
    table.free_pages[2] = -5
    batch = table.reserve([0], [50])  # pages 0, 4711, -5, 3
    assert batch.slot_mapping.tolist() == list(range(16)) + [-1] * 32 + [48, 49]
    with pytest.raises(RuntimeError, match="out of range"):
        table.check()
    batch = table.reserve([0], [1])
    assert batch.slot_mapping.tolist() == [50]
    table.check()
    table.truncate([0], [20])  # gives -5 and 3 back, reports the first
    assert table.free_count() == 8
    with pytest.raises(RuntimeError, match="out of range"):
        table.check()
    for bad in (-1, 97):
        table.context_lens[1] = bad
        before = table.pool_state[:2].clone()
        batch = table.reserve([1], [1])
        assert batch.slot_mapping.tolist() == [-1] and torch.equal(table.pool_state[:2], before)
        with pytest.raises(RuntimeError, match="out of range"):
            table.check()
    table.context_lens[1] = 0
    for head, count in ((-1, 3), (10, 3), (0, 11), (0, -1)):
        table.pool_state[0], table.pool_state[1] = head, count
        assert table.reserve([1], [1]).slot_mapping.tolist() == [-1]
        table.truncate([2])
        assert table.pool_state.tolist() == [head, count, 16, 0]
        with pytest.raises(RuntimeError):
            table.check()


def test_page_table_step_in_a_graph():
    """A captured decode step: one token per row, replayed; half of the rows are cut back in between."""
    from memopt import DevicePageTable

    host, table = Host(400, 16, 6, 60), DevicePageTable(400, 16, 6, 960)
    rows = torch.arange(6, dtype=torch.int32, device=DEV)
    one = torch.ones_like(rows)
    args = (table.block_tables, table.context_lens, table.free_pages, table.pool_state, rows, one, 16, 8)
    C().reserve_slots(*args)
    host.reserve(range(6), [1] * 6)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cu, slots, pos, tables, lens = C().reserve_slots(*args)
    for step in range(40):
        graph.replay()
        want, at = host.reserve(range(6), [1] * 6)
        assert slots.tolist() == want + [-1, -1] and pos.tolist() == at + [0, 0]
        assert lens.tolist() == host.lens
        if step % 7 == 3:
            table.truncate([1, 3, 5], [3, 0, 1])
            host.truncate([1, 3, 5], [3, 0, 1])
    host.same(table)


# ---- together -----------------------------------------------------------------------
@pytest.mark.parametrize("kv_format", ["fp16", "int4"])
def test_cache_prompt_decode_draft_evict(kv_format):
    """Prompts of different lengths, decode steps, rejected drafts, a finished
    row and an exact eviction: attention stays that over the tokens that are
    cached (read back from the pool) and no page is lost."""
    from memopt import PackedKVCache, RotaryPositions

    H, KVH, D, BS = 8, 2, 128, 16
    rot = RotaryPositions(D, sections=[16, 24, 24])
    cache = PackedKVCache(200, KVH, D, BS, max_seqs=4, max_seq_len=640, kv_format=kv_format, rotary=rot)
    g = torch.Generator(device=DEV).manual_seed(2)

    def tokens(n):
        x = torch.randn(n, H + 2 * KVH, D, generator=g, device=DEV).half()
        return x[:, :H], x[:, H:H + KVH], x[:, H + KVH:]

    lens = [70, 1, 300]
    batch = cache.admit([0, 3, 1], lens)
    q, k, v = tokens(371)
    grid = torch.randint(0, 50, (3, 371), generator=g, device=DEV, dtype=torch.int32)
    out = cache.prompt(q, k, v, batch, 300, positions=grid)
    q64, _ = rotary_ref(q, grid, rot.inv_freq, rot.sections, False)
    k64, _ = rotary_ref(k, grid, rot.inv_freq, rot.sections, False)
    ref, mag = attention_ref(q64, k64, v, lens, -1, True)
    # q and k are rounded to fp16: half a step of each of the products of a score
    size = (q64.abs().amax() * k64.abs().amax() * math.sqrt(D)).item()
    assert ((out.double() - ref).abs() <= attention_tol(ref, mag, v, 300, torch.float16) +
            2.0 ** -10 * min(size, 64.0) * mag).all()

    if kv_format == "int4":  # the turned keys are what the pool holds, to half a step of their group's scale
        kcodes, kscale, _, _ = C().get_int4_pool_tensors()
        for i, row in enumerate([0, 3, 1]):
            n, first = lens[i], sum(lens[:i])
            pages = cache.table.block_tables[row, : -(-n // BS)].long()
            c = kcodes[pages].transpose(1, 2).reshape(-1, KVH, D // 2)[:n].long()
            codes = torch.stack([c & 15, c >> 4], -1).reshape(n, KVH, D) - 8
            scale = kscale[pages].transpose(1, 2).reshape(-1, KVH, D // 64)[:n].double().repeat_interleave(64, -1)
            key = k64[first:first + n]
            # half a step, the fp16 rounding of the key and that of the scale (7 steps of it)
            tol = scale * (0.5 + 7 * 2.0 ** -11) + 2.0 ** -11 * key.abs() + 1e-6
            assert ((codes * scale - key).abs() <= tol).all()

    def rows_of(row):  # this row's cached keys and values [n, KVH, D]
        n = int(cache.table.context_lens[row])
        pages = cache.table.block_tables[row, : -(-n // BS)].long()
        return [c[pages].reshape(-1, KVH, D)[:n].double() for c in C().get_pool_tensors()]

    def step(n):
        batch = cache.extend([0, 1, 3], n)
        q, k, v = tokens(3 * n)
        out = cache.decode(q, k, v, batch)
        if kv_format == "fp16":
            pos = batch.positions.expand(3, -1)
            q64, _ = rotary_ref(q, pos, rot.inv_freq, rot.sections, False)
            for i, row in enumerate([0, 1, 3]):
                kk, vv = rows_of(row)
                m = kk.shape[0]
                full = torch.zeros(m, H, D, dtype=torch.float64, device=DEV)
                full[m - n:] = q64[i * n:(i + 1) * n].half().double()
                ref, mag = attention_ref(full, kk, vv, [m], -1, True)
                err = (out[i * n:(i + 1) * n].double() - ref[m - n:]).abs()
                assert (err <= 2e-3 + 1e-2 * ref[m - n:].abs()).all()  # the paged kernels' own tolerance
        assert torch.isfinite(out.float()).all()
        return batch

    for _ in range(20):
        step(1)
    step(4)
    cache.table.truncate([0, 1, 3], [91, 321, 22])  # three of four drafts rejected
    step(1)
    assert cache.table.context_lens.tolist() == [92, 322, 0, 23]
    cache.finish([3])
    scores = torch.rand(4, KVH, 322, generator=g, device=DEV)
    kept, count = cache.evict(scores, 0.5)
    assert count.tolist() == [46, 161, 0, 0]
    batch = cache.extend([0, 1])
    q, k, v = tokens(2)
    assert torch.isfinite(cache.decode(q, k, v, batch).float()).all()
    assert cache.table.context_lens.tolist() == [47, 162, 0, 0]
    cache.finish([0, 1])
    cache.table.check()
    assert cache.table.free_count() == 200
    assert sorted(cache.table.free_pages.tolist()) == list(range(200))


def test_layer_forward_packed_matches_each_prompt_alone():
    """A layer over a packed batch gives what it gives to each prompt alone
    (dense fp64 attention of the fp16 projections), then decodes."""
    from memopt import DynamicAttention, PackedKVCache

    torch.manual_seed(0)
    layer = DynamicAttention(256, 4).half().to(DEV)
    cache = PackedKVCache(64, 4, 64, 16, max_seqs=3, max_seq_len=256)
    lens = [37, 5, 130]
    x = torch.randn(sum(lens), 256, device=DEV).half()
    y = layer.forward_packed(x, cache, cache.admit([2, 0, 1], lens), 130)
    q, k, v = (p(x).detach().reshape(-1, 4, 64) for p in (layer.q_proj, layer.k_proj, layer.v_proj))
    ref, mag = attention_ref(q, k, v, lens, -1, True)
    w = layer.out_proj.weight.detach().double()
    want = ref.reshape(-1, 256) @ w.T
    # the attention's own tolerance through |w|, the rounding of the product's
    # result and of its fp32 sums of 256 terms
    tol = attention_tol(ref, mag, v, 130, torch.float16).reshape(-1, 256) @ w.abs().T
    tol = tol + 2.0 ** -11 * want.abs() + 2.0 ** -15 * (ref.reshape(-1, 256).abs() @ w.abs().T) + 2.0 ** -25
    assert ((y.detach().double() - want).abs() <= tol).all()
    assert y.requires_grad  # the output projection still trains; the attention does not
    step = layer.forward_packed(torch.randn(3, 256, device=DEV).half(), cache, cache.extend([2, 0, 1]))
    assert step.shape == (3, 256) and torch.isfinite(step.float()).all()
    assert cache.table.context_lens.tolist() == [6, 131, 38]
    with pytest.raises(ValueError):
        layer.forward_packed(x, cache, cache.admit([0], [1]))
    cache.table.check()


def test_whole_step_in_a_graph():
    """Reserve, rotary with the cache write and paged decode captured once and
    replayed step by step give what the same calls give one by one."""
    from memopt import DevicePageTable, RotaryPositions

    H, KVH, D, BS, B = 4, 2, 64, 16, 3
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(B, H + 2 * KVH, D, generator=g, device=DEV).half()
    rot = RotaryPositions(D)
    rows = torch.tensor([2, 0, 1], dtype=torch.int32, device=DEV)
    one = torch.ones_like(rows)

    def fresh():
        table = DevicePageTable(40, BS, B, 160)
        pools = [torch.zeros(40, BS, KVH, D, dtype=torch.float16, device=DEV) for _ in range(2)]
        return table, pools

    def step(table, pools):
        b = table.reserve(rows, one, B)
        q, _ = rot.write(x[:, :H], x[:, H:H + KVH], x[:, H + KVH:], b.positions, b.slot_mapping, *pools)
        return C().dynamic_sparse_attention(q[:, None], *pools, b.block_tables, b.context_lens, 160, 160, True)

    table, pools = fresh()
    plain = [step(table, pools).clone() for _ in range(20)]
    table2, pools2 = fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*fresh())  # warm-up on the capture stream: its attention workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step(table2, pools2)
        for want in plain:
            graph.replay()
            assert torch.equal(out, want)
    side.synchronize()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(pools, pools2))
    assert torch.equal(table.block_tables, table2.block_tables)
    table2.check()


def test_calls_back_to_back_wait_for_each_other():
    """Each kernel may begin before the one ahead of it has ended, but reads its
    results: chains without a synchronisation give what they give with one."""
    from memopt import DevicePageTable, RotaryPositions

    lens = [300, 5, 900, 33]
    q, k, v = make_qkv(lens, 8, 8, 64, torch.bfloat16, seed=9, spread=1.0)
    cu, rot = cu_of(lens), RotaryPositions(64)
    pos = torch.arange(sum(lens), dtype=torch.int32, device=DEV)

    def chain(after):
        a, b, x = q, k, v
        for _ in range(12):
            a, b = rot.apply(a, b, pos)
            after()
            x = C().packed_attention(a, b, x, cu, 900)
            after()
        return a, b, x

    want = chain(torch.cuda.synchronize)
    for _ in range(5):
        assert all(torch.equal(g, w) for g, w in zip(chain(lambda: None), want))

    rng = random.Random(1)
    host, table = Host(3000, 16, 40, 90), DevicePageTable(3000, 16, 40, 1440)
    plan = []
    for _ in range(150):
        rows = rng.sample(range(40), 20)
        new = [rng.randint(0, 60) if host.lens[r] < 1300 else 0 for r in rows]
        want = host.reserve(rows, new)
        cut = rng.sample(range(40), 10)
        keep = [rng.randint(0, host.lens[r]) for r in cut]
        host.truncate(cut, keep)
        plan.append(([table.ints(z) for z in (rows, new, cut, keep)], sum(new), want))
    torch.cuda.synchronize()
    got = []
    for (rows, new, cut, keep), n, _ in plan:
        got.append(table.reserve(rows, new, n))
        table.truncate(cut, keep)
    host.same(table)
    for batch, (_, _, want) in zip(got, plan):
        assert (batch.slot_mapping.tolist(), batch.positions.tolist()) == want


def test_two_streams_at_once():
    """Two batches in flight on two streams do not disturb each other."""
    sets = [make_qkv([700, 40, 300], 8, 2, 128, torch.float16, seed=s) for s in (1, 2)]
    cu = cu_of([700, 40, 300])
    want = [C().packed_attention(*s, cu, 700) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(C().packed_attention(*sets[i], cu, 700))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in (0, 1) for o in got[i])


def test_offsets_past_32_bits():
    """Rows, outputs and slots beyond 2^31 elements."""
    H, D, T = 64, 128, 270000  # 2.2e9 elements
    q = torch.zeros(T, H, D, dtype=torch.float16, device=DEV)
    k = torch.zeros(T, 2, D, dtype=torch.float16, device=DEV)
    v = torch.zeros_like(k)
    lens = [300, 1, 129]
    n = sum(lens)
    a, b, c = make_qkv(lens, H, 2, D, torch.float16, seed=4)
    q[-n:], k[-n:], v[-n:] = a, b, c
    out = torch.zeros_like(q)
    C().packed_attention(q, k, v, cu_of(lens) + (T - n), 300, -1, True, out)
    assert torch.equal(out[-n:], C().packed_attention(a, b, c, cu_of(lens), 300))
    assert not out[:4].any() and not out[T // 2: T // 2 + 4].any()
    del out
    freq = 10000.0 ** (-torch.arange(64, device=DEV, dtype=torch.float64) / 64)
    pos = torch.arange(T, device=DEV, dtype=torch.int32)
    NB = 540000  # slots: 540000 * 16 * 2 * 128 = 2.2e9 elements
    kc, vc = (torch.zeros(NB, 16, 2, D, dtype=torch.float16, device=DEV) for _ in range(2))
    slots = torch.full((T,), -1, dtype=torch.int32, device=DEV)
    slots[-n:] = torch.arange(NB * 16 - n, NB * 16, device=DEV, dtype=torch.int32)
    q2, k2 = C().rotary_write_cache(q, k, v, pos, freq, [64], slots, kc, vc)
    q3, k3 = C().apply_rotary(a, b, pos[-n:], freq, [64])
    assert torch.equal(q2[-n:], q3) and torch.equal(k2[-n:], k3)
    assert torch.equal(kc.view(-1, 2, D)[-n:], k3) and torch.equal(vc.view(-1, 2, D)[-n:], c)
    assert not kc[:100].any() and not kc.view(-1, 2, D)[-n - 16:-n].any()


def test_overlapping_arguments_are_refused():
    q, k, v = make_qkv([8], 2, 2, 64, torch.float16)
    for out in (q, k, v):
        with pytest.raises(RuntimeError, match="overlap"):
            C().packed_attention(q, k, v, cu_of([8]), 8, -1, True, out)
    from memopt import DevicePageTable

    t = DevicePageTable(8, 16, 2, 64)
    rows = torch.arange(2, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="overlap"):
        t.truncate(rows, t.context_lens)
    with pytest.raises(RuntimeError, match="overlap"):
        t.reserve(rows, t.context_lens, 4)


def test_caches_and_rows_that_overlap_are_refused():
    q, k, v = make_qkv([16], 2, 2, 64, torch.float16)
    kc, vc = torch.zeros(1, 16, 2, 64, device=DEV, dtype=torch.float16), torch.zeros(1, 16, 2, 64, device=DEV,
                                                                                     dtype=torch.float16)
    pos = torch.arange(16, device=DEV, dtype=torch.int32)
    freq = torch.ones(32, device=DEV, dtype=torch.float64)
    for caches, kk in (((kc, kc), k), ((kc, vc), kc.reshape(16, 2, 64)), ((kc, vc), vc.reshape(16, 2, 64))):
        with pytest.raises(RuntimeError, match="overlap"):
            C().rotary_write_cache(q, kk, v, pos, freq, [32], pos, *caches)
    tables = torch.full((4, 4), -1, device=DEV, dtype=torch.int32)
    lens, ring = torch.zeros(4, device=DEV, dtype=torch.int32), torch.arange(8, device=DEV, dtype=torch.int32)
    state = torch.tensor([0, 8, 0, 0], device=DEV, dtype=torch.int32)
    for rows in (lens[:2], tables[1, :2]):
        with pytest.raises(RuntimeError, match="overlap"):
            C().reserve_slots(tables, lens, ring, state, rows, torch.ones(2, device=DEV, dtype=torch.int32), 16, 2)
        with pytest.raises(RuntimeError, match="overlap"):
            C().truncate_rows(tables, lens, ring, state, rows, None, 16)


def test_pages_of_more_rows_than_a_call_takes_come_back():
    """An eviction frees pages for every row of the table, also of more than 8192 rows."""
    from memopt import DevicePageTable

    rows = 9000
    t = DevicePageTable(rows * 2, 1, rows, 4)
    for at in range(0, rows, 6000):
        n = min(6000, rows - at)
        t.reserve(range(at, at + n), [2] * n)
    assert t.free_count() == 0
    pages, counts = t.block_tables.clone(), torch.full((rows,), 2, device=DEV, dtype=torch.int32)
    counts[5::7] = 1
    given = int(counts.sum())
    t.release_pages(pages, counts)
    assert t.free_count() == given and int(counts.sum()) == 0
    t.check()
    want = torch.cat([t.block_tables[i, :2 - (i % 7 == 5)].cpu() for i in range(rows)])
    assert torch.equal(t.free_pages[:given].cpu(), want)


@pytest.mark.parametrize("strides", ["sliced", "odd", "expanded", "transposed"])
def test_layouts_other_than_contiguous(strides):
    """Rows apart by any multiple of 8 elements are read in place, everything
    else through a copy: the same result either way."""
    lens, H, D = [40, 90], 4, 64
    q, k, v = make_qkv(lens, H, H, D, torch.bfloat16, seed=6)
    want = C().packed_attention(q, k, v, cu_of(lens), 90)

    def lay(x):
        T = x.shape[0]
        if strides == "sliced":
            return torch.cat([x, x, x], 1)[:, H:2 * H]
        if strides == "odd":  # tokens 4 elements off a multiple of 8
            y = torch.zeros(T, H * D + 4, dtype=x.dtype, device=DEV)
            y[:, :H * D] = x.reshape(T, -1)
            return y.as_strided((T, H, D), (H * D + 4, D, 1))
        if strides == "transposed":
            return x.transpose(0, 1).contiguous().transpose(0, 1)
        return x[:, :1].expand(-1, H, -1)

    if strides == "expanded":
        want = C().packed_attention(q, k[:, :1].contiguous(), v[:, :1].contiguous(), cu_of(lens), 90)
        got = C().packed_attention(q, lay(k), lay(v), cu_of(lens), 90)
        ref, mag = attention_ref(q, k[:, :1], v[:, :1], lens, -1, True)
        tol = attention_tol(ref, mag, v, 90, torch.bfloat16)
        assert ((got.double() - ref).abs() <= tol).all() and ((want.double() - ref).abs() <= tol).all()
    else:
        assert torch.equal(C().packed_attention(lay(q), lay(k), lay(v), cu_of(lens), 90), want)


@pytest.mark.parametrize("many,D", [(3000, 64), (900, 128), (260, 128)])
def test_many_long_and_short_sequences_find_their_items(many, D):
    """Hundreds to thousands of sequences (more than a CTA keeps the bounds of,
    with one and with two tiles an item): every row belongs to exactly one item."""
    rng = random.Random(many)
    if many == 260:  # long ones: two tiles an item
        lens = [rng.randint(700, 900) for _ in range(many)]
    else:
        lens = [rng.choice([0, 1, 5, 40, 65, 130, 300]) for _ in range(many)] + [2500]
    for causal in (True, False):
        T = sum(lens)
        q = torch.zeros(T, 2, D, dtype=torch.float16, device=DEV)
        k = torch.zeros(T, 1, D, dtype=torch.float16, device=DEV)
        v = (torch.arange(T, device=DEV) % 7).half()[:, None, None].expand(T, 1, D).contiguous()
        out = torch.full_like(q, float("nan"))
        C().packed_attention(q, k, v, cu_of(lens), 2500, -1, causal, out)
        # equal scores: the mean of the visible values
        x = v[:, 0, 0].double()
        cum = torch.cat([x.new_zeros(1), x.cumsum(0)])
        start = torch.repeat_interleave(cu_of(lens)[:-1].long(), torch.tensor(lens, device=DEV))
        end = torch.repeat_interleave(cu_of(lens)[1:].long(), torch.tensor(lens, device=DEV))
        at = torch.arange(T, device=DEV) + 1 if causal else end
        mean = (cum[at] - cum[start]) / (at - start)
        # weights of 1 are exact; the sum and one rounding of the result remain
        assert ((out[:, :, 0].double() - mean[:, None]).abs() <= 2.0 ** -11 * mean[:, None] + 1e-5).all()
        assert torch.equal(out, out[:, :1, :1].expand_as(out))


def test_grad_inputs_are_refused():
    q, k, v = make_qkv([8], 2, 2, 64, torch.float16)
    q.requires_grad_(True)
    with pytest.raises(RuntimeError, match="no gradient"):
        C().packed_attention(q, k, v, cu_of([8]), 8)
    with torch.no_grad():
        C().packed_attention(q, k, v, cu_of([8]), 8)
    freq = torch.ones(32, dtype=torch.float64, device=DEV)
    with pytest.raises(RuntimeError, match="no gradient"):
        C().apply_rotary(q, k, torch.zeros(8, dtype=torch.int32, device=DEV), freq, [32])
