"""attn_prompt_packed on the GPU against a plain 64-bit statement, within the
bound that bf16 weights and outputs leave (kv_ref.attend)."""
import numpy as np
import pytest
import torch

import kv_ref as R
from time_b200 import attn as A

pytestmark = pytest.mark.gpu

D = 128


def f64(t):
    return t.double().cpu().numpy()


def rows(rng, *shape):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(torch.bfloat16)


def cu_of(lens, gpu, first=0):
    return torch.tensor(np.concatenate([[first], first + np.cumsum(lens)]), dtype=torch.int32, device=gpu)


def check(out, q, k, v, lens, scale, first=0):
    at = first
    for n in lens:
        if n == 0:
            continue
        s = slice(at, at + n)
        ref, tol = R.attend(f64(q[s]), f64(k[s]), f64(v[s]), np.arange(1, n + 1), scale)
        got = f64(out[s])
        assert (np.abs(got - ref) <= tol).all(), (n, np.max(np.abs(got - ref) / tol))
        at += n


@pytest.mark.parametrize("nq,nkv,lens", [
    (12, 1, [1]), (12, 1, [1, 2, 3, 1]), (12, 1, [21, 22, 43, 64, 65]), (4, 4, [130, 1, 127, 128, 129]),
    (1, 1, [300]), (16, 1, [100, 33]), (7, 1, [300, 5]), (6, 2, [257, 256, 255]), (96, 8, [150, 3, 40]),
    (8, 8, [513]), (12, 1, [700, 10]), (2, 1, [1100]), (12, 1, [5] * 100)])
def test_packed_prompts(gpu, nq, nkv, lens):
    rng = np.random.default_rng(nq * 1000 + len(lens))
    T = sum(lens)
    q, k, v = rows(rng, T, nq, D).to(gpu), rows(rng, T, nkv, D).to(gpu), rows(rng, T, nkv, D).to(gpu)
    err = torch.zeros(1, dtype=torch.int32, device=gpu)
    out, _, _ = A.prompt_packed(q, k, v, cu_of(lens, gpu), D ** -0.5, error_word=err)
    assert int(err) == 0
    check(out, q, k, v, lens, D ** -0.5)


@pytest.mark.parametrize("scale,mag", [(1.0, 4.0), (0.02, 1.0), (3.0, 0.01)])
def test_sharp_and_flat_softmax(gpu, scale, mag):
    """Weights concentrated on one key (the running maximum moves often) and spread evenly."""
    rng = np.random.default_rng(1)
    n = 600
    q, k, v = (rows(rng, n, 2, D) * mag).to(gpu), (rows(rng, n, 1, D) * mag).to(gpu), rows(rng, n, 1, D).to(gpu)
    k *= torch.linspace(0.2, 2, n, device=gpu)[:, None, None]        # later keys score higher
    out, _, _ = A.prompt_packed(q, k, v, cu_of([n], gpu), scale)
    check(out, q, k, v, [n], scale)


def test_strides_empty_sequences_and_rows_outside(gpu):
    """q, k and v inside the projection's rows, sequences of length 0, rows before the first and behind the last."""
    rng = np.random.default_rng(2)
    nq, nkv, T = 6, 2, 60
    qkv = rows(rng, T, (nq + 2 * nkv) * D).to(gpu).unflatten(1, (nq + 2 * nkv, D))
    q, k, v = qkv[:, :nq], qkv[:, nq:nq + nkv], qkv[:, nq + nkv:]
    cu = torch.tensor([3, 3, 20, 20, 50, 50], dtype=torch.int32, device=gpu)
    out = torch.full((T, nq, D), 7.0, dtype=torch.bfloat16, device=gpu)
    A.prompt_packed(q, k, v, cu, 0.1, out=out)
    check(out, q, k, v, [17, 30], 0.1, first=3)
    assert (out[:3] == 7).all() and (out[50:] == 7).all()


def test_from_a_bad_bound_on_sequences_are_skipped(gpu):
    rng = np.random.default_rng(3)
    q, k, v = rows(rng, 40, 2, D).to(gpu), rows(rng, 40, 1, D).to(gpu), rows(rng, 40, 1, D).to(gpu)
    for cu, good in [([0, 30, 20, 40], [(0, 30)]), ([-1, 10, 20], []), ([0, 10, 41], [(0, 10)])]:
        out = torch.full((40, 2, D), 7.0, dtype=torch.bfloat16, device=gpu)
        err = torch.zeros(1, dtype=torch.int32, device=gpu)
        A.prompt_packed(q, k, v, torch.tensor(cu, dtype=torch.int32, device=gpu), 0.1, out=out, error_word=err)
        assert int(err) == 5
        for a, b in good:
            check(out[a:b], q[a:b], k[a:b], v[a:b], [b - a], 0.1)
        untouched = [t for t in range(40) if not any(x <= t < y for x, y in good)]
        assert (out[untouched] == 7).all()


@pytest.mark.parametrize("nq,nkv", [(12, 1), (4, 4)])
def test_nan_and_infinity_reach_only_the_rows_that_attend_them(gpu, nq, nkv):
    rng = np.random.default_rng(4)
    lens = [90, 300]
    T = sum(lens)
    q, k, v = rows(rng, T, nq, D), rows(rng, T, nkv, D), rows(rng, T, nkv, D)
    clean = A.prompt_packed(q.to(gpu), k.to(gpu), v.to(gpu), cu_of(lens, gpu), 0.1)[0]
    bad_v = v.clone()
    bad_v[40, 0, 3] = float("inf")
    bad_v[60, 0, 3] = float("-inf")
    bad_v[41, 0, 9] = float("nan")
    bad_v[89, 0] = float("nan")                            # last row of the first sequence
    bad_v[90 + 135, 0, 5] = float("inf")
    out = A.prompt_packed(q.to(gpu), k.to(gpu), bad_v.to(gpu), cu_of(lens, gpu), 0.1)[0]
    G = nq // nkv
    want = clean.clone()
    want[40:60, :G, 3] = float("inf")
    want[60:90, :G, 3] = float("nan")
    want[41:90, :G, 9] = float("nan")
    want[89, :G] = float("nan")
    want[90 + 135:, :G, 5] = float("inf")
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(torch.isinf(out), torch.isinf(want))
    fine = torch.isfinite(want)
    assert torch.equal(out[fine], clean[fine]) and (out[40:60, :G, 3] > 0).all()
    # keys: a NaN score makes the rows from there on NaN, those before keep their bits
    bad_k = k.clone()
    bad_k[90 + 140, 0, 0] = float("nan")
    out = A.prompt_packed(q.to(gpu), bad_k.to(gpu), v.to(gpu), cu_of(lens, gpu), 0.1)[0]
    assert torch.isnan(out[90 + 140:, :G]).all() and torch.equal(out[:90 + 140], clean[:90 + 140])
    assert torch.equal(out[:, G:], clean[:, G:])
    # and a NaN query its own row and head
    bad_q = q.clone()
    bad_q[17, nq - 1, 100] = float("nan")
    out = A.prompt_packed(bad_q.to(gpu), k.to(gpu), v.to(gpu), cu_of(lens, gpu), 0.1)[0]
    assert torch.isnan(out[17, nq - 1]).all()
    out[17, nq - 1] = clean[17, nq - 1]
    assert torch.equal(out, clean)


def test_minus_infinite_scores(gpu):
    """-inf scores weigh 0 as long as a row attends any other; a row of nothing else is 0 / 0."""
    n = 200
    q = torch.zeros(n, 1, D, dtype=torch.bfloat16, device=gpu)
    k, v = torch.zeros_like(q), rows(np.random.default_rng(5), n, 1, D).to(gpu)
    q[..., 0] = -3e38
    k[:150, :, 0] = 64.0                                   # times the scale: below the fp32 range
    out = f64(A.prompt_packed(q, k, v, cu_of([n], gpu), 4.0)[0])
    assert np.isnan(out[:150]).all()
    vf = f64(v)
    for t in (150, 151, 199):
        ref, size = vf[150:t + 1, 0].mean(axis=0), np.abs(vf[150:t + 1, 0]).mean(axis=0)
        assert (np.abs(out[t, 0] - ref) <= 2.0 ** -8 * 1.01 * (np.abs(ref) + size) + 1e-6).all()


def test_quantised_rows(gpu):
    rng = np.random.default_rng(6)
    lens, nq = [33, 100], 12
    T = sum(lens)
    q, k, v = rows(rng, T, nq, D).to(gpu), rows(rng, T, 1, D).to(gpu), rows(rng, T, 1, D).to(gpu)
    v[5] = 0
    v[0] = 0
    out, oq, os_ = A.prompt_packed(q, k, v, cu_of(lens, gpu), 0.1, quant=True)
    got = f64(out)
    e4m3 = oq.view(torch.float8_e4m3fn).double().cpu().numpy().reshape(T, nq, D)
    sc = os_.double().cpu().numpy()[:, :T].T[..., None]
    # half an e4m3 step (2^-4, or 2^-10 below the smallest normal) of the fp32 row, which the bf16 row is 2^-8 from
    amax = np.abs(got).max(axis=-1, keepdims=True) * (1 + 2.0 ** -7)
    assert (np.abs(e4m3 * sc - got) <= (2.0 ** -4 + 2.0 ** -7) * np.abs(got) + amax / 448 * 2.0 ** -10 * 1.01).all()
    assert not oq[0].any() and not os_[:, 0].any()
    assert torch.equal(out, A.prompt_packed(q, k, v, cu_of(lens, gpu), 0.1)[0])


def test_rows_do_not_depend_on_the_packing(gpu):
    rng = np.random.default_rng(7)
    lens, nq, nkv = [130, 7, 400], 12, 2
    T = sum(lens)
    q, k, v = rows(rng, T, nq, D).to(gpu), rows(rng, T, nkv, D).to(gpu), rows(rng, T, nkv, D).to(gpu)
    out = A.prompt_packed(q, k, v, cu_of(lens, gpu), 0.1)[0]
    at = 0
    for n in lens:
        one = A.prompt_packed(q[at:at + n].contiguous(), k[at:at + n], v[at:at + n], cu_of([n], gpu), 0.1)[0]
        assert torch.equal(one, out[at:at + n])
        at += n


def test_stream_and_graph(gpu):
    rng = np.random.default_rng(8)
    q, k, v = rows(rng, 90, 4, D).to(gpu), rows(rng, 90, 2, D).to(gpu), rows(rng, 90, 2, D).to(gpu)
    cu = cu_of([30, 60], gpu)
    want = A.prompt_packed(q, k, v, cu, 0.1)[0].clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = A.prompt_packed(q, k, v, cu, 0.1, stream=s)[0]
    s.synchronize()
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = A.prompt_packed(q, k, v, cu, 0.1)[0]
    cu.copy_(torch.tensor([0, 50, 90]))
    g.replay()
    assert torch.equal(o, A.prompt_packed(q, k, v, cu, 0.1)[0])
    check(o, q, k, v, [50, 40], 0.1)


def test_agrees_with_the_paged_prefill(gpu):
    """The same prompt through bf16 pages and the paged prefill kernel: both within their bound of the same values."""
    rng = np.random.default_rng(9)
    n, nq, nkv = 150, 12, 1
    q, k, v = rows(rng, n, nq, D).to(gpu), rows(rng, n, nkv, D).to(gpu), rows(rng, n, nkv, D).to(gpu)
    out = A.prompt_packed(q, k, v, cu_of([n], gpu), 0.1)[0]
    pages = -(-n // 16)
    kc = torch.zeros(pages, 16, nkv, D, dtype=torch.bfloat16, device=gpu)
    vc = torch.zeros_like(kc)
    kc.view(-1, nkv, D)[:n], vc.view(-1, nkv, D)[:n] = k, v
    pt = torch.arange(pages, dtype=torch.int32, device=gpu)[None].contiguous()
    paged = A.paged_rows(q, kc, vc, pt, torch.zeros(n, dtype=torch.int32, device=gpu),
                         torch.arange(1, n + 1, dtype=torch.int32, device=gpu), nq, nkv, 0.1, prefill_rows=n)[0]
    ref, tol = R.attend(f64(q), f64(k), f64(v), np.arange(1, n + 1), 0.1)
    assert (np.abs(f64(out) - ref) <= tol).all() and (np.abs(f64(paged) - ref) <= tol).all()


@pytest.mark.parametrize("scale", [-0.1, 0.0])
def test_scales_of_any_sign(gpu, scale):
    rng = np.random.default_rng(10)
    n = 300
    q, k, v = rows(rng, n, 6, D).to(gpu), rows(rng, n, 2, D).to(gpu), rows(rng, n, 2, D).to(gpu)
    out, _, _ = A.prompt_packed(q, k, v, cu_of([n], gpu), scale)
    ref, tol = R.attend(f64(-q if scale < 0 else q), f64(k), f64(v), np.arange(1, n + 1), abs(scale))
    assert (np.abs(f64(out) - ref) <= tol).all()


def test_many_uneven_prompts(gpu):
    """More tiles than SMs, one M tile and two, one step and several: what a CTA carries from tile to tile."""
    rng = np.random.default_rng(11)
    nq, nkv = 32, 8
    lens = [int(x) for x in np.exp(rng.uniform(0, np.log(700), 70))]
    T = sum(lens)
    q, k, v = rows(rng, T, nq, D).to(gpu), rows(rng, T, nkv, D).to(gpu), rows(rng, T, nkv, D).to(gpu)
    for _ in range(3):
        out, _, _ = A.prompt_packed(q, k, v, cu_of(lens, gpu), 0.1)
    at = 0
    for n in lens:
        if n < 200 or n == max(lens):
            s = slice(at, at + n)
            ref, tol = R.attend(f64(q[s]), f64(k[s]), f64(v[s]), np.arange(1, n + 1), 0.1)
            assert (np.abs(f64(out[s]) - ref) <= tol).all()
        at += n
    assert torch.equal(out, A.prompt_packed(q, k, v, cu_of(lens, gpu), 0.1)[0])


def test_more_sequences_than_a_warp(gpu):
    """Sequences of none, one and several tiles in an order that mixes them, past the 32 that are counted in registers."""
    rng = np.random.default_rng(12)
    nq, nkv = 4, 2
    lens = [int(x) for x in rng.choice([0, 1, 3, 17, 127, 128, 129, 300], 150)]
    T = sum(lens)
    q, k, v = rows(rng, T, nq, D).to(gpu), rows(rng, T, nkv, D).to(gpu), rows(rng, T, nkv, D).to(gpu)
    out = torch.full((T + 5, nq, D), 7.0, dtype=torch.bfloat16, device=gpu)[:T]
    A.prompt_packed(q, k, v, cu_of(lens, gpu), 0.1, out=out)
    check(out, q, k, v, lens, 0.1)
    # 5000 one-token prompts: every row is its value
    q, k, v = rows(rng, 5000, nq, D).to(gpu), rows(rng, 5000, nkv, D).to(gpu), rows(rng, 5000, nkv, D).to(gpu)
    out = A.prompt_packed(q, k, v, torch.arange(5001, dtype=torch.int32, device=gpu), 0.1)[0]
    assert torch.equal(out, v.repeat_interleave(nq // nkv, dim=1))


def test_two_calls_at_once(gpu):
    """The same buffers attended on two streams at the same time."""
    rng = np.random.default_rng(13)
    lens = [900, 40, 300]
    T = sum(lens)
    q, k, v = rows(rng, T, 16, D).to(gpu), rows(rng, T, 4, D).to(gpu), rows(rng, T, 4, D).to(gpu)
    want = A.prompt_packed(q, k, v, cu_of(lens, gpu), 0.1)[0]
    cu = cu_of(lens, gpu)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[A.prompt_packed(q, k, v, cu, 0.1, stream=s)[0] for s in streams] for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for pair in outs for o in pair)


@pytest.mark.parametrize("G", range(1, 17))
def test_every_group_size(gpu, G):
    """Whole and part-filled tiles of every group size, with rows outside that stay as they were; the same bits with and
    without the quantised rows."""
    rng = np.random.default_rng(G)
    nkv, first, lens = 2, 2, [256 // G * 2 + 3, 1, 70, 256 // G]
    T = first + sum(lens) + 5
    q, k, v = rows(rng, T, nkv * G, D).to(gpu), rows(rng, T, nkv, D).to(gpu), rows(rng, T, nkv, D).to(gpu)
    out = torch.full_like(q, 3.0)
    A.prompt_packed(q, k, v, cu_of(lens, gpu, first), 0.1, out=out)
    check(out, q, k, v, lens, 0.1, first)
    assert (out[:first] == 3).all() and (out[first + sum(lens):] == 3).all()
    again, _, _ = A.prompt_packed(q, k, v, cu_of(lens, gpu, first), 0.1, quant=True, out=torch.full_like(q, 3.0))
    assert torch.equal(out, again)


def test_element_numbers_past_32_bits(gpu):
    """q and out of 2.3e9 elements: prompts on both sides of element 2^31 and the last one."""
    nq, nkv, n = 128, 8, 500
    seqs = 280
    T = seqs * n
    assert T * nq * D > 2 ** 31
    g = torch.Generator(device=gpu).manual_seed(5)
    q, k, v = (torch.randn(T, h, D, dtype=torch.bfloat16, device=gpu, generator=g) for h in (nq, nkv, nkv))
    err = torch.zeros(1, dtype=torch.int32, device=gpu)
    out, _, _ = A.prompt_packed(q, k, v, cu_of([n] * seqs, gpu), D ** -0.5, error_word=err)
    assert int(err) == 0
    for s in (0, 2 ** 31 // (nq * D * n), seqs - 1):
        r = slice(s * n, (s + 1) * n)
        for h in (0, nq - 1):
            kv = h * nkv // nq
            ref, tol = R.attend(f64(q[r, h:h + 1]), f64(k[r, kv:kv + 1]), f64(v[r, kv:kv + 1]), np.arange(1, n + 1), D ** -0.5)
            assert (np.abs(f64(out[r, h:h + 1]) - ref) <= tol).all()


@pytest.mark.parametrize("G", [1, 12])
def test_quantised_rows_before_a_nan(gpu, G):
    """A NaN and an infinity in v, in tiles that are whole and in part filled: the rows before them keep their bits, as bf16
    and as e4m3 with its scale."""
    rng = np.random.default_rng(G)
    n = 300
    q, k, v = rows(rng, n, G, D).to(gpu), rows(rng, n, 1, D).to(gpu), rows(rng, n, 1, D).to(gpu)
    clean = A.prompt_packed(q, k, v, cu_of([n], gpu), 0.1, quant=True)
    for at in (1, 20, 64, 255, 290, 299):
        bad = v.clone()
        bad[at, 0, 7], bad[at, 0, 100] = float("nan"), float("-inf")
        out, oq, os_ = A.prompt_packed(q, k, bad, cu_of([n], gpu), 0.1, quant=True)
        assert torch.equal(out[:at], clean[0][:at]) and torch.equal(oq[:at], clean[1][:at])
        assert torch.equal(os_[:, :at], clean[2][:, :at])
        assert torch.isnan(out[at:, :, 7]).all() and (out[at:, :, 100] == float("-inf")).all()
        others = [d for d in range(D) if d not in (7, 100)]
        assert torch.equal(out[at:][..., others], clean[0][at:][..., others])


def test_rows_do_not_depend_on_the_size_of_the_call(gpu):
    """A prompt alone, which is run in smaller tiles, and among many others."""
    rng = np.random.default_rng(17)
    lens, nq = [400] + [300] * 20, 12
    T = sum(lens)
    q, k, v = rows(rng, T, nq, D).to(gpu), rows(rng, T, 1, D).to(gpu), rows(rng, T, 1, D).to(gpu)
    out = A.prompt_packed(q, k, v, cu_of(lens, gpu), 0.1)[0]
    for first, n in ((0, 400), (400, 300), (T - 300, 300)):
        s = slice(first, first + n)
        assert torch.equal(A.prompt_packed(q[s], k[s], v[s], cu_of([n], gpu), 0.1)[0], out[s])


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("long,short", [(13, 4), (16, 1), (21, 5), (19, 10)])
def test_short_tiles_right_behind_longer_ones(gpu, long, short, quant):
    """Every CTA's tiles alternate between two M tiles and one, so that a part of the epilogue that is done with the long
    one can be through the short one before the rest: the bits of each prompt alone, in every one of several runs."""
    rng = np.random.default_rng(long)
    nq, sms = 12, torch.cuda.get_device_properties(gpu).multi_processor_count
    lens = [long if i // sms % 2 == 0 else short for i in range(7 * sms)]
    T = sum(lens)
    q, k, v = rows(rng, T, nq, D).to(gpu), rows(rng, T, 1, D).to(gpu), rows(rng, T, 1, D).to(gpu)
    cu, err = cu_of(lens, gpu), torch.zeros(1, dtype=torch.int32, device=gpu)
    runs = [A.prompt_packed(q, k, v, cu, 0.1, quant=quant, error_word=err) for _ in range(10)]
    assert int(err) == 0
    at = 0
    want = [torch.empty_like(runs[0][0]), None, None]
    if quant:
        want = [want[0], torch.empty_like(runs[0][1]), torch.empty(nq, T, device=gpu)]
    for n in lens:
        s = slice(at, at + n)
        one = A.prompt_packed(q[s], k[s], v[s], cu_of([n], gpu), 0.1, quant=quant)
        want[0][s] = one[0]
        if quant:
            want[1][s], want[2][:, s] = one[1], one[2][:, :n]
        at += n
    for out, oq, os_ in runs:
        assert torch.equal(out, want[0])
        if quant:
            assert torch.equal(oq, want[1]) and torch.equal(os_[:, :T], want[2])


def e4m3_rows(oq, os_, T, nq):
    """The e4m3 rows times their scales, [T][nq][128] in 64 bits."""
    return oq.view(torch.float8_e4m3fn).double().reshape(T, nq, D) * os_[:, :T].double().t()[..., None]


@pytest.mark.parametrize("G", [1, 12])
@pytest.mark.parametrize("where", ["q", "k", "v", "v one dim", "v one dim of zeros"])
def test_nan_reaches_the_quantised_rows(gpu, G, where):
    """What is NaN in the bf16 rows is NaN in the e4m3 rows, rows that are NaN throughout among them; the rest keeps its
    codes and scales."""
    rng = np.random.default_rng(G)
    n = 300
    q, k, v = rows(rng, n, G, D).to(gpu), rows(rng, n, 1, D).to(gpu), rows(rng, n, 1, D).to(gpu)
    if where == "v one dim of zeros":
        v.zero_()
    _, clean_q, clean_s = A.prompt_packed(q, k, v, cu_of([n], gpu), 0.1, quant=True)
    for at in (0, 1, 70, 255, 299):
        bad = {"q": q, "k": k, "v": v}
        bad[where[0]] = b = bad[where[0]].clone()
        b[at, :, 7 if where[0] != "v" or where != "v" else slice(None)] = float("nan")
        out, oq, os_ = A.prompt_packed(bad["q"], bad["k"], bad["v"], cu_of([n], gpu), 0.1, quant=True)
        hit = torch.zeros(n, G, D, dtype=torch.bool, device=gpu)
        if where == "q":
            hit[at] = True
        elif where in ("k", "v"):
            hit[at:] = True
        else:
            hit[at:, :, 7] = True
        assert torch.equal(torch.isnan(out), hit) and torch.equal(torch.isnan(e4m3_rows(oq, os_, n, G)), hit)
        rows_hit = hit.any(dim=2)
        assert torch.equal(oq.view(n, G, D)[~rows_hit], clean_q.view(n, G, D)[~rows_hit])
        assert torch.equal(os_[:, :n].t()[~rows_hit], clean_s[:, :n].t()[~rows_hit])


def same(a, b):
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(nan=0.0), b.nan_to_num(nan=0.0))


@pytest.mark.parametrize("G", [1, 12])
@pytest.mark.parametrize("scores", ["far below", "left behind", "alike"])
def test_an_infinity_does_not_depend_on_the_tile(gpu, G, scores):
    """A weight that underflows is still positive: an infinity in v is infinite in every row that attends it and two of
    opposite signs are NaN, wherever the tiles begin; the other dims keep their bits, alone and in a batch."""
    rng = np.random.default_rng(G)
    n = 400
    k, v = torch.zeros(n, 1, D), rows(rng, n, 1, D)
    q = torch.zeros(n, G, D)
    q[..., 0] = 1.0
    c = torch.from_numpy(rng.standard_normal(n).astype(np.float32))
    # some positions 300 below the rest, or every 64 positions 100 above those before
    c += -300.0 * (torch.arange(n) % 50 == 3) if scores == "far below" else 100.0 * (torch.arange(n) // 64) if scores == "left behind" else 0
    k[:, 0, 0] = c
    q, k, v = q.to(torch.bfloat16).to(gpu), k.to(torch.bfloat16).to(gpu), v.to(gpu)
    clean = A.prompt_packed(q, k, v, cu_of([n], gpu), 1.0, quant=True)
    bad, want = v.clone(), clean[0].clone()
    for dim, at in ((3, [3]), (5, [53, 203]), (70, [203]), (127, [63]), (64, [64])):
        bad[at, 0, dim] = float("inf")
        want[at[0]:, :, dim] = float("inf")
    bad[103, 0, 9] = float("-inf")
    want[103:, :, 9] = float("-inf")
    bad[3, 0, 11], bad[253, 0, 11] = float("inf"), float("-inf")
    want[3:253, :, 11], want[253:, :, 11] = float("inf"), float("nan")
    bad[153, 0, 80] = float("nan")
    want[153:, :, 80] = float("nan")
    alone = A.prompt_packed(q, k, bad, cu_of([n], gpu), 1.0)[0]
    assert same(alone, want)
    # among many others the tiles are of another size
    r = 40
    batch = A.prompt_packed(q.repeat(r, 1, 1), k.repeat(r, 1, 1), bad.repeat(r, 1, 1), cu_of([n] * r, gpu), 1.0, quant=True)
    one = A.prompt_packed(q, k, bad, cu_of([n], gpu), 1.0, quant=True)
    assert same(one[0], want)
    for i in (0, 17, r - 1):
        s = slice(i * n, (i + 1) * n)
        assert same(batch[0][s], want)
        assert torch.equal(batch[1][s], one[1]) and same(batch[2][:, s], one[2][:, :n])
    hit = ~torch.isfinite(want)
    held = one[1].view(torch.float8_e4m3fn).double().reshape(n, G, D) * one[2][:, :n].double().t()[..., None]
    assert not torch.isfinite(held[hit]).any()
    rest = ~hit.any(dim=2)
    assert torch.equal(one[1].view(n, G, D)[rest], clean[1].view(n, G, D)[rest])


def test_quantised_rows_of_tiny_values(gpu):
    """Rows whose 448 / max is past the fp32 range: zeros stay zeros, the rest within half an e4m3 step."""
    n, nq = 20, 12
    rng = np.random.default_rng(14)
    q, k = rows(rng, n, nq, D).to(gpu), rows(rng, n, 1, D).to(gpu)
    for mag in (1e-36, 2.0 ** -125):
        v = (rows(rng, n, 1, D).sign() * mag).to(torch.bfloat16).to(gpu)
        v[..., 64:] = 0
        out, oq, os_ = A.prompt_packed(q, k, v, cu_of([n], gpu), 0.1, quant=True)
        got, held = out.double(), e4m3_rows(oq, os_, n, nq)
        # the scale is a subnormal number, half of 2^-149 off; the row's bf16 rounding may be of one, too
        amax = got.abs().amax(dim=2, keepdim=True) * (1 + 2.0 ** -7) + 2.0 ** -134
        tol = (2.0 ** -4 + 2.0 ** -7) * got.abs() + amax / 448 * 2.0 ** -10 * 1.01 + 448 * 2.0 ** -150 + 2.0 ** -134
        assert not held[..., 64:].any() and ((held - got).abs() <= tol).all()


def test_a_long_prompt(gpu):
    """16384 tokens, rows at the ends of steps and tiles and between, each against all the keys it attends."""
    rng = np.random.default_rng(16)
    n, nq = 16384, 12
    q, k, v = rows(rng, n, nq, D).to(gpu), rows(rng, n, 1, D).to(gpu), rows(rng, n, 1, D).to(gpu)
    err = torch.zeros(1, dtype=torch.int32, device=gpu)
    out, _, _ = A.prompt_packed(q, k, v, cu_of([n], gpu), D ** -0.5, error_word=err)
    at = [0, 20, 21, 63, 64, 1100, 4095, 8190, 8191, 12345, 16319, 16320, 16383]
    ref, tol = R.attend(f64(q[at]), f64(k), f64(v), [t + 1 for t in at], D ** -0.5)
    assert int(err) == 0 and (np.abs(f64(out[at]) - ref) <= tol).all()


@pytest.mark.parametrize("G,many", [(1, False), (5, False), (12, True), (16, False)])
def test_infinities_and_nan_anywhere(gpu, G, many):
    """Rows far behind them, in sequences of several lengths and two heads of keys: each dim is what the values that its row
    attends make it; whole rows of NaN, from which on everything is."""
    rng = np.random.default_rng(G)
    lens = [1500, 3, 700, 64, 257]
    T, nkv = sum(lens), 2
    q, k, v = torch.zeros(T, nkv * G, D), torch.zeros(T, nkv, D), rows(rng, T, nkv, D)
    q[..., 0] = 1.0
    k[..., 0] = torch.from_numpy(rng.standard_normal((T, nkv)).astype(np.float32) - 300.0 * (rng.random((T, nkv)) < 0.3))
    bad = rng.random((T, nkv, D)) < (0.02 if many else 0.0005)
    kind = rng.choice([np.inf, -np.inf, np.nan], (T, nkv, D))
    if not many:
        bad[900], kind[900] = True, np.nan
        bad[1600], kind[1600] = True, np.nan
    bv = torch.where(torch.from_numpy(bad), torch.from_numpy(kind).to(torch.bfloat16), v)
    q, k = q.to(torch.bfloat16).to(gpu), k.to(torch.bfloat16).to(gpu)
    cu = cu_of(lens, gpu)
    clean = A.prompt_packed(q, k, torch.where(torch.from_numpy(bad), torch.zeros_like(v), v).to(gpu), cu, 1.0)[0]
    out, oq, os_ = A.prompt_packed(q, k, bv.to(gpu), cu, 1.0, quant=True)
    assert same(out, A.prompt_packed(q, k, bv.to(gpu), cu, 1.0)[0])
    want = clean.cpu()
    at = 0
    for n in lens:
        s = slice(at, at + n)
        plus, minus, nan = (np.maximum.accumulate(bad[s] & c, axis=0) for c in
                            (kind[s] == np.inf, kind[s] == -np.inf, np.isnan(kind[s])))
        for hit, x in ((plus, np.inf), (minus, -np.inf), (nan | (plus & minus), np.nan)):
            want[s][torch.from_numpy(hit.repeat(G, axis=1))] = x
        at += n
    assert same(out.cpu(), want)
    held = oq.view(torch.float8_e4m3fn).double().reshape(T, nkv * G, D).cpu()
    assert torch.equal(torch.isnan(held * os_[:, :T].double().t()[..., None].cpu()).any(dim=2), (~torch.isfinite(want)).any(dim=2))
