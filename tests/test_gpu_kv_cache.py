"""The 4-bit cache and the page operators (include/kv_cache.h) on the GPU
against plain 64-bit statements (kv_ref): bytes and tables exactly, attention
within the bound that bf16 weights and outputs leave."""
import numpy as np
import pytest
import torch

import kv_ref as R
from time_b200 import attn as A
from time_b200 import kvcache as KV

pytestmark = pytest.mark.gpu

D, PAGE = 128, 16


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def f64(t):
    return t.double().cpu().numpy()


def normal_bf16(rng, *shape):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(torch.bfloat16)


def table_of(rng, lens, pool, extra=2):
    """Disjoint random pages, -1 behind each row's."""
    ids = rng.permutation(pool)
    pt = np.full((len(lens), max(1, max(map(R.pages, lens))) + extra), -1, np.int32)
    o = 0
    for b, n in enumerate(lens):
        pt[b, :R.pages(n)] = ids[o:o + R.pages(n)]
        o += R.pages(n)
    return pt


def random_cache(rng, pool, nkv):
    """Codes and scales a quantiser can have written, uint8 [pool][nkv][1152]."""
    x = rng.standard_normal((pool, nkv, PAGE, D)).astype(np.float32)
    c = np.zeros((pool, nkv, R.PAGE4), np.uint8)
    codes, s = R.quantise(x)
    out = {}
    for which in "kv":
        c = np.zeros((pool, nkv, R.PAGE4), np.uint8)
        for t in range(PAGE):
            byte, shift = R.code_place(which, t)
            np.bitwise_or.at(c, (slice(None), slice(None), byte), (codes[:, :, t] << shift.astype(np.uint8)).astype(np.uint8))
        c[:, :, R.CODE_BYTES:] = R.bf16_bits(s).astype("<u2").reshape(pool, nkv, -1).view(np.uint8)
        out[which] = c
        x = rng.standard_normal((pool, nkv, PAGE, D)).astype(np.float32)
        codes, s = R.quantise(x)
    return out["k"], out["v"]


def seq_values(cache, which, row, n):
    """[n][nkv][128] of one sequence."""
    return np.stack([np.stack([R.load(cache[row[t // PAGE], h], which, t % PAGE) for h in range(cache.shape[1])])
                     for t in range(n)]) if n else np.zeros((0, cache.shape[1], D))


# ---------------------------------------------------------------- write and read

@pytest.mark.parametrize("nq,nkv,rot,rows", [(12, 1, 64, 37), (96, 8, 64, 5), (4, 4, 128, 20), (7, 7, 0, 3), (6, 2, 6, 18),
                                             (1, 1, 2, 1), (16, 1, 126, 40)])
def test_write_and_read(gpu, nq, nkv, rot, rows):
    rng = np.random.default_rng(nq * 100 + rot)
    heads = nq + 2 * nkv
    qkv = normal_bf16(rng, rows, heads * D)
    qkv[0, :D] *= 1e4                                    # widely different rows
    qkv[-1] *= 1e-4
    if rows > 2:
        qkv[1, nq * D:] = 0                              # all-zero groups
        qkv[2, (nq + nkv) * D + 5] = float("inf")        # a v group that cannot be stored
        qkv[2, nq * D + 127] = float("nan")              # and a k group, outside the rotated dims unless rot = 128
    # two sequences, positions interleaved and out of order, far ones among them
    row_seq = (np.arange(rows) % 2).astype(np.int32)
    pos = np.where(row_seq == 0, np.arange(rows) // 2, 70000 + 3 * (np.arange(rows) // 2)).astype(np.int32)
    order = rng.permutation(rows)
    row_seq, pos = row_seq[order], pos[order]
    mp = 70000 // PAGE + 20
    used = sorted({(int(s), int(p) // PAGE) for s, p in zip(row_seq, pos)})
    pool = len(used) + 3
    pt = np.full((2, mp), -1, np.int32)
    for (s, j), id in zip(used, rng.permutation(pool)):
        pt[s, j] = id
    kc = torch.from_numpy(rng.integers(0, 256, (pool, nkv, 1152)).astype(np.uint8)).to(gpu)
    vc = torch.from_numpy(rng.integers(0, 256, (pool, nkv, 1152)).astype(np.uint8)).to(gpu)
    k_ref, v_ref = kc.cpu().numpy().copy(), vc.cpu().numpy().copy()
    f = A.rope_inv_freq(max(rot, 2), 1e6)
    err, lens = i32([0], gpu), i32([0] * rows, gpu)
    q, k = KV.kv4_rope_write(qkv.to(gpu), i32(pos, gpu), i32(row_seq, gpu), i32(pt, gpu), kc, vc, nq, rot,
                             torch.from_numpy(f).to(gpu), keys=True, seq_lens_out=lens, error_word=err)
    assert int(err) == 0 and lens.tolist() == (pos + 1).tolist()
    # rotation: the angle is the fp32 product; two products and a sum in fp32, one rounding to bf16
    x = f64(qkv).reshape(rows, heads, D)[:, :nq + nkv]
    ang = (pos.astype(np.float32)[:, None] * f[None, :rot // 2]).astype(np.float64)[:, None]
    a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    ref = np.concatenate([a * np.cos(ang) - b * np.sin(ang), a * np.sin(ang) + b * np.cos(ang), x[..., rot:]], axis=-1)
    size = np.concatenate([np.abs(a) + np.abs(b)] * 2 + [np.zeros_like(x[..., rot:])], axis=-1)
    got = np.concatenate([f64(q), f64(k)], axis=1)
    ok = np.isfinite(ref)
    assert np.array_equal(np.isfinite(got), ok)
    # sincosf is within two steps (2^-22)
    assert (np.abs(got - ref)[ok] <= (2.0 ** -8 * np.abs(ref) + 2.0 ** -21 * size)[ok]).all()
    # pages, byte for byte, from the rotated keys that the call returned
    kf, vf = k.float().cpu().numpy(), qkv.float().numpy().reshape(rows, heads, D)[:, nq + nkv:]
    (kcode, ks), (vcode, vs) = R.quantise(kf), R.quantise(vf)
    for r in range(rows):
        page, t = pt[row_seq[r], pos[r] // PAGE], pos[r] % PAGE
        for h in range(nkv):
            R.store(k_ref[page, h], "k", t, kcode[r, h], ks[r, h])
            R.store(v_ref[page, h], "v", t, vcode[r, h], vs[r, h])
    assert np.array_equal(kc.cpu().numpy(), k_ref) and np.array_equal(vc.cpu().numpy(), v_ref)
    kr, vr = KV.kv4_read_rows(kc, vc, i32(pos, gpu), i32(row_seq, gpu), i32(pt, gpu), error_word=err)
    assert int(err) == 0
    np.testing.assert_array_equal(f64(kr), R.values(kcode, ks).reshape(rows, nkv, D))
    np.testing.assert_array_equal(f64(vr), R.values(vcode, vs).reshape(rows, nkv, D))


def test_write_extreme_magnitudes(gpu):
    """The smallest and largest storable groups, and those just outside."""
    x = torch.zeros(1, 3 * D, dtype=torch.bfloat16)
    v = x[0, 2 * D:]
    v[0], v[1] = 2.0 ** -133, -(2.0 ** -130)             # below the smallest scale
    v[32], v[33] = 2.0 ** 119 * 1.9921875, -1.0          # the largest group that is stored
    v[64] = 2.0 ** 120                                   # not stored
    v[96], v[97] = 3.0e-38, -1.5e-38
    kc, vc = KV.kv4_cache(1, 1, gpu), KV.kv4_cache(1, 1, gpu)
    KV.kv4_rope_write(x.to(gpu), i32([4], gpu), None, i32([[0]], gpu), kc, vc, 1, 0, None)
    _, vr = KV.kv4_read_rows(kc, vc, i32([4], gpu), None, i32([[0]], gpu))
    codes, s = R.quantise(v.float().numpy()[None])
    np.testing.assert_array_equal(f64(vr)[0], R.values(codes, s))
    assert torch.isnan(vr[0, 0, 64:96]).all() and torch.isfinite(vr[0, 0, 32:64]).all()


@pytest.mark.parametrize("rot", [64, 36])
def test_write_rounds_each_product(gpu, rot):
    """Both products and their sum are rounded to fp32, whatever a compiler would contract: the bits of the same steps in
    torch, one operation at a time.  (The same cosf and sinf give the angles there.)"""
    rng = np.random.default_rng(rot)
    rows, nq, nkv = 300, 12, 1
    qkv = normal_bf16(rng, rows, nq + 2 * nkv, D).to(gpu)
    pos = i32(rng.permutation(rows), gpu)
    f = torch.from_numpy(A.rope_inv_freq(rot, 1e6)).to(gpu)
    pages = -(-rows // PAGE)
    kc, vc = KV.kv4_cache(pages, nkv, gpu), KV.kv4_cache(pages, nkv, gpu)
    q, k = KV.kv4_rope_write(qkv.flatten(1), pos, i32([0] * rows, gpu), i32([list(range(pages))], gpu), kc, vc, nq, rot, f,
                             keys=True)
    ang = (pos.float()[:, None] * f)[:, None]
    c, s = ang.cos(), ang.sin()
    x = qkv[:, :nq + nkv].float()
    a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    ac, bs, as_, bc = a * c, b * s, a * s, b * c
    want = torch.cat([ac - bs, as_ + bc, x[..., rot:]], dim=-1).bfloat16()
    assert torch.equal(torch.cat([q, k], dim=1), want)


@pytest.mark.parametrize("exp", [-132, -126, -122, -118, -59, -58, -57, -56, 0, 60, 117])
def test_write_rounds_every_quotient(gpu, exp):
    """Groups whose largest value is 2^exp times 1 to 2: every scale of four bits there with every bf16 value of both
    signs down to 2^-7 of the largest, halves between two codes among them.  Codes are exact, so nothing is tolerated."""
    tops = 2.0 ** exp * (1 + np.arange(128) / 128)
    tops = torch.from_numpy(tops).to(torch.bfloat16)           # subnormal below 2^-126
    _, s = R.quantise(tops.double().numpy().repeat(D).reshape(-1, D))
    groups = []
    for v in np.unique(s[:, 0]):
        top = tops[s[:, 0] == v].max()                         # the largest group of that scale
        x = (top.view(torch.int16).to(torch.int32) - torch.arange(7 * 128)).clamp(min=0).to(torch.int16).view(torch.bfloat16)
        x = torch.cat([x, -x, torch.zeros(-2 * len(x) % 31, dtype=torch.bfloat16)]).reshape(-1, 31)
        groups.append(torch.cat([top.repeat(len(x), 1), x], dim=1))
    x = torch.cat(groups)
    x = torch.cat([x, x[:-len(x) % 4]]).reshape(-1, D)
    rows = len(x)
    qkv = torch.cat([torch.zeros_like(x), x, -x], dim=1).to(gpu)
    pages = -(-rows // PAGE)
    kc, vc = KV.kv4_cache(pages, 1, gpu), KV.kv4_cache(pages, 1, gpu)
    pt, pos, seq = i32([list(range(pages))], gpu), i32(list(range(rows)), gpu), i32([0] * rows, gpu)
    KV.kv4_rope_write(qkv, pos, seq, pt, kc, vc, 1, 0, None)
    for got, want in zip(KV.kv4_read_rows(kc, vc, pos, seq, pt), (x, -x)):
        np.testing.assert_array_equal(f64(got)[:, 0], R.values(*R.quantise(want.double().numpy())))


def test_write_and_read_bounds(gpu):
    rng = np.random.default_rng(3)
    nq, nkv = 4, 1
    qkv = normal_bf16(rng, 5, (nq + 2 * nkv) * D).to(gpu)
    kc, vc = KV.kv4_cache(2, nkv, gpu), KV.kv4_cache(2, nkv, gpu)
    pt = i32([[0, 7], [1, -1]], gpu)
    f = torch.from_numpy(A.rope_inv_freq(64, 1e6)).to(gpu)
    # position past the table, page ids 7 and -1, sequences 2 and -1
    for pos, seq, code in [(32, 0, 4), (-1, 0, 4), (16, 0, 6), (16, 1, 6), (0, 2, 7), (0, -1, 7)]:
        err = i32([0], gpu)
        lens = i32([9], gpu)
        KV.kv4_rope_write(qkv[:1], i32([pos], gpu), i32([seq], gpu), pt, kc, vc, nq, 64, f, seq_lens_out=lens, error_word=err)
        assert int(err) == code and int(lens) == (pos + 1 if pos >= 0 and seq in (0, 1) else 0)
        err.zero_()
        k, v = KV.kv4_read_rows(kc, vc, i32([pos], gpu), i32([seq], gpu), pt, error_word=err)
        assert int(err) == code and not k.any() and not v.any()
    assert not kc.any() and not vc.any()
    # a good row beside bad ones is written
    err = i32([0], gpu)
    KV.kv4_rope_write(qkv[:3], i32([3, 3, 99], gpu), i32([5, 0, 1], gpu), pt, kc, vc, nq, 64, f, error_word=err)
    assert int(err) in (4, 7)
    codes, s = R.quantise(qkv[1, 5 * D:].float().cpu().numpy()[None])
    want = np.zeros(R.PAGE4, np.uint8)
    R.store(want, "v", 3, codes[0], s[0])
    assert np.array_equal(vc[0, 0].cpu().numpy(), want)


# ---------------------------------------------------------------- decode

def check_decode(gpu, rng, nq, nkv, lens, split, q=None, row_seq=None, quant=False, **kw):
    pool = sum(map(R.pages, lens)) + 3
    kc, vc = random_cache(rng, pool, nkv)
    pt = table_of(rng, lens, pool)
    rows = list(range(len(lens))) if row_seq is None else row_seq
    q = normal_bf16(rng, len(rows), nq, D) if q is None else q
    err = i32([0], gpu)
    row_lens = kw.pop("row_lens", [lens[s] for s in rows])
    out, oq, os_ = KV.kv4_decode(q.to(gpu), torch.from_numpy(kc).to(gpu), torch.from_numpy(vc).to(gpu), i32(pt, gpu),
                                 i32(row_lens, gpu), D ** -0.5, row_seq=None if row_seq is None else i32(row_seq, gpu),
                                 split_tokens=split, quant=quant, error_word=err, **kw)
    assert int(err) == 0
    got = f64(out)
    for b, (s, n) in enumerate(zip(rows, row_lens)):
        if n <= 0:
            assert not got[b].any()
            continue
        ref, tol = R.attend(f64(q[b:b + 1]), seq_values(kc, "k", pt[s], n), seq_values(vc, "v", pt[s], n), [n], D ** -0.5)
        assert (np.abs(got[b] - ref[0]) <= tol[0]).all(), np.max(np.abs(got[b] - ref[0]) / tol[0])
    return got, oq, os_


@pytest.mark.parametrize("nq,nkv,lens,split", [
    (12, 1, [1], 64), (12, 1, [1, 17, 600], 512), (96, 8, [33, 250], 64), (8, 2, [300, 0, 2048], 512), (4, 4, [100, 16], 16),
    (7, 1, [15, 31, 65], None), (16, 1, [1025, 15, 512, 513], 256), (1, 1, [3, 64], None), (6, 2, [1, 2, 3, 4, 5], None),
    (32, 2, [4100], 8192)])
def test_decode(gpu, nq, nkv, lens, split):
    check_decode(gpu, np.random.default_rng(nq + len(lens)), nq, nkv, lens, split)


def test_decode_rows_of_sequences_and_quantised_output(gpu):
    """Rows that map to sequences (several rows of one), shorter than them, and the e4m3 rows for o_proj."""
    rng = np.random.default_rng(5)
    got, oq, os_ = check_decode(gpu, rng, 12, 1, [70, 40, 33], 32, row_seq=[2, 0, 0, 1, 0], row_lens=[33, 5, 70, 40, 0],
                                quant=True)
    e4m3 = oq.view(torch.float8_e4m3fn).double().cpu().numpy().reshape(5, 12, D)
    sc = os_.double().cpu().numpy()[:, :5].T[..., None]
    # half an e4m3 step (2^-4, or 2^-10 below the smallest normal) of the fp32 row, which the bf16 row is 2^-8 from
    amax = np.abs(got).max(axis=-1, keepdims=True) * (1 + 2.0 ** -7)
    assert (np.abs(e4m3 * sc - got) <= (2.0 ** -4 + 2.0 ** -7) * np.abs(got) + amax / 448 * 2.0 ** -10 * 1.01).all()
    assert not oq[4].any() and not os_[:, 4].any()


def test_decode_ignores_slots_past_the_length(gpu):
    """NaN scales and every code in the slots behind a sequence change nothing; nor do pages behind it."""
    rng = np.random.default_rng(6)
    nq, nkv, n = 12, 2, 21
    kc, vc = random_cache(rng, 4, nkv)
    pt = np.array([[2, 0, 3]], np.int32)
    q = normal_bf16(rng, 1, nq, D).to(gpu)
    outs = []
    for fill in (0, 255):
        for c, which in ((kc, "k"), (vc, "v")):
            for h in range(nkv):
                for t in range(n - 16, 16):
                    byte, _ = R.code_place(which, t)
                    c[0, h, byte] = fill
                    c[0, h, R.CODE_BYTES + 8 * t:R.CODE_BYTES + 8 * t + 8] = fill     # 0xFFFF: NaN
            c[3] = fill
        outs.append(KV.kv4_decode(q, torch.from_numpy(kc).to(gpu), torch.from_numpy(vc).to(gpu), i32(pt, gpu), i32([n], gpu),
                                  D ** -0.5)[0])
    assert torch.isfinite(outs[0].float()).all() and torch.equal(outs[0], outs[1])


def test_decode_nan_and_infinite_inputs_stay_in_their_rows(gpu):
    rng = np.random.default_rng(7)
    kc, vc = random_cache(rng, 8, 1)
    pt = np.array([[0, 1, 2], [3, 4, 5]], np.int32)
    # an unstorable V group (dims 32..63) at position 20 of sequence 0
    vc[1, 0, R.CODE_BYTES + 8 * 4 + 2:R.CODE_BYTES + 8 * 4 + 4] = [0xC0, 0x7F]
    q = normal_bf16(rng, 3, 4, D)
    q[2, 1, 7] = float("nan")
    lens = [40, 40, 20]
    out = f64(KV.kv4_decode(q.to(gpu), torch.from_numpy(kc).to(gpu), torch.from_numpy(vc).to(gpu), i32(pt, gpu),
                            i32(lens, gpu), 0.1, row_seq=i32([0, 1, 0], gpu), split_tokens=16)[0])
    assert np.isnan(out[0, :, 32:64]).all() and np.isfinite(out[0, :, :32]).all() and np.isfinite(out[0, :, 64:]).all()
    assert np.isfinite(out[1]).all()                       # the other sequence
    assert np.isnan(out[2, 1]).all() and np.isfinite(out[2, [0, 2, 3]]).all()   # length 20 does not reach position 20


def test_decode_first_split_all_minus_infinity(gpu):
    """Scores of -inf in the first pages and finite ones later: weight 0, as a softmax gives."""
    nq = 2
    q = torch.zeros(1, nq, D, dtype=torch.bfloat16)
    q[..., 0] = float("-inf")
    kc, vc = random_cache(np.random.default_rng(8), 4, 1)
    x = np.zeros((64, D), np.float32)
    x[:, 1:] = 0
    x[:40, 0] = 7.0                    # -inf * 7
    x[40:, 0] = 0.0                    # -inf * 0: NaN
    for t in range(64):
        codes, s = R.quantise(x[t:t + 1])
        R.store(kc[t // 16, 0], "k", t % 16, codes[0], s[0])
    pt = i32([[0, 1, 2, 3]], gpu)
    run = lambda n, split: KV.kv4_decode(q.to(gpu), torch.from_numpy(kc).to(gpu), torch.from_numpy(vc).to(gpu), pt,  # noqa: E731
                                         i32([n], gpu), 1.0, split_tokens=split)[0]
    assert torch.isnan(run(64, 16).float()).all()          # NaN scores
    assert torch.isnan(run(32, 16).float()).all()          # nothing but -inf: 0 / 0
    big = torch.zeros(1, nq, D, dtype=torch.bfloat16)
    big[..., 0] = -3e38                                    # -3e38 * 7 * 4: -inf; 0 for the later keys
    out = KV.kv4_decode(big.to(gpu), torch.from_numpy(kc).to(gpu), torch.from_numpy(vc).to(gpu), pt, i32([64], gpu), 4.0,
                        split_tokens=16)[0]
    ref = seq_values(vc, "v", np.arange(4), 64)[40:, 0].mean(axis=0)
    tol = (2.0 ** -8 * np.abs(ref) + 2.0 ** -8 * np.abs(seq_values(vc, "v", np.arange(4), 64)[40:, 0]).mean(axis=0)) * 1.01
    assert (np.abs(f64(out)[0] - ref) <= tol + 1e-6).all()


@pytest.mark.parametrize("scale", [-0.1, 0.0, 0.02, 2.0])
def test_decode_scales(gpu, scale):
    rng = np.random.default_rng(13)
    kc, vc = random_cache(rng, 30, 2)
    pt, lens = table_of(rng, [250, 100], 30), [250, 100]
    q = normal_bf16(rng, 2, 8, D)
    out = f64(KV.kv4_decode(q.to(gpu), torch.from_numpy(kc).to(gpu), torch.from_numpy(vc).to(gpu), i32(pt, gpu),
                            i32(lens, gpu), scale, split_tokens=64)[0])
    for b, n in enumerate(lens):
        ref, tol = R.attend(f64(-q[b:b + 1] if scale < 0 else q[b:b + 1]), seq_values(kc, "k", pt[b], n),
                            seq_values(vc, "v", pt[b], n), [n], abs(scale))
        assert (np.abs(out[b] - ref[0]) <= tol[0]).all()


def test_empty_batches(gpu):
    kc = KV.kv4_cache(2, 1, gpu)
    none = i32([], gpu)
    table = torch.zeros(0, 3, dtype=torch.int32, device=gpu)
    q = torch.zeros(0, 4, D, dtype=torch.bfloat16, device=gpu)
    assert KV.kv4_decode(q, kc, kc, table, none, 0.1)[0].shape == (0, 4, D)
    x = torch.zeros(0, 6 * D, dtype=torch.bfloat16, device=gpu)
    f = torch.zeros(32, device=gpu)
    assert KV.kv4_rope_write(x, none, None, table, kc, kc, 4, 64, f)[0].shape == (0, 4, D)
    assert KV.kv4_read_rows(kc, kc, none, None, table)[0].shape == (0, 1, D)
    t, n = KV.fork_pages(kc[None], i32([[0]], gpu), i32([1], gpu), none)
    assert t.shape == (0, 1) and n.numel() == 0


def test_decode_bounds(gpu):
    rng = np.random.default_rng(9)
    kc, vc = random_cache(rng, 4, 1)
    kd, vd = torch.from_numpy(kc).to(gpu), torch.from_numpy(vc).to(gpu)
    q = normal_bf16(rng, 1, 4, D).to(gpu)
    err = i32([0], gpu)
    a = KV.kv4_decode(q, kd, vd, i32([[0, 1]], gpu), i32([100], gpu), 0.1, split_tokens=16, error_word=err)[0]
    assert int(err) == 5
    b = KV.kv4_decode(q, kd, vd, i32([[0, 1]], gpu), i32([32], gpu), 0.1, split_tokens=16)[0]
    assert torch.equal(a, b)
    for bad in (1000, -1, 4):
        err.zero_()
        out = KV.kv4_decode(q, kd, vd, i32([[0, bad]], gpu), i32([20], gpu), 0.1, split_tokens=16, error_word=err)[0]
        # the page reads as zeros: keys that score 0 and values of 0
        ref, tol = R.attend(f64(q), np.concatenate([seq_values(kc, "k", [0], 16), np.zeros((4, 1, D))]),
                            np.concatenate([seq_values(vc, "v", [0], 16), np.zeros((4, 1, D))]), [20], 0.1)
        assert int(err) == 6 and (np.abs(f64(out) - ref) <= tol).all()
    err.zero_()
    out = KV.kv4_decode(q, kd, vd, i32([[0, 1]], gpu), i32([20], gpu), 0.1, row_seq=i32([1], gpu), error_word=err)[0]
    assert int(err) == 7 and not out.any()


@pytest.mark.parametrize("bad", [[0], [1], [0, 1], [9, 24], [8, 9, 46], list(range(0, 48, 5))])
def test_decode_bad_ids_among_many_pages(gpu, bad):
    """One split of 48 pages with ids outside the cache: those pages read as zeros, and the good ones that come into the
    same places of shared memory after them as themselves."""
    rng = np.random.default_rng(len(bad))
    pages = 48
    kc, vc = random_cache(rng, pages, 1)
    q = normal_bf16(rng, 1, 12, D).to(gpu)
    row = rng.permutation(pages)
    ids = row.copy()
    ids[bad] = [1000, -1, pages][len(bad) % 3]
    k, v = seq_values(kc, "k", row, pages * PAGE), seq_values(vc, "v", row, pages * PAGE)
    for x in (k, v):
        x.reshape(pages, -1)[bad] = 0
    ref, tol = R.attend(f64(q), k, v, [pages * PAGE], 0.1)
    kd, vd = torch.from_numpy(kc).to(gpu), torch.from_numpy(vc).to(gpu)
    for _ in range(20):
        err = i32([0], gpu)
        out = KV.kv4_decode(q, kd, vd, i32(ids[None], gpu), i32([pages * PAGE], gpu), 0.1, split_tokens=pages * PAGE,
                            error_word=err)[0]
        assert int(err) == 6 and (np.abs(f64(out) - ref) <= tol).all()


def test_decode_row_bits_do_not_depend_on_the_batch(gpu):
    rng = np.random.default_rng(10)
    lens = [200, 1, 77, 130]
    kc, vc = random_cache(rng, 40, 2)
    kd, vd = torch.from_numpy(kc).to(gpu), torch.from_numpy(vc).to(gpu)
    pt = i32(table_of(rng, lens, 40), gpu)
    q = normal_bf16(rng, 4, 16, D).to(gpu)
    all_ = KV.kv4_decode(q, kd, vd, pt, i32(lens, gpu), 0.1, split_tokens=64)[0]
    for b in range(4):
        one = KV.kv4_decode(q[b:b + 1], kd, vd, pt, i32(lens[b:b + 1], gpu), 0.1, row_seq=i32([b], gpu), split_tokens=64)[0]
        assert torch.equal(one[0], all_[b])


def test_pages_beyond_32_bit_offsets(gpu):
    """Pages whose byte offset passes 2^32: written, read back and attended."""
    nq, nkv, pool = 8, 8, 480_000                          # 4.4 GB a cache
    kc = torch.empty(pool, nkv, 1152, dtype=torch.uint8, device=gpu)
    vc = torch.empty_like(kc)
    ids = [pool - 1, 3, 466_034, 240_000]                  # 466034 * 9216 is just past 2^32
    pt = i32([ids], gpu)
    rng = np.random.default_rng(11)
    n = 60
    x = normal_bf16(rng, n, (nq + 2 * nkv) * D)
    q, k = KV.kv4_rope_write(x.to(gpu), i32(range(n), gpu), i32([0] * n, gpu), pt, kc, vc, nq, 0, None, keys=True)
    kr, vr = KV.kv4_read_rows(kc, vc, i32(range(n), gpu), i32([0] * n, gpu), pt)
    kcode, ks = R.quantise(k.float().cpu().numpy())
    np.testing.assert_array_equal(f64(kr), R.values(kcode, ks))
    out = KV.kv4_decode(q[-1:], kc, vc, pt, i32([n], gpu), D ** -0.5, split_tokens=32)[0]
    ref, tol = R.attend(f64(q[-1:]), f64(kr), f64(vr), [n], D ** -0.5)
    assert (np.abs(f64(out) - ref) <= tol).all()


def test_decode_other_stream_and_graph(gpu):
    """On a stream of its own, and captured once and replayed with other lengths; two graphs with workspaces of their own."""
    rng = np.random.default_rng(12)
    kc, vc = random_cache(rng, 30, 1)
    kd, vd = torch.from_numpy(kc).to(gpu), torch.from_numpy(vc).to(gpu)
    pt = i32(table_of(rng, [200, 150], 30), gpu)
    q = normal_bf16(rng, 2, 12, D).to(gpu)
    lens = i32([200, 150], gpu)
    want = KV.kv4_decode(q, kd, vd, pt, lens, 0.1, split_tokens=64)[0].clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = KV.kv4_decode(q, kd, vd, pt, lens, 0.1, split_tokens=64, stream=s)[0]
    s.synchronize()
    assert torch.equal(got, want)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = KV.kv4_decode(q, kd, vd, pt, lens, 0.1, split_tokens=64)[0]
        graphs.append((g, o))
    lens.copy_(i32([33, 150], gpu))
    want = KV.kv4_decode(q, kd, vd, pt, lens, 0.1, split_tokens=64)[0]
    for g, o in graphs:
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for _, o in graphs)


# ---------------------------------------------------------------- pages

def fork_case(rng, seqs, rows, longest, pool_extra, caches=3, words=36):
    """Tables of a pool in use: some rows share their first pages, as earlier forks leave them."""
    lens = rng.integers(0, longest + 1, seqs)
    pool = int(sum(map(R.pages, lens))) + pool_extra
    pt = table_of(rng, lens, pool, extra=4)
    for s in range(1, seqs):
        if rng.random() < 0.5:
            p = rng.integers(0, s)
            n = min(lens[s], lens[p]) // PAGE
            pt[s, :n] = pt[p, :n]
            if rng.random() < 0.5 and lens[p] % PAGE:      # the page in part filled too
                pt[s], lens[s] = pt[p], lens[p]
    c = rng.integers(0, 1 << 31, (caches, pool, words)).astype(np.int32)
    parents = rng.integers(-1, seqs, rows)
    reserve = rng.choice([0, 1, 1, 3, 17, 40], rows)
    return c, pt, lens.astype(np.int32), parents.astype(np.int32), reserve.astype(np.int32)


@pytest.mark.parametrize("seqs,rows,longest,extra", [(1, 1, 1, 1), (4, 8, 100, 40), (3, 1, 50, 4), (40, 120, 300, 600),
                                                     (5, 5, 16, 20), (7, 30, 33, 5), (2, 40, 20, 0), (600, 1500, 40, 6000),
                                                     (300, 1500, 400, 9000), (9, 20, 100, 40000)])
def test_fork(gpu, seqs, rows, longest, extra):
    for seed in range(3):
        rng = np.random.default_rng(seed * 1000 + seqs)
        c, pt, lens, parents, reserve = fork_case(rng, seqs, rows, longest, extra)
        out, n, cref, short = R.fork(c, pt, lens, parents, reserve)
        cd, err = torch.from_numpy(c).to(gpu), i32([0], gpu)
        t, ln = KV.fork_pages(cd, i32(pt, gpu), i32(lens, gpu), i32(parents, gpu), i32(reserve, gpu), error_word=err)
        # a reservation past the table's columns is cut and recorded as well
        cut = any((lens[p] if p >= 0 else 0) + r > pt.shape[1] * PAGE for p, r in zip(parents, reserve))
        assert int(err) in ([8, 4] if short and cut else [8] if short else [4] if cut else [0])
        assert np.array_equal(t.cpu().numpy(), out) and np.array_equal(ln.cpu().numpy(), n)
        assert np.array_equal(cd.cpu().numpy(), cref)


@pytest.mark.parametrize("words", [4, 288, 1024, 2052])
def test_fork_page_sizes_and_layers_apart(gpu, words):
    """Pages of 16 bytes to 8 KB; caches that lie apart inside a larger allocation keep what is between them."""
    rng = np.random.default_rng(words)
    c, pt, lens, parents, reserve = fork_case(rng, 6, 20, 90, 80, caches=5, words=words)
    big = torch.from_numpy(rng.integers(0, 1 << 31, (5, c.shape[1] + 3, words)).astype(np.int32)).to(gpu)
    before = big.clone()
    view = big[:, :c.shape[1]]
    view.copy_(torch.from_numpy(c))
    out, n, cref, _ = R.fork(c, pt, lens, parents, reserve)
    t, _ = KV.fork_pages(view, i32(pt, gpu), i32(lens, gpu), i32(parents, gpu), i32(reserve, gpu))
    assert np.array_equal(t.cpu().numpy(), out) and np.array_equal(view.cpu().numpy(), cref)
    assert torch.equal(big[:, c.shape[1]:], before[:, c.shape[1]:])


def test_fork_bounds(gpu):
    c = torch.zeros(1, 8, 64, dtype=torch.uint8, device=gpu)
    pt, lens = i32([[0, 99, -1], [2, 3, 4]], gpu), i32([20, 1000], gpu)
    for parents, reserve, code, row in [([5], [0], 7, [-1, -1, -1]), ([-2], [0], 7, [-1, -1, -1]), ([1], [0], 5, [2, 3, 4]),
                                        ([0], [0], 6, [0, -1, -1]), ([0], [0], 6, [0, -1, -1])]:
        err = i32([0], gpu)
        t, _ = KV.fork_pages(c, pt, lens, i32(parents, gpu), i32(reserve, gpu), error_word=err)
        assert int(err) == code and t.tolist() == [row]
    err = i32([0], gpu)
    t, n = KV.fork_pages(c, i32([[1, -1, -1]], gpu), i32([3], gpu), i32([0], gpu), i32([100], gpu), error_word=err)
    assert int(err) == 4 and t.tolist() == [[1, 0, 2]] and n.tolist() == [3]
    # lengths below zero are empty rows, no reservation
    t, n = KV.fork_pages(c, i32([[1, 2, 3]], gpu), i32([-5], gpu), i32([0, 0], gpu))
    assert t.tolist() == [[-1] * 3] * 2 and n.tolist() == [0, 0]


def test_fork_no_caches_and_replay(gpu):
    """Tables alone, captured: a replay on the tables it wrote before gives the next step's."""
    c = torch.empty(0, 50, 64, dtype=torch.uint8, device=gpu)
    k = KV.lib()
    pt, lens = i32([[4, -1, -1, -1]] * 2, gpu), i32([10, 0], gpu)
    ws = torch.empty(k.kv_pages_workspace_bytes(50, 2), dtype=torch.uint8, device=gpu)
    parents, reserve = i32([0, 0], gpu), i32([1, 1], gpu)
    KV.fork_pages(torch.empty(1, 50, 64, dtype=torch.uint8, device=gpu), pt, lens, parents, reserve)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        t, n = KV.fork_pages(torch.empty(1, 50, 64, dtype=torch.uint8, device=gpu), pt, lens, parents, reserve, workspace=ws)
    g.replay()
    assert t.tolist() == [[4, -1, -1, -1], [0, -1, -1, -1]] and n.tolist() == [10, 10]
    lens.copy_(i32([16, 3], gpu))
    g.replay()
    assert t.tolist() == [[4, 0, -1, -1], [4, 1, -1, -1]] and n.tolist() == [16, 16]


@pytest.mark.parametrize("seqs,longest,extra", [(1, 1, 3), (4, 100, 40), (40, 300, 500), (3, 16, 0), (600, 40, 6000),
                                                  (1100, 400, 4000), (9, 100, 40000)])
def test_compact(gpu, seqs, longest, extra):
    for seed in range(3):
        rng = np.random.default_rng(seed * 77 + seqs)
        c, pt, lens, _, _ = fork_case(rng, seqs, 1, longest, extra)
        out, U, cref = R.compact(c, pt, lens)
        for in_place in (False, True):
            cd, td = torch.from_numpy(c).to(gpu), i32(pt, gpu)
            t, used = KV.compact_pages(cd, td, i32(lens, gpu), out=td if in_place else None)
            assert int(used) == U and np.array_equal(t.cpu().numpy(), out)
            assert np.array_equal(cd.cpu().numpy()[:, :U], cref[:, :U])
            # nothing but the pages moved to is written
            assert np.array_equal(cd.cpu().numpy()[:, U:], c[:, U:])


def test_compact_bad_entries(gpu):
    c = torch.arange(8, dtype=torch.int32, device=gpu)[None, :, None].repeat(2, 1, 4)
    err = i32([0], gpu)
    t, used = KV.compact_pages(c, i32([[7, 100, 5], [-3, 6, 1]], gpu), i32([48, 20], gpu), error_word=err)
    assert int(err) == 6 and int(used) == 3 and t.tolist() == [[2, -1, 0], [-1, 1, -1]]
    assert c[1, :3, 0].tolist() == [5, 6, 7]


# ---------------------------------------------------------------- together

def test_prompt_fork_decode_compact(gpu):
    """Prompts written to the 4-bit pages and attended, forked into samples, three decode steps with the page
    operators between them, some samples dropped and the pool compacted: every step's attention against the values
    the cache holds."""
    rng = np.random.default_rng(20)
    nq, nkv, pool, mp = 12, 2, 64, 8
    scale = D ** -0.5
    f = torch.from_numpy(A.rope_inv_freq(64, 1e6)).to(gpu)
    caches = torch.randint(0, 256, (2, pool, nkv, 1152), dtype=torch.uint8, device=gpu)
    kc, vc = caches[0], caches[1]
    lens = [37, 5, 16]
    T = sum(lens)
    table, _ = KV.fork_pages(caches, torch.full((1, mp), -1, dtype=torch.int32, device=gpu), i32([0], gpu),
                             i32([-1, -1, -1], gpu), i32(lens, gpu))       # empty rows with room for the prompts
    assert table[0, :3].tolist() == [0, 1, 2] and table[2].tolist() == [4] + [-1] * 7
    pos = [i for n in lens for i in range(n)]
    seq = [s for s, n in enumerate(lens) for _ in range(n)]
    qkv = normal_bf16(rng, T, (nq + 2 * nkv) * D).to(gpu)
    q, k = KV.kv4_rope_write(qkv, i32(pos, gpu), i32(seq, gpu), table, kc, vc, nq, 64, f, keys=True)
    v = qkv.unflatten(1, (nq + 2 * nkv, D))[:, nq + nkv:]
    cu = i32(np.concatenate([[0], np.cumsum(lens)]), gpu)
    out = A.prompt_packed(q, k, v, cu, scale)[0]
    at = 0
    held = []                                              # values each sample's cache must hold
    for n in lens:
        ref, tol = R.attend(f64(q[at:at + n]), f64(k[at:at + n]), f64(v[at:at + n]), np.arange(1, n + 1), scale)
        assert (np.abs(f64(out[at:at + n]) - ref) <= tol).all()
        held.append([R.values(*R.quantise(x[at:at + n].float().cpu().numpy())) for x in (k, v)])
        at += n
    n = i32(lens, gpu)
    parents = [0, 0, 1, 1, 1, 2]
    for step in range(3):
        rows = len(parents)
        table, n = KV.fork_pages(caches, table, n, i32(parents, gpu), i32([1] * rows, gpu))
        held = [[x.copy() for x in held[p]] for p in parents]
        x = normal_bf16(rng, rows, (nq + 2 * nkv) * D).to(gpu)
        lens_out = torch.empty(rows, dtype=torch.int32, device=gpu)
        q, k = KV.kv4_rope_write(x, n, None, table, kc, vc, nq, 64, f, keys=True, seq_lens_out=lens_out)
        n = lens_out
        out = KV.kv4_decode(q, kc, vc, table, n, scale)[0]
        for b in range(rows):
            for i, new in enumerate((k, x.unflatten(1, (nq + 2 * nkv, D))[:, nq + nkv:])):
                held[b][i] = np.concatenate([held[b][i], R.values(*R.quantise(new[b:b + 1].float().cpu().numpy()))])
            ref, tol = R.attend(f64(q[b:b + 1]), held[b][0], held[b][1], [len(held[b][0])], scale)
            assert (np.abs(f64(out[b:b + 1]) - ref) <= tol).all()
        parents = [[5, 1, 1, 3], [0, 2, 3], []][step]
        if step == 1:
            table, used = KV.compact_pages(caches, table, n)
            caches[:, int(used):] = 255                    # given up
    r = i32([0, 1, 2], gpu)
    kr, vr = KV.kv4_read_rows(kc, vc, n - 1, r, table)
    for b in range(3):
        np.testing.assert_array_equal(f64(kr[b]), held[b][0][-1])
        np.testing.assert_array_equal(f64(vr[b]), held[b][1][-1])


def test_tensors_on_the_host_are_refused(gpu):
    """One tensor that is not on the device, in every place, is refused before anything is launched."""
    cpu = torch.device("cpu")
    c = KV.kv4_cache(4, 1, gpu)
    z = lambda *n: torch.zeros(*n, dtype=torch.int32, device=gpu)
    q = torch.zeros(2, 4, D, dtype=torch.bfloat16, device=gpu)
    calls = [
        (KV.kv4_rope_write, [torch.zeros(2, 6 * D, dtype=torch.bfloat16, device=gpu), z(2), z(2), z(2, 4), c, c, 4, 64,
                             torch.zeros(32, device=gpu)]),
        (KV.kv4_read_rows, [c, c, z(2), z(2), z(2, 4)]),
        (KV.kv4_decode, [q, c, c, z(2, 4), z(2), 0.1, z(2)]),
        (A.prompt_packed, [q, q, q, z(2), 0.1]),
        (KV.fork_pages, [c[None], z(2, 4), z(2), z(2), z(2)]),
        (KV.compact_pages, [c[None], z(2, 4), z(2), z(2, 4)]),
    ]
    for call, args in calls:
        for i, a in enumerate(args):
            if isinstance(a, torch.Tensor):
                with pytest.raises(ValueError, match="device|beside"):
                    call(*args[:i], a.to(cpu), *args[i + 1:])
        call(*args)
    torch.cuda.synchronize()


@pytest.mark.parametrize("split", [128, 16])
@pytest.mark.parametrize("where", ["q", "k", "v", "v one group", "v one group of zeros"])
def test_decode_nan_reaches_the_quantised_rows(gpu, where, split):
    """What is NaN in the bf16 rows is NaN in the e4m3 rows, rows that are NaN throughout among them, with one split and with
    several; the rest keeps its codes and scales."""
    rng = np.random.default_rng(split)
    nq, n = 6, 100
    kc, vc = random_cache(rng, 16, 1)
    if where == "v one group of zeros":
        vc[...] = 0                                        # scales of 0
    pt = i32([[0, 1, 2, 3, 4, 5, 6, 15], list(range(7, 15))], gpu)
    q = normal_bf16(rng, 2, nq, D)
    run = lambda: KV.kv4_decode(q.to(gpu), torch.from_numpy(kc).to(gpu), torch.from_numpy(vc).to(gpu), pt, i32([n, n], gpu),  # noqa: E731
                                0.1, split_tokens=split, quant=True)
    clean = run()
    hit = np.zeros((2, nq, D), bool)
    nan = [0xC0, 0x7F]
    at = R.CODE_BYTES + 8 * 4                              # scales of token 4 of a page
    if where == "q":
        q[0, 1, 7] = float("nan")
        hit[0, 1] = True
    elif where == "k":
        kc[3, 0, at + 2:at + 4] = nan
        hit[0] = True
    elif where == "v":
        vc[3, 0, at:at + 8] = nan * 4
        hit[0] = True
    else:
        vc[3, 0, at + 2:at + 4] = nan
        hit[0, :, 32:64] = True
    out, oq, os_ = run()
    hit = torch.from_numpy(hit).to(gpu)
    assert torch.equal(torch.isnan(out), hit)
    held = oq.view(torch.float8_e4m3fn).double().reshape(2, nq, D) * os_[:, :2].double().t()[..., None]
    assert torch.equal(torch.isnan(held), hit)
    rest = ~hit.any(dim=2)
    assert torch.equal(oq.view(2, nq, D)[rest], clean[1].view(2, nq, D)[rest])
    assert torch.equal(os_[:, :2].t()[rest], clean[2][:, :2].t()[rest])


@pytest.mark.parametrize("nq,nkv,B,split", [(12, 1, 50, 16), (96, 8, 7, 32)])
def test_decode_row_bits_do_not_depend_on_a_large_batch(gpu, nq, nkv, B, split):
    """Rows of one to thirty splits alone and in a batch whose rows fill the GPU: the bf16 rows, the e4m3 rows and their
    fp32 scales."""
    rng = np.random.default_rng(B)
    lens = [int(x) for x in rng.integers(1, 30 * split, B)]
    lens[0], lens[1], lens[2] = 30 * split, 20 * split + 1, 1
    pool = sum(map(R.pages, lens))
    kc, vc = random_cache(rng, pool, nkv)
    kd, vd = torch.from_numpy(kc).to(gpu), torch.from_numpy(vc).to(gpu)
    pt = i32(table_of(rng, lens, pool), gpu)
    q = normal_bf16(rng, B, nq, D).to(gpu)
    assert B * nq > 4 * 148 > 6 * nq
    out, oq, os_ = KV.kv4_decode(q, kd, vd, pt, i32(lens, gpu), 0.1, split_tokens=split, quant=True)
    for b in range(B):
        for rows in ([b], [b] * 5):
            one, one_q, one_s = KV.kv4_decode(q[rows], kd, vd, pt, i32([lens[i] for i in rows], gpu), 0.1,
                                              row_seq=i32(rows, gpu), split_tokens=split, quant=True)
            assert torch.equal(one[-1], out[b]) and torch.equal(one_q[-1], oq[b])
            assert torch.equal(one_s[:, len(rows) - 1], os_[:, b])
    # and where one split holds the context, whether there is a second or not
    short = i32([min(n, split) for n in lens], gpu)
    a = KV.kv4_decode(q, kd, vd, pt, short, 0.1, split_tokens=split, max_splits=1, quant=True)
    b = KV.kv4_decode(q, kd, vd, pt, short, 0.1, split_tokens=split, quant=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.equal(a[2][:, :B], b[2][:, :B])


@pytest.mark.parametrize("split", [64, 16])
def test_decode_quantised_rows_of_tiny_values(gpu, split):
    """Rows whose 448 / max is past the fp32 range: zeros stay zeros, the rest within half an e4m3 step."""
    rng = np.random.default_rng(15)
    nq, n = 6, 50
    for mag in (1e-36, 2.0 ** -125):
        x = np.zeros((n, D), np.float32)
        x[:, :64] = np.sign(rng.standard_normal((n, 64))) * mag
        kc, vc = random_cache(rng, 4, 1)
        for t, (codes, s) in enumerate(zip(*R.quantise(x))):
            R.store(vc[t // PAGE, 0], "v", t % PAGE, codes, s)
        q = normal_bf16(rng, 1, nq, D).to(gpu)
        out, oq, os_ = KV.kv4_decode(q, torch.from_numpy(kc).to(gpu), torch.from_numpy(vc).to(gpu), i32([[0, 1, 2, 3]], gpu),
                                     i32([n], gpu), 0.1, split_tokens=split, quant=True)
        got = out.double()
        held = oq.view(torch.float8_e4m3fn).double().reshape(1, nq, D) * os_[:, :1].double().t()[..., None]
        # the scale is a subnormal number, half of 2^-149 off; the row's bf16 rounding may be of one, too
        amax = got.abs().amax(dim=2, keepdim=True) * (1 + 2.0 ** -7) + 2.0 ** -134
        tol = (2.0 ** -4 + 2.0 ** -7) * got.abs() + amax / 448 * 2.0 ** -10 * 1.01 + 448 * 2.0 ** -150 + 2.0 ** -134
        assert not held[..., 64:].any() and ((held - got).abs() <= tol).all()


def test_streams_of_another_device_are_refused(gpu):
    """Launches on another device's stream would run there on this one's tensors.  A stand-in has what is asked of a stream."""
    other = type("Stream", (), {"device_index": 1, "cuda_stream": 0})()
    c = KV.kv4_cache(4, 1, gpu)
    z = lambda *n: torch.zeros(*n, dtype=torch.int32, device=gpu)
    q = torch.zeros(2, 4, D, dtype=torch.bfloat16, device=gpu)
    for call in (lambda s: KV.kv4_rope_write(torch.zeros(2, 6 * D, dtype=torch.bfloat16, device=gpu), z(2), z(2), z(2, 4), c, c, 4,
                                             64, torch.zeros(32, device=gpu), stream=s),
                 lambda s: KV.kv4_read_rows(c, c, z(2), z(2), z(2, 4), stream=s),
                 lambda s: KV.kv4_decode(q, c, c, z(2, 4), z(2), 0.1, stream=s),
                 lambda s: A.prompt_packed(q, q, q, z(2), 0.1, stream=s),
                 lambda s: KV.fork_pages(c[None], z(2, 4), z(2), z(2), stream=s),
                 lambda s: KV.compact_pages(c[None], z(2, 4), z(2), stream=s)):
        with pytest.raises(ValueError, match="stream"):
            call(other)
        call(torch.cuda.Stream(gpu))
        torch.cuda.synchronize()                           # before the call's tensors go


@pytest.mark.parametrize("nq,nkv,lens", [(12, 1, [300, 1, 2000]), (16, 8, [700])])
def test_decode_under_a_table_much_wider_than_the_contexts(gpu, nq, nkv, lens):
    """Room for 131072 tokens a row, the split that goes by it, and what is behind a row's pages not looked at."""
    rng = np.random.default_rng(nkv)
    pool = sum(map(R.pages, lens)) + 3
    kc, vc = random_cache(rng, pool, nkv)
    pt = np.full((len(lens), 8192), 1 << 30, np.int32)
    narrow = table_of(rng, lens, pool)
    for b, n in enumerate(lens):
        pt[b, :R.pages(n)] = narrow[b, :R.pages(n)]
    q = normal_bf16(rng, len(lens), nq, D)
    err = i32([0], gpu)
    out = f64(KV.kv4_decode(q.to(gpu), torch.from_numpy(kc).to(gpu), torch.from_numpy(vc).to(gpu), i32(pt, gpu), i32(lens, gpu),
                            D ** -0.5, error_word=err)[0])
    assert int(err) == 0
    for b, n in enumerate(lens):
        ref, tol = R.attend(f64(q[b:b + 1]), seq_values(kc, "k", pt[b], n), seq_values(vc, "v", pt[b], n), [n], D ** -0.5)
        assert (np.abs(out[b] - ref[0]) <= tol[0]).all()
