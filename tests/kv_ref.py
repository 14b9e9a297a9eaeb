"""Plain 64-bit statements of the cache operators for their tests (numpy):
the 4-bit quantiser and page layout, attention, and the page operators."""
import numpy as np

D, PAGE, GROUP = 128, 16, 32
CODE_BYTES, PAGE4 = 1024, 1152


def bf16_bits(x) -> np.ndarray:
    """Bits of values that are bf16 numbers."""
    return (np.asarray(x, np.float32).view(np.uint32) >> 16).astype(np.uint16)


def quantise(x: np.ndarray):
    """x [...][128] (bf16 values) -> codes n + 8 [...][128] uint8, scales [...][4] float32 (NaN: not storable)."""
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], D // GROUP, GROUP)
    with np.errstate(invalid="ignore"):
        a = np.abs(g).max(axis=-1)
        bad = ~(a < 2.0 ** 120)
        t = np.where(bad, 1.0, a) / 7.5
        e = np.where(t > 0, np.floor(np.log2(np.where(t > 0, t, 1.0))), 0)
        s = np.maximum(np.ceil(t / 2.0 ** (e - 3)) * 2.0 ** (e - 3), 2.0 ** -126)
        n = np.clip(np.rint(np.where(bad[..., None], 0.0, g) / s[..., None]), -8, 7)   # rint: half to even
    codes = (n + 8).astype(np.uint8).reshape(x.shape)
    return codes, np.where(bad, np.nan, s).astype(np.float32)


def values(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    n = codes.astype(np.float64) - 8
    return (n.reshape(*n.shape[:-1], D // GROUP, GROUP) * scales.astype(np.float64)[..., None]).reshape(n.shape)


def code_place(which: str, t: int):
    """(byte, shift) of the 128 dims of token t inside a page."""
    d = np.arange(D)
    if which == "k":
        byte = t * 64 + d % 32 // 8 * 16 + d // 32 * 4 + d % 8 // 2
    else:
        byte = t // 8 * 512 + (4 * (d % 32 // 4) + t % 8 // 2) * 16 + t % 2 * 8 + 2 * (d // 32) + d % 4 // 2
    return byte, 4 * (d % 2)


def store(tile: np.ndarray, which: str, t: int, codes: np.ndarray, scales: np.ndarray) -> None:
    """One token into one (page, head) tile, uint8 [1152]."""
    byte, shift = code_place(which, t)
    tile[byte] = 0
    np.bitwise_or.at(tile, byte, (codes.astype(np.uint8) << shift).astype(np.uint8))
    bits = np.where(np.isnan(scales), np.uint16(0x7FC0), bf16_bits(scales))
    tile[CODE_BYTES + 8 * t:CODE_BYTES + 8 * t + 8] = bits.astype("<u2").view(np.uint8)


def load(tile: np.ndarray, which: str, t: int) -> np.ndarray:
    byte, shift = code_place(which, t)
    bits = tile[CODE_BYTES + 8 * t:CODE_BYTES + 8 * t + 8].copy().view("<u2").astype(np.uint32) << 16
    return values((tile[byte] >> shift) & 15, bits.view(np.float32))


def attend(q, k, v, limit, scale):
    """q [n][nq][D] over k, v [m][nkv][D], row i over the first limit[i] keys.  Returns the output and the bound of
    |kernel - output| for bf16 weights and outputs (64 bits)."""
    n, nq, _ = q.shape
    m, nkv, _ = k.shape
    G = nq // nkv
    out, tol = np.zeros_like(q), np.zeros_like(q)
    mask = np.arange(m)[None] < np.asarray(limit)[:, None]
    for h in range(nq):
        kh, vh = k[:, h // G], v[:, h // G]
        s = np.where(mask, q[:, h] @ kh.T * scale, -np.inf)
        # fp32 products and sums of 128 terms on the tensor cores (each at most one 2^-23 step off the largest),
        # the scale times log2(e), and exp2: the relative error of a weight
        d = 2 * (132 * 2.0 ** -23) * np.where(mask, np.abs(q[:, h]) @ np.abs(kh).T, 0).max(axis=1) * scale + 2.0 ** -20
        w = np.exp(s - s.max(axis=1, keepdims=True))
        w /= w.sum(axis=1, keepdims=True)
        out[:, h] = w @ vh
        # a weight is rounded to bf16 (2^-8 at most) but not in the sum that divides, the output once more
        size = w @ np.abs(vh)
        tol[:, h] = 2.0 ** -8 * np.abs(out[:, h]) * 1.01 + (2.0 ** -8 + 2 * d[:, None] + m * 2.0 ** -23) * size * 1.01
    return out, tol


# ---------------------------------------------------------------- pages

def pages(n: int) -> int:
    return -(-n // PAGE)


def fork(caches, table, lens, parents, reserve):
    """The result of kv_pages_fork row by row: (table, lens, caches, exhausted)."""
    caches, num_pages, mp = caches.copy(), caches.shape[1], table.shape[1]
    rows = []
    for i, p in enumerate(parents):
        n = int(lens[p]) if p >= 0 else 0
        own = [int(x) for x in table[p, :pages(n)]] if p >= 0 else []
        rows.append((n, own, min(pages(n + int(reserve[i])), mp), bool(reserve[i] > 0 and n % PAGE)))
    best = {}
    for i, (n, own, need, writes) in enumerate(rows):
        for j, id in enumerate(own):
            key = (min(n - PAGE * j, PAGE), writes and j == len(own) - 1, -i)
            best[id] = max(best.get(id, (0, False, 0)), key)
    free = [p for p in range(num_pages) if p not in best]
    at, src, dst, short = 0, [], [], False
    out = np.full((len(parents), mp), -1, np.int32)
    for i, (n, own, need, writes) in enumerate(rows):
        row = list(own)
        if writes and best[own[-1]] != (n - PAGE * (len(own) - 1), True, -i):
            new = free[at] if at < len(free) else -1
            short |= new < 0
            at += 1
            if new >= 0:
                src.append(own[-1])
                dst.append(new)
            row[-1] = new
        for _ in range(need - len(own)):
            row.append(free[at] if at < len(free) else -1)
            short |= row[-1] < 0
            at += 1
        out[i, :len(row)] = row
    caches[:, dst] = caches[:, src]
    return out, np.array([r[0] for r in rows], np.int32), caches, short


def compact(caches, table, lens):
    caches = caches.copy()
    owned = {int(table[s, j]) for s in range(len(lens)) for j in range(pages(int(lens[s])))}
    U = len(owned)
    high, low = [p for p in sorted(owned) if p >= U], [p for p in range(U) if p not in owned]
    to = {p: p for p in owned} | dict(zip(high, low))
    caches[:, low] = caches[:, high]
    out = np.full_like(table, -1)
    for s in range(len(lens)):
        for j in range(pages(int(lens[s]))):
            out[s, j] = to[int(table[s, j])]
    return out, U, caches
