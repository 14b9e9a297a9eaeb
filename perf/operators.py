"""Workloads of the serving operators: attention over packed prompts, the
4-bit KV cache (write with RoPE, read back, decode attention) and the page
operators (fork, compact).

`own` false: every operator in plain torch operations, in 32 bits, rounded
once at the end.  `own` true: the package's own entry points on the same data.

4-bit page of one kv head (1152 bytes; K and V in caches of their own,
uint8 [pages][nkv][1152]): 16 tokens x 128 dims of codes n + 8 (n in -8..7),
then bf16 scales [token][4], one per 32 dims; the value is n * scale.
K codes: dim 32 j + 8 w + i of a token at byte token*64 + w*16 + j*4 + i/2.
V codes: dim 32 j + 4 g + i of token 8 a + 2 w + b at byte
a*512 + (4 g + w)*16 + b*8 + 2 j + i/2.  Even i: the low half of the byte.
"""
import random

import torch

own = False

D, PAGE, GROUP = 128, 16, 32
CODES = PAGE * D // 2
PAGE4 = CODES + PAGE * (D // GROUP) * 2


# ---------------------------------------------------------------- cases

def listed():
    return [
        # chat prompts of one to a few hundred tokens arriving together, one tensor-parallel rank of eight
        {"name": "prompt_short_mix", "op": "prompt", "seqs": 24, "longest": 201, "nq": 12, "nkv": 1, "mix": 1},
        # a packed prefill batch of uneven prompts, all heads on one GPU
        {"name": "prompt_packed_96h", "op": "prompt", "seqs": 7, "longest": 1201, "nq": 96, "nkv": 8, "mix": 2},
        # one long document, one rank of eight
        {"name": "prompt_long", "op": "prompt", "seqs": 1, "longest": 16384, "nq": 12, "nkv": 1, "mix": 3},
        # the new tokens of a decode step, 64 sequences, all heads
        {"name": "kv4_write_step", "op": "write", "seqs": 64, "longest": 1, "past": 8191, "nq": 96, "nkv": 8, "mix": 4},
        # a prefill forward of several prompts
        {"name": "kv4_write_prefill", "op": "write", "seqs": 5, "longest": 2047, "past": 300, "nq": 96, "nkv": 8, "mix": 5},
        # decode with a few short contexts: latency
        {"name": "kv4_decode_few", "op": "decode", "seqs": 4, "longest": 500, "nq": 12, "nkv": 1, "mix": 6},
        # decode of one rank of eight: 64 sequences up to 32K tokens
        {"name": "kv4_decode_64x32k", "op": "decode", "seqs": 64, "longest": 32768, "nq": 12, "nkv": 1, "mix": 7},
        # decode with all heads on one GPU, odd lengths
        {"name": "kv4_decode_16x8k_96h", "op": "decode", "seqs": 16, "longest": 8191, "nq": 96, "nkv": 8, "mix": 8},
        # parallel samples of a few requests: tables mostly, few pages copied
        {"name": "fork_small", "op": "fork", "seqs": 4, "out": 8, "longest": 300, "caches": 6, "page_bytes": 1152, "mix": 9},
        # a beam step over all layers of a bf16 cache
        {"name": "fork_beam_184", "op": "fork", "seqs": 32, "out": 64, "longest": 700, "caches": 184, "page_bytes": 4096, "mix": 10},
        # a small pool after a few requests ended
        {"name": "compact_small", "op": "compact", "seqs": 6, "longest": 200, "caches": 6, "page_bytes": 1152, "mix": 11},
        # a fragmented 4-bit pool over all layers
        {"name": "compact_92", "op": "compact", "seqs": 24, "longest": 1000, "caches": 92, "page_bytes": 9216, "mix": 12},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "write", "decode", "decode", "fork", "compact"])
    c = {"op": op, "mix": rng.randrange(1 << 20)}
    if op in ("prompt", "write", "decode"):
        c["nkv"] = rng.choice([1, 2, 4, 8])
        c["nq"] = c["nkv"] * rng.choice([1, 2, 4, 7, 8, 12, 16])
    if op == "prompt":
        # padded plain scores: seqs * nq * longest^2 at most those of the longest listed prompt
        top = int((12 * 16384 ** 2 / c["nq"]) ** 0.5)
        c["longest"] = _spread(rng, 1, min(16384, top))
        c["seqs"] = _spread(rng, 1, max(1, min(64, 12 * 16384 ** 2 // (c["nq"] * c["longest"] ** 2))))
    elif op == "write":
        c["longest"] = _spread(rng, 1, 2048)
        c["seqs"] = _spread(rng, 1, max(1, min(128, 8192 // c["longest"])))
        c["past"] = _spread(rng, 1, 8192)
    elif op == "decode":
        c["longest"] = _spread(rng, 1, 32768)
        c["seqs"] = _spread(rng, 1, max(1, min(64, 64 * 32768 // (c["nkv"] * c["longest"]))))
    else:
        c["seqs"] = _spread(rng, 1, 32)
        c["longest"] = _spread(rng, 1, 1000)
        c["page_bytes"] = rng.choice([1152, 2304, 4096, 9216])
        c["caches"] = _spread(rng, 1, 92)
        if op == "fork":
            c["out"] = _spread(rng, 1, 64)
    return c


def _lens(case):
    """Lengths of the case's sequences: the first the longest, the others spread over the logarithm below it, or,
    for contexts in decode, evenly from a thirty-second of it on."""
    rng = random.Random(case["mix"])
    if case["op"] == "decode":
        return [case["longest"]] + [rng.randint(max(1, case["longest"] // 32), case["longest"]) for _ in range(case["seqs"] - 1)]
    return [case["longest"]] + [_spread(rng, 1, case["longest"]) for _ in range(case["seqs"] - 1)]


def _pages(n):
    return -(-n // PAGE)


def _fork_plan(case):
    """(lengths, parents, tokens each child will append): parents repeat, some are left without a child, and one
    child in eight is an empty row."""
    lens = _lens(case)
    rng = random.Random(case["mix"] + 1)
    parents = [rng.randrange(-(case["seqs"] // 8) - 1, case["seqs"]) for _ in range(case["out"])]
    parents = [max(-1, p) for p in parents]
    if all(p < 0 for p in parents):
        parents[0] = 0
    return lens, parents, [rng.choice([0, 1, 1, 1, 5, 40]) for _ in parents]


def _max_pages(case):
    return _pages(case["longest"] + 40) + 1


def _pool(case):
    """Pages of the pool: those in use, room for the children, and as many again that other requests left."""
    used = sum(map(_pages, _lens(case)))
    return used + (case["out"] * 4 if case["op"] == "fork" else 0) + used * 2 // 3 + 3


def work(case):
    lens = _lens(case)
    if case["op"] == "prompt":
        T = sum(lens)
        return {"bytes": T * (2 * case["nq"] + 2 * case["nkv"]) * D * 2,
                "flops": 4 * D * case["nq"] * sum(n * (n + 1) // 2 for n in lens)}
    if case["op"] == "write":
        T, nq, nkv = sum(lens), case["nq"], case["nkv"]
        # qkv in; q, rotated k out; pages out; pages in; k and v rows out
        return {"bytes": T * ((nq + 2 * nkv) * 256 + nq * 256 + nkv * 256 + 2 * nkv * 144 + 2 * nkv * 256), "flops": 0}
    if case["op"] == "decode":
        return {"bytes": sum(lens) * case["nkv"] * 144 + 2 * len(lens) * case["nq"] * 256,
                "flops": 4 * D * case["nq"] * sum(lens)}
    mp = _max_pages(case)
    if case["op"] == "fork":
        lens, parents, reserve = _fork_plan(case)
        # every child of a parent with a page in part filled that appends writes into it: all but one copy it
        writers = {}
        for p, r in zip(parents, reserve):
            if p >= 0 and r > 0 and lens[p] % PAGE:
                writers[p] = writers.get(p, 0) + 1
        copies = sum(n - 1 for n in writers.values())
        tables = 4 * mp * (case["seqs"] + case["out"])
        return {"bytes": 2 * copies * case["caches"] * case["page_bytes"] + tables, "flops": 0}
    used = sum(map(_pages, lens))
    ids = random.Random(case["mix"] + 2).sample(range(_pool(case)), used)
    moved = sum(i >= used for i in ids)
    return {"bytes": 2 * moved * case["caches"] * case["page_bytes"] + 8 * mp * case["seqs"], "flops": 0}


# ---------------------------------------------------------------- inputs

def _table(lens, max_pages, ids, dev):
    """Page table [seqs][max_pages] over the given page ids, -1 behind each sequence's pages."""
    rows, at = [], 0
    for n in lens:
        rows.append(ids[at:at + _pages(n)] + [-1] * (max_pages - _pages(n)))
        at += _pages(n)
    return torch.tensor(rows, dtype=torch.int32, device=dev)


def _i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _random_cache(pages, nkv, gen, dev):
    """A 4-bit cache as quantised normal values fill it: codes around 8, scales within a factor of four."""
    n = torch.randn(pages, nkv, 2 * CODES, generator=gen, device=dev).mul_(2.7).round_().clamp_(-8, 7).add_(8).to(torch.uint8)
    codes = n[..., :CODES] | (n[..., CODES:] << 4)
    s = torch.rand(pages, nkv, PAGE * (D // GROUP), generator=gen, device=dev).mul_(2).exp2_().mul_(0.2)
    s = _up4(s).to(torch.bfloat16)
    return torch.cat([codes, s.view(torch.uint8)], dim=-1)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    lens = _lens(case)
    s = dict(case)
    if case["op"] == "prompt":
        T, nq, nkv = sum(lens), case["nq"], case["nkv"]
        qkv = torch.randn(T, (nq + 2 * nkv) * D, generator=gen, device=dev).to(torch.bfloat16)
        s["q"] = qkv[:, :nq * D].reshape(T, nq, D).contiguous()
        s["k"] = qkv[:, nq * D:(nq + nkv) * D].reshape(T, nkv, D).contiguous()
        s["v"] = qkv[:, (nq + nkv) * D:].unflatten(1, (nkv, D))      # the projection's rows as they are
        s["cu"] = torch.tensor([0] + lens, device=dev).cumsum(0).to(torch.int32)
        s["longest"] = max(lens)
    elif case["op"] == "write":
        T, nq, nkv = sum(lens), case["nq"], case["nkv"]
        rng = random.Random(seed)
        past = [rng.randrange(case["past"]) for _ in lens]
        ends = [p + n for p, n in zip(past, lens)]
        pool = sum(map(_pages, ends)) + 3
        s["qkv"] = torch.randn(T, (nq + 2 * nkv) * D, generator=gen, device=dev).to(torch.bfloat16)
        s["positions"] = _i32([p + i for p, n in zip(past, lens) for i in range(n)], dev)
        s["row_seq"] = _i32([b for b, n in enumerate(lens) for _ in range(n)], dev)
        s["table"] = _table(ends, max(map(_pages, ends)) + 2, rng.sample(range(pool), sum(map(_pages, ends))), dev)
        s["k_cache"] = torch.zeros(pool, nkv, PAGE4, dtype=torch.uint8, device=dev)
        s["v_cache"] = torch.zeros_like(s["k_cache"])
        i = torch.arange(32, dtype=torch.float64, device=dev)
        s["inv_freq"] = (1e6 ** (-2.0 * i / 64)).float()
    elif case["op"] == "decode":
        nq, nkv = case["nq"], case["nkv"]
        pool = sum(map(_pages, lens)) + 5
        ids = random.Random(seed).sample(range(pool), sum(map(_pages, lens)))
        s["q"] = torch.randn(len(lens), nq, D, generator=gen, device=dev).to(torch.bfloat16)
        s["k_cache"] = _random_cache(pool, nkv, gen, dev)
        s["v_cache"] = _random_cache(pool, nkv, gen, dev)
        s["table"] = _table(lens, max(map(_pages, lens)) + 1, ids, dev)
        s["lens"] = _i32(lens, dev)
    else:
        pool = _pool(case)
        # the ids follow from the case, so that every seed moves as many pages
        ids = random.Random(case["mix"] + 2).sample(range(pool), sum(map(_pages, lens)))
        s["caches"] = torch.randint(0, 256, (case["caches"], pool, case["page_bytes"]), dtype=torch.uint8, generator=gen,
                                    device=dev)
        s["table"] = _table(lens, _max_pages(case), ids, dev)
        s["lens"] = _i32(lens, dev)
        if case["op"] == "fork":
            _, parents, reserve = _fork_plan(case)
            s["parents"], s["reserve"] = _i32(parents, dev), _i32(reserve, dev)
    return s


# ---------------------------------------------------------------- plain forms

def _up4(x):
    """fp32 rounded up to four significant bits."""
    return ((x.view(torch.int32) + 0x000FFFFF) & ~0x000FFFFF).view(torch.float32)


def _quantise(x):
    """bf16 values [...][128] -> (codes 0..15 [...][4][32], scales bf16 [...][4])."""
    x = x.float().unflatten(-1, (D // GROUP, GROUP))
    a = x.abs().amax(dim=-1)
    s = _up4(a / torch.full_like(a, 7.5)).clamp_min(2.0 ** -126)
    n = torch.round(x / s.unsqueeze(-1)).clamp(-8, 7)
    bad = ~(a < 2.0 ** 120)
    codes = torch.where(bad.unsqueeze(-1), torch.zeros_like(n), n).add(8).to(torch.uint8)
    return codes, torch.where(bad, torch.full_like(s, float("nan")), s).to(torch.bfloat16)


def _k_bytes(codes):
    """codes [...][j 4][w 4 x i 8] -> bytes [...][64] in a token's order."""
    c = codes.unflatten(-1, (4, 4, 2))                       # j, w, i/2, i%2
    return (c[..., 0] | (c[..., 1] << 4)).transpose(-3, -2).flatten(-3)


def _v_bytes(codes):
    """codes [...][j 4][g 8 x i 4] -> bytes [...][g 8][8]: a token's share of each g."""
    c = codes.unflatten(-1, (8, 2, 2))                       # j, g, i/2, i%2
    return (c[..., 0] | (c[..., 1] << 4)).transpose(-3, -2).flatten(-2)


def _halves(b):
    return torch.stack([b & 15, b >> 4], dim=-1)


def _values(codes, scales):
    """codes [...][16][128], scales [...][16][4] -> fp32 values."""
    n = codes.float() - 8
    return (n.unflatten(-1, (D // GROUP, GROUP)) * scales.float().unsqueeze(-1)).flatten(-2)


def _scales(cache):
    return cache[..., CODES:].view(torch.bfloat16).unflatten(-1, (PAGE, D // GROUP))


def _k_values(cache):
    """uint8 [...][1152] -> fp32 [...][16][128]."""
    c = _halves(cache[..., :CODES].unflatten(-1, (PAGE, 4, 4, 4)))         # token, w, j, i/2, i%2
    return _values(c.transpose(-4, -3).flatten(-4), _scales(cache))


def _v_values(cache):
    c = _halves(cache[..., :CODES].unflatten(-1, (2, 8, 4, 2, 4, 2)))      # a, g, w, b, j, i/2, i%2
    n = c.dim() - 7
    c = c.permute(*range(n), n, n + 2, n + 3, n + 4, n + 1, n + 5, n + 6)  # a, w, b, j, g, i/2, i%2
    return _values(c.flatten(-4).flatten(-4, -2), _scales(cache))


def _plain_prompt(s):
    q, k, v, cu, S = s["q"], s["k"], s["v"], s["cu"].long(), s["longest"]
    T, nq, _ = q.shape
    nkv = k.shape[1]
    at = cu[:-1, None] + torch.arange(S, device=q.device)                  # [seqs][S] rows, past the end clamped
    at = at.clamp_max(T - 1)
    qp = q[at].float().unflatten(2, (nkv, nq // nkv))                      # [b][S][nkv][G][D]
    kp, vp = k[at].float(), v[at].float()
    x = torch.matmul(qp.permute(0, 2, 3, 1, 4), kp.permute(0, 2, 3, 1).unsqueeze(2)) * D ** -0.5
    x.masked_fill_(torch.ones(S, S, dtype=torch.bool, device=q.device).triu(1), float("-inf"))
    x.sub_(x.amax(dim=-1, keepdim=True)).exp_()
    o = torch.matmul(x, vp.permute(0, 2, 1, 3).unsqueeze(2)) / x.sum(dim=-1, keepdim=True)
    o = o.permute(0, 3, 1, 2, 4).reshape(-1, nq, D)                        # [b * S][nq][D]
    r = torch.arange(T, device=q.device)
    b = torch.searchsorted(cu, r, right=True) - 1
    return o[b * S + r - cu[b]].to(torch.bfloat16)


def _plain_write(s):
    qkv, nq, nkv = s["qkv"], s["nq"], s["nkv"]
    f = s["inv_freq"]
    x = qkv.float().unflatten(1, (nq + 2 * nkv, D))
    # the angle is the fp32 product of the position and the frequency
    ang = s["positions"].float()[:, None, None] * f
    cs, sn = torch.cos(ang), torch.sin(ang)
    h = f.numel()
    a, b = x[:, :nq + nkv, :h], x[:, :nq + nkv, h:2 * h]
    rot = torch.cat([a * cs - b * sn, a * sn + b * cs, x[:, :nq + nkv, 2 * h:]], dim=-1).to(torch.bfloat16)
    q, k, v = rot[:, :nq], rot[:, nq:], qkv.unflatten(1, (nq + 2 * nkv, D))[:, nq + nkv:]
    pos = s["positions"].long()
    page, t = s["table"][s["row_seq"].long(), pos // PAGE].long(), pos % PAGE
    (kc, ks), (vc, vs) = _quantise(k), _quantise(v)
    s["k_cache"][..., :CODES].unflatten(-1, (PAGE, 64))[page, :, t] = _k_bytes(kc)
    s["v_cache"][..., :CODES].unflatten(-1, (2, 8, 4, 2, 8))[page, :, t // 8, :, t % 8 // 2, t % 2] = _v_bytes(vc)
    _scales(s["k_cache"])[page, :, t] = ks
    _scales(s["v_cache"])[page, :, t] = vs
    # read the rows back out of the pages
    r = torch.arange(pos.numel(), device=pos.device)
    kr = _k_values(s["k_cache"][page])[r, :, t].to(torch.bfloat16)
    vr = _v_values(s["v_cache"][page])[r, :, t].to(torch.bfloat16)
    return q.contiguous(), k.contiguous(), kr, vr


def _plain_decode(s):
    q, table, lens = s["q"], s["table"].long().clamp_min(0), s["lens"].long()
    nkv = s["k_cache"].shape[1]
    k = _k_values(s["k_cache"])[table].transpose(1, 2).flatten(2, 3)       # [b][nkv][positions][D]
    x = torch.matmul(q.float().unflatten(1, (nkv, -1)), k.transpose(2, 3)) * D ** -0.5
    out = torch.arange(x.shape[-1], device=q.device) >= lens[:, None, None, None]
    x.masked_fill_(out, float("-inf"))
    x.sub_(x.amax(dim=-1, keepdim=True)).exp_()
    v = _v_values(s["v_cache"])[table].transpose(1, 2).flatten(2, 3)
    o = torch.matmul(x, v) / x.sum(dim=-1, keepdim=True)
    return o.flatten(1, 2).to(torch.bfloat16)


def _plain_fork(s):
    caches, table, parents, reserve = s["caches"], s["table"].long(), s["parents"].long(), s["reserve"].long()
    pool, mp, dev = caches.shape[1], table.shape[1], table.device
    n = torch.where(parents >= 0, s["lens"].long()[parents.clamp_min(0)], 0)
    have, need = (n + PAGE - 1) // PAGE, (n + reserve + PAGE - 1) // PAGE
    j, i = torch.arange(mp, device=dev), torch.arange(parents.numel(), device=dev)
    tab = table[parents.clamp_min(0)]
    held = j < have[:, None]
    last = j == have[:, None] - 1
    writes = ((reserve > 0) & (n % PAGE != 0))[:, None] & last
    # who may keep a page: the child with the most tokens in it, a writer before a reader, the lowest row
    key = ((n[:, None] - PAGE * j).clamp(0, PAGE) << 41) | (writes.long() << 40) | ((1 << 40) - 1 - i[:, None])
    keys = torch.zeros(pool + 1, dtype=torch.int64, device=dev)
    at = torch.where(held, tab, pool)
    keys.scatter_reduce_(0, at.flatten(), key.flatten(), "amax")
    copy = writes & (keys[at] != key)
    fresh = copy | ((j >= have[:, None]) & (j < need[:, None]))
    free = keys[:pool] == 0
    ids = torch.zeros(pool + 1, dtype=torch.int64, device=dev)
    ids[torch.where(free, free.cumsum(0) - 1, pool)] = torch.arange(pool, device=dev)
    new = ids[(fresh.flatten().cumsum(0) - 1).clamp(0, pool - 1)].view_as(fresh)
    out = torch.where(fresh, new, torch.where(held, tab, -1))
    r, c = torch.nonzero(copy, as_tuple=True)
    caches[:, out[r, c]] = caches[:, tab[r, c]]
    return out.to(torch.int32), n.to(torch.int32), caches


def _plain_compact(s):
    caches, table = s["caches"], s["table"].long()
    pool, dev = caches.shape[1], table.device
    held = torch.arange(table.shape[1], device=dev) < ((s["lens"].long() + PAGE - 1) // PAGE)[:, None]
    used = torch.zeros(pool + 1, dtype=torch.bool, device=dev)
    used[torch.where(held, table, pool)] = True
    used = used[:pool]
    count = used.sum()
    p = torch.arange(pool, device=dev)
    src = torch.nonzero(used & (p >= count)).flatten()
    dst = torch.nonzero(~used & (p < count)).flatten()
    to = p.clone()
    to[src] = dst
    caches[:, dst] = caches[:, src]
    out = torch.where(held, to[table.clamp_min(0)], -1)
    return out.to(torch.int32), count.to(torch.int32).reshape(1), caches


# ---------------------------------------------------------------- one pass

def _own(s):
    from time_b200 import attn, kvcache
    if s["op"] == "prompt":
        return attn.prompt_packed(s["q"], s["k"], s["v"], s["cu"], D ** -0.5)[0]
    if s["op"] == "write":
        q, k = kvcache.kv4_rope_write(s["qkv"], s["positions"], s["row_seq"], s["table"], s["k_cache"], s["v_cache"],
                                      s["nq"], 64, s["inv_freq"], keys=True)
        kr, vr = kvcache.kv4_read_rows(s["k_cache"], s["v_cache"], s["positions"], s["row_seq"], s["table"])
        return q, k, kr, vr
    if s["op"] == "decode":
        return kvcache.kv4_decode(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], D ** -0.5)[0]
    if s["op"] == "fork":
        table, lens = kvcache.fork_pages(s["caches"], s["table"], s["lens"], s["parents"], s["reserve"])
        return table, lens, s["caches"]
    table, count = kvcache.compact_pages(s["caches"], s["table"], s["lens"])
    return table, count, s["caches"]


_PLAIN = {"prompt": _plain_prompt, "write": _plain_write, "decode": _plain_decode, "fork": _plain_fork,
          "compact": _plain_compact}


def run(state):
    return _own(state) if own else _PLAIN[state["op"]](state)


# ---------------------------------------------------------------- 64 bits

def _attend(q, k, v, causal):
    """q [n][nq][D], k and v [m][nkv][D] in 64 bits, one sequence; row i of q is position m - n + i where causal."""
    G = q.shape[1] // k.shape[1]
    o = torch.empty_like(q)
    for h in range(q.shape[1]):
        w = q[:, h] @ k[:, h // G].T / D ** 0.5
        if causal:
            w = torch.where(torch.ones_like(w, dtype=torch.bool).tril(), w, -torch.inf)
        o[:, h] = torch.softmax(w, dim=1) @ v[:, h // G]
    return o


def _read64(cache, which, table, n):
    """The first n positions of one sequence out of its pages: [n][nkv][D] in 64 bits, by the byte formulas of the head of this file."""
    dev = cache.device
    page = cache[table[:_pages(n)].long()]                                  # [pages][nkv][1152]
    t, d = torch.arange(PAGE, device=dev)[:, None], torch.arange(D, device=dev)
    if which == "k":
        byte, i = t * 64 + d % 32 // 8 * 16 + d // 32 * 4 + d % 8 // 2, d % 2
    else:
        byte, i = t // 8 * 512 + (4 * (d % 32 // 4) + t % 8 // 2) * 16 + t % 2 * 8 + 2 * (d // 32) + d % 4 // 2, d % 2
    code = (page[:, :, byte].long() >> (4 * i)) & 15
    at = CODES + 2 * (4 * t + d // 32)
    bits = page[:, :, at].long() | (page[:, :, at + 1].long() << 8)
    scale = (bits << 16).to(torch.int32).view(torch.float32).double()
    return ((code - 8).double() * scale).transpose(1, 2).flatten(0, 1)[:n]


def exact(case, seed):
    s, lens = prepare(case, seed), _lens(case)
    if case["op"] == "prompt":
        cu, parts = 0, []
        for n in lens:
            q, k, v = (s[x][cu:cu + n].double() for x in ("q", "k", "v"))
            parts.append(_attend(q, k, v, True))
            cu += n
        return torch.cat(parts)
    if case["op"] == "write":
        nq, nkv = s["nq"], s["nkv"]
        x = s["qkv"].double().unflatten(1, (nq + 2 * nkv, D))[:, :nq + nkv]
        z = torch.polar(torch.ones((), dtype=torch.float64, device=x.device),
                        s["positions"].double()[:, None] * s["inv_freq"].double()).unsqueeze(1)
        h = s["inv_freq"].numel()
        y = torch.complex(x[..., :h], x[..., h:2 * h]) * z
        x[..., :h], x[..., h:2 * h] = y.real, y.imag
        # the nearest code has no value that nearby inputs share
        return x[:, :nq], x[:, nq:], None, None
    if case["op"] == "decode":
        return torch.cat([_attend(s["q"][b:b + 1].double(), _read64(s["k_cache"], "k", s["table"][b], n),
                                  _read64(s["v_cache"], "v", s["table"][b], n), False) for b, n in enumerate(lens)])
    return None
