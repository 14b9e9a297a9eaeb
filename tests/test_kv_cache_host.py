"""include/kv_cache.h and attn_prompt_packed without a GPU: symbols, sizes,
and the refusal of bad arguments before any CUDA call; the plain statements of
the operators against small cases worked out by hand."""
import ctypes
import re
import subprocess
from pathlib import Path

import numpy as np
import pytest

import kv_ref as R
from time_b200 import attn as A
from time_b200 import kvcache as KV

ROOT = Path(__file__).resolve().parent.parent
OK, INVALID, UNSUPPORTED, WORKSPACE = 0, 1, 3, 6
P = 1 << 20            # a 16-byte aligned address that no refused call reads


@pytest.fixture(scope="module")
def k():
    A.lib()
    return KV.lib()


def test_header_symbols_exported():
    import time_b200
    text = re.sub(r"/\*.*?\*/", " ", (ROOT / "include" / "kv_cache.h").read_text(), flags=re.S)
    names = set(re.findall(r"\b((?:attn_kv4|kv_pages)_\w+)\s*\(", text))
    assert len(names) == 9
    out = subprocess.run(["nm", "-D", "--defined-only", str(time_b200.lib_path("libkernels.so"))], capture_output=True,
                         text=True, check=True).stdout
    syms = {line.split()[-1] for line in out.splitlines()}
    assert names | {"attn_prompt_packed"} <= syms


def test_sizes(k):
    assert k.attn_kv4_page_bytes(8) == 8 * KV.PAGE4_BYTES == 8 * 1152
    assert k.attn_kv4_page_bytes(0) == 0
    assert k.attn_kv4_decode_workspace_bytes(3, 12, 5) >= 3 * 12 * 5 * 130 * 4
    assert k.attn_kv4_decode_workspace_bytes(0, 12, 5) == 0
    for B, nkv, ctx in [(1, 1, 1), (1, 1, 1 << 20), (64, 8, 32768), (5000, 8, 100)]:
        s = k.attn_kv4_split_tokens(B, nkv, ctx)
        assert s > 0 and s % 16 == 0 and s <= 8192
    assert k.kv_pages_workspace_bytes(1000, 10) >= 4 * (2 * 1000 + 10)
    assert k.kv_pages_workspace_bytes(0, 10) == 0


WRITE = dict(qkv=P, B=2, nq=4, nkv=2, d=128, rot=64, f=P, pos=P, row_seq=None, num_seqs=2, table=P, max_pages=4, page=16,
             pages=8, q=P, k_out=None, kc=P, vc=P, lens=None, err=None, stream=None)
READ = dict(kc=P, vc=P, pages=8, pos=P, row_seq=None, num_seqs=2, table=P, max_pages=4, page=16, B=2, nkv=2, d=128, k=P,
            v=P, err=None, stream=None)
DECODE = dict(q=P, kc=P, vc=P, pages=8, table=P, max_pages=4, row_seq=None, num_seqs=2, lens=P, B=2, nq=4, nkv=2, d=128,
              page=16, scale=0.1, split=64, splits=1, ws=P, ws_bytes=1 << 20, out=P, out_q=None, out_s=None, ld=4,
              err=None, stream=None)
PROMPT = dict(q=P, qs=512, k=P, ks=256, v=P, vs=256, cu=P, seqs=1, T=4, nq=4, nkv=2, d=128, scale=0.1, out=P, out_q=None,
              out_s=None, ld=4, err=None, stream=None)
FORK = dict(caches=P, stride=8 * 64, n=2, pages=8, page_bytes=64, page=16, table=P, max_pages=4, lens=2 * P, seqs=2,
            parents=3 * P, reserve=4 * P, rows=3, out=5 * P, lens_out=6 * P, ws=7 * P, ws_bytes=1 << 20, err=None,
            stream=None)
COMPACT = dict(caches=P, stride=8 * 64, n=2, pages=8, page_bytes=64, page=16, table=P, max_pages=4, lens=2 * P, seqs=2,
               out=5 * P, used=6 * P, ws=7 * P, ws_bytes=1 << 20, err=None, stream=None)


@pytest.mark.parametrize("change", [
    dict(B=-1), dict(nq=0), dict(nkv=0), dict(nq=5), dict(d=64), dict(page=32), dict(pages=0), dict(num_seqs=0),
    dict(rot=3), dict(rot=130), dict(rot=-2), dict(max_pages=0), dict(qkv=None), dict(f=None), dict(pos=None),
    dict(table=None), dict(q=None), dict(kc=None), dict(vc=None), dict(qkv=P + 8), dict(q=P + 2), dict(k_out=P + 4),
    dict(kc=P + 1), dict(vc=P + 8)])
def test_write_refusals(k, change):
    assert k.attn_kv4_rope_write_rows(*{**WRITE, **change}.values()) == INVALID


def test_nothing_to_do_is_ok(k):
    assert k.attn_kv4_rope_write_rows(*{**WRITE, "B": 0}.values()) == OK
    assert k.attn_kv4_read_rows(*{**READ, "B": 0}.values()) == OK
    assert k.attn_kv4_read_rows(*{**READ, "k": None, "v": None}.values()) == OK
    assert k.attn_kv4_decode_rows(*{**DECODE, "B": 0}.values()) == OK
    assert k.attn_prompt_packed(*{**PROMPT, "T": 0}.values()) == OK
    assert k.attn_prompt_packed(*{**PROMPT, "seqs": 0}.values()) == OK
    assert k.kv_pages_fork(*{**FORK, "rows": 0}.values()) == OK


@pytest.mark.parametrize("change", [
    dict(B=-1), dict(nkv=0), dict(d=64), dict(page=8), dict(pages=0), dict(num_seqs=0), dict(max_pages=0), dict(pos=None),
    dict(table=None), dict(kc=None), dict(vc=None), dict(kc=P + 8), dict(v=P + 8)])
def test_read_refusals(k, change):
    assert k.attn_kv4_read_rows(*{**READ, **change}.values()) == INVALID


@pytest.mark.parametrize("change,code", [
    (dict(B=-1), INVALID), (dict(nq=34), INVALID), (dict(nq=0), INVALID), (dict(nkv=3), INVALID), (dict(d=64), INVALID),
    (dict(page=32), INVALID), (dict(split=24), INVALID), (dict(split=0), INVALID), (dict(split=8208), INVALID),
    (dict(splits=0), INVALID), (dict(max_pages=0), INVALID), (dict(pages=0), INVALID), (dict(num_seqs=0), INVALID),
    (dict(q=None), INVALID), (dict(kc=None), INVALID), (dict(vc=None), INVALID), (dict(table=None), INVALID),
    (dict(lens=None), INVALID), (dict(ws=None), INVALID), (dict(out=None), INVALID), (dict(q=P + 2), INVALID),
    (dict(kc=P + 4), INVALID), (dict(ws=P + 4), INVALID), (dict(out_q=P), INVALID), (dict(out_q=P, out_s=P, ld=1), INVALID),
    (dict(ws_bytes=100), WORKSPACE), (dict(B=40000), UNSUPPORTED)])
def test_decode_refusals(k, change, code):
    assert k.attn_kv4_decode_rows(*{**DECODE, **change}.values()) == code


@pytest.mark.parametrize("split,splits,code", [
    (8192, 262143, UNSUPPORTED), (8192, 262144, UNSUPPORTED), (16, 1 << 27, UNSUPPORTED), (48, 0x7FFFFFFF // 48, UNSUPPORTED),
    (16, 0x7FFFFFFF, UNSUPPORTED), (8192, 262142, WORKSPACE), (16, (1 << 27) - 600, WORKSPACE)])
def test_decode_splits_of_more_tokens_than_32_bits_count(k, split, splits, code):
    """A split's first token and the end of a context are 32-bit numbers; what is refused for its workspace alone is not
    refused before."""
    assert k.attn_kv4_decode_rows(*{**DECODE, "split": split, "splits": splits}.values()) == code


@pytest.mark.parametrize("change,code", [
    (dict(T=-1), INVALID), (dict(seqs=-1), INVALID), (dict(nq=34), INVALID), (dict(nq=3), INVALID), (dict(nkv=0), INVALID),
    (dict(d=64), INVALID), (dict(qs=511), INVALID), (dict(qs=516), INVALID), (dict(ks=128), INVALID), (dict(vs=250), INVALID),
    (dict(vs=260), INVALID), (dict(q=None), INVALID), (dict(k=None), INVALID), (dict(v=None), INVALID),
    (dict(cu=None), INVALID), (dict(out=None), INVALID), (dict(q=P + 8), INVALID), (dict(v=P + 2), INVALID),
    (dict(out=P + 4), INVALID), (dict(out_q=P), INVALID), (dict(out_q=P, out_s=P, ld=3), INVALID),
    (dict(nq=65536, nkv=65536, qs=1 << 23, ks=1 << 23, vs=1 << 23), UNSUPPORTED)])
def test_prompt_refusals(k, change, code):
    assert k.attn_prompt_packed(*{**PROMPT, **change}.values()) == code


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 3e38])
def test_scales_that_are_not_finite(k, scale):
    """3e38 is a float whose product with log2(e) is not."""
    assert k.attn_prompt_packed(*{**PROMPT, "scale": scale}.values()) == INVALID
    assert k.attn_kv4_decode_rows(*{**DECODE, "scale": scale}.values()) == INVALID


def test_prompt_quantised_rows_32_byte_aligned(k):
    assert k.attn_prompt_packed(*{**PROMPT, "out_q": 32 * P + 16, "out_s": P}.values()) == INVALID


@pytest.mark.parametrize("change,code", [
    (dict(n=-1), INVALID), (dict(pages=0), INVALID), (dict(page=8), INVALID), (dict(max_pages=0), INVALID),
    (dict(seqs=0), INVALID), (dict(rows=-1), INVALID), (dict(caches=None), INVALID), (dict(caches=P + 8), INVALID),
    (dict(page_bytes=0), INVALID), (dict(page_bytes=40), INVALID), (dict(stride=8 * 64 - 16), INVALID),
    (dict(stride=8 * 64 + 8), INVALID), (dict(table=None), INVALID), (dict(lens=None), INVALID),
    (dict(parents=None), INVALID), (dict(out=None), INVALID), (dict(lens_out=None), INVALID), (dict(ws=None), INVALID),
    (dict(ws=7 * P + 4), INVALID), (dict(out=P), INVALID), (dict(out=P + 16), INVALID), (dict(lens_out=2 * P), INVALID),
    (dict(out=3 * P - 4), INVALID), (dict(ws_bytes=100), WORKSPACE), (dict(rows=1 << 26), UNSUPPORTED),
    (dict(max_pages=1 << 28), UNSUPPORTED), (dict(max_pages=1 << 20, rows=1 << 20), UNSUPPORTED)])
def test_fork_refusals(k, change, code):
    assert k.kv_pages_fork(*{**FORK, **change}.values()) == code


@pytest.mark.parametrize("change,code", [
    (dict(n=-1), INVALID), (dict(pages=0), INVALID), (dict(page=8), INVALID), (dict(seqs=0), INVALID),
    (dict(caches=None), INVALID), (dict(stride=64), INVALID), (dict(table=None), INVALID), (dict(lens=None), INVALID),
    (dict(out=None), INVALID), (dict(used=None), INVALID), (dict(ws=None), INVALID), (dict(out=P + 4), INVALID),
    (dict(out=2 * P), INVALID), (dict(ws_bytes=100), WORKSPACE)])
def test_compact_refusals(k, change, code):
    assert k.kv_pages_compact(*{**COMPACT, **change}.values()) == code


def test_python_checks_refuse_before_the_call():
    import torch
    c = torch.zeros(4, 1, 1152, dtype=torch.uint8)
    with pytest.raises(ValueError):
        KV.kv4_decode(torch.zeros(2, 4, 128, dtype=torch.bfloat16), c[..., :1000], c, torch.zeros(2, 4, dtype=torch.int32),
                      torch.ones(2, dtype=torch.int32), 0.1)
    with pytest.raises(ValueError):
        KV.kv4_decode(torch.zeros(2, 4, 128, dtype=torch.float16), c, c, torch.zeros(2, 4, dtype=torch.int32),
                      torch.ones(2, dtype=torch.int32), 0.1)
    with pytest.raises(ValueError):
        KV.fork_pages(c[None], torch.zeros(2, 4, dtype=torch.int64), torch.zeros(2, dtype=torch.int32),
                      torch.zeros(2, dtype=torch.int32))
    x = torch.zeros(4, 4, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        A.prompt_packed(x, x[:3], x[:3], torch.tensor([0, 4], dtype=torch.int32), 0.1)
    with pytest.raises(ValueError):
        A.prompt_packed(x, x.transpose(1, 2), x, torch.tensor([0, 4], dtype=torch.int32), 0.1)


@pytest.mark.parametrize("change", [
    dict(inv_freq="float64"), dict(inv_freq=31), dict(seq_lens_out=3), dict(positions="int64"), dict(error_word="int64")])
def test_python_write_checks(change):
    import torch
    i32 = lambda n: torch.zeros(n, dtype=torch.int32)
    c = torch.zeros(4, 1, 1152, dtype=torch.uint8)
    args = dict(inv_freq=torch.zeros(32), seq_lens_out=i32(2), positions=i32(2), error_word=i32(1))
    for name, to in change.items():
        args[name] = args[name].to(getattr(torch, to)) if isinstance(to, str) else torch.zeros(to, dtype=args[name].dtype)
    with pytest.raises(ValueError, match="inv_freq|one entry per row|int32"):
        KV.kv4_rope_write(torch.zeros(2, 6 * 128, dtype=torch.bfloat16), args["positions"], None, torch.zeros(2, 4, dtype=torch.int32),
                          c, c, 4, 64, args["inv_freq"], seq_lens_out=args["seq_lens_out"], error_word=args["error_word"])


@pytest.mark.parametrize("shape", [(8,), (2, 2, 2), ()])
@pytest.mark.parametrize("rows", [False, True])
def test_page_tables_have_two_dimensions(shape, rows):
    import torch
    i32 = lambda *n: torch.zeros(*n, dtype=torch.int32)
    c = torch.zeros(4, 1, 1152, dtype=torch.uint8)
    table, seq = torch.zeros(shape, dtype=torch.int32), i32(2) if rows else None
    with pytest.raises(ValueError, match="page table"):
        KV.kv4_rope_write(torch.zeros(2, 6 * 128, dtype=torch.bfloat16), i32(2), seq, table, c, c, 4, 64, torch.zeros(32))
    with pytest.raises(ValueError, match="page table"):
        KV.kv4_read_rows(c, c, i32(2), seq, table)
    with pytest.raises(ValueError, match="page table"):
        KV.kv4_decode(torch.zeros(2, 4, 128, dtype=torch.bfloat16), c, c, table, i32(2), 0.1, row_seq=seq)
    with pytest.raises(ValueError, match="page table|page-table"):
        KV.fork_pages(c[None], table, i32(2), i32(2))
    with pytest.raises(ValueError, match="page table|page-table"):
        KV.compact_pages(c[None], table, i32(2))


@pytest.mark.parametrize("shared", ["expanded", "strided"])
def test_workspaces_are_contiguous(shared):
    """A workspace of more elements than memory would be written past its end."""
    import torch
    i32 = lambda *n: torch.zeros(*n, dtype=torch.int32)
    ws = torch.zeros(1, dtype=torch.uint8).expand(1 << 20) if shared == "expanded" else torch.zeros(1 << 20, dtype=torch.uint8)[::2]
    c = torch.zeros(4, 1, 1152, dtype=torch.uint8)
    with pytest.raises(ValueError, match="workspace"):
        KV.kv4_decode(torch.zeros(2, 4, 128, dtype=torch.bfloat16), c, c, i32(2, 4), i32(2), 0.1, workspace=ws)
    with pytest.raises(ValueError, match="workspace"):
        KV.fork_pages(c[None], i32(2, 4), i32(2), i32(2), workspace=ws)
    with pytest.raises(ValueError, match="workspace"):
        KV.compact_pages(c[None], i32(2, 4), i32(2), workspace=ws)


# ---------------------------------------------------------------- the plain statements themselves

def test_quantiser_by_hand():
    x = np.zeros((1, 128), np.float32)
    x[0, 0], x[0, 1] = 7.5, -7.5           # scale 1: 7.5 is clipped to 7, -7.5 rounds to -8
    x[0, 32:64] = 0.0                      # an all-zero group
    x[0, 64] = np.inf
    x[0, 96] = 1.0                         # 1 / 7.5 = 0.1333, up to four bits: 0.140625
    codes, s = R.quantise(x)
    assert s[0, 0] == 1.0 and codes[0, 0] == 15 and codes[0, 1] == 0
    assert s[0, 1] == np.float32(2.0 ** -126) and (codes[0, 32:64] == 8).all()
    assert np.isnan(s[0, 2]) and (codes[0, 64:96] == 8).all()
    assert s[0, 3] == 0.140625 and codes[0, 96] == 15


def test_quantiser_error_bound():
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((2000, 128)) * np.exp(rng.standard_normal((2000, 1)) * 5)).astype(np.float32)
    x = (x.view(np.uint32) & 0xFFFF0000).view(np.float32)          # bf16 numbers
    codes, s = R.quantise(x)
    y = R.values(codes, s)
    assert (np.abs(y - x) <= np.repeat(s.astype(np.float64), 32, axis=1) / 2).all()
    # scales have four significant bits, values are bf16 numbers
    m, _ = np.frexp(s.astype(np.float64))
    assert (m * 16 == np.rint(m * 16)).all()
    assert (y.astype(np.float32).view(np.uint32) & 0xFFFF == 0).all() and (y == y.astype(np.float32)).all()


@pytest.mark.parametrize("which", ["k", "v"])
def test_layout_is_a_bijection(which):
    seen = set()
    for t in range(16):
        byte, shift = R.code_place(which, t)
        assert ((byte[0::2] == byte[1::2]) & (shift[0::2] == 0) & (shift[1::2] == 4)).all()
        seen |= set(zip(byte.tolist(), shift.tolist()))
    assert len(seen) == 2048 and max(b for b, _ in seen) == 1023
    rng = np.random.default_rng(1)
    tile = rng.integers(0, 256, 1152).astype(np.uint8)
    codes, s = R.quantise(rng.standard_normal((16, 128)).astype(np.float32))
    for t in (3, 0, 15, 7, 8, 1, 2, 4, 5, 6, 9, 14, 10, 13, 12, 11):
        R.store(tile, which, t, codes[t], s[t])
    for t in range(16):
        assert np.array_equal(R.load(tile, which, t), R.values(codes[t], s[t]))


def test_fork_by_hand():
    # two rows of 20 tokens share page 3 (full); pages 5 and 6 hold 4 tokens each; pool of 9
    caches = np.arange(9)[None, :, None].repeat(2, axis=0).copy()
    table = np.array([[3, 5, -1], [3, 6, -1]], np.int32)
    lens = np.array([20, 20], np.int32)
    out, n, c, short = R.fork(caches, table, lens, [0, 0, -1, 0], [1, 1, 0, 0])
    # row 0 keeps page 5, row 1 copies it to the lowest free page, row 3 only reads it; page 6 is free now
    assert out.tolist() == [[3, 5, -1], [3, 0, -1], [-1, -1, -1], [3, 5, -1]] and n.tolist() == [20, 20, 0, 20]
    assert c[0, 0, 0] == 5 and not short
    out, n, c, short = R.fork(caches, table, lens, [1], [13])
    assert out.tolist() == [[3, 6, 0]]


def test_compact_by_hand():
    caches = np.arange(6)[None, :, None].copy()
    table = np.array([[5, 1, 9], [4, -1, 2]], np.int32)
    out, U, c = R.compact(caches, table, np.array([32, 3], np.int32))
    assert U == 3 and out.tolist() == [[2, 1, -1], [0, -1, -1]] and c[0, :3, 0].tolist() == [4, 1, 5]
