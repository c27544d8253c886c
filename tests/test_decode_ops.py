"""Decoding operators (pero_ocr_amd/decode_ops.py): paged cache of keys and values in 8 bits, attention of drafted tokens over it, scores
of given tokens - against 64-bit restatements (oracle/decode_oracle.py), with tolerances that follow from the arithmetic."""
import ctypes as C
import math
import os
import subprocess

import numpy as np
import pytest
import torch

from oracle import decode_oracle as oracle
from pero_ocr_amd import _native, decode_ops as ops

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------------------------- CPU: refusals, masks, index arithmetic
def _fake_pages(**kw):
    d = dict(k=1 << 20, v=1 << 20, k_exp=1 << 20, v_exp=1 << 20, num_pages=4, kv_heads=2, page_size=16, head_dim=64, format=1)
    d.update(kw)
    return _native.KvPages(*(d[f] for f, _t in _native.KvPages._fields_))


def _err():
    return _native.load().pocr_last_error().decode()


@pytest.mark.parametrize("kw, word", [
    (dict(k=None), "NULL"), (dict(v=None), "NULL"), (dict(k_exp=None), "8-bit"), (dict(head_dim=48), "head_dim"), (dict(head_dim=0), "head_dim"),
    (dict(page_size=24), "page_size"), (dict(page_size=8), "page_size"), (dict(page_size=0), "page_size"), (dict(page_size=-16), "page_size"),
    (dict(num_pages=0), "num_pages"), (dict(kv_heads=0), "num_pages"), (dict(k=(1 << 20) + 8), "16 bytes"), (dict(format=2), "format")])
def test_c_entries_refuse_a_bad_cache(kw, word):
    lib, pages = _native.load(), _fake_pages(**kw)
    p = 1 << 20
    assert lib.pocr_kv_write(0, None, pages, _native.KvRows(p, p, p, 128, 64, 128, 64, 3, 0, 1)) == 1 and word in _err()
    assert lib.pocr_kv_read(0, None, pages, p, 1, 3, p, p, 0) == 1 and word in _err()
    args = _native.TreeAttentionArgs(q=p, out=p, page_table=p, lengths=p, q_start=p, tokens=1, seqs=1, heads=2, max_pages=1)
    assert lib.pocr_tree_attention(0, None, pages, args) == 1 and word in _err()
    assert lib.pocr_tree_attention_workspace(pages, args) <= 0


def test_c_entries_refuse_bad_arguments():
    lib, pages, p = _native.load(), _fake_pages(), 1 << 20
    for kw, word in ((dict(dtype=7), "dtype"), (dict(k=p + 1, dtype=1), "aligned"), (dict(slots=p + 4), "aligned"), (dict(slots=None), "NULL"), (dict(v=None), "NULL"),
                     (dict(tokens=-1), "tokens"), (dict(tokens=1 << 40), "2^31")):
        base = dict(k=p, v=p, slots=p, k_token_stride=128, k_head_stride=64, v_token_stride=128, v_head_stride=64, tokens=3, dtype=0, slots64=1)
        base.update(kw)
        assert lib.pocr_kv_write(0, None, pages, _native.KvRows(**base)) == 1 and word in _err(), kw
    assert lib.pocr_kv_write(0, None, pages, None) == 1 and "NULL" in _err()
    assert lib.pocr_kv_write(0, None, pages, _native.KvRows(tokens=0)) == 0                              # nothing to do
    assert lib.pocr_kv_read(0, None, pages, p, 1, 3, p + 4, p, 0) == 1 and "16 bytes" in _err()
    assert lib.pocr_kv_read(0, None, pages, p, 1, 3, p, p, 3) == 1 and "dtype" in _err()
    for kw, word in ((dict(q=None), "NULL"), (dict(lengths=None), "NULL"), (dict(page_table=None), "NULL"), (dict(heads=3), "heads"), (dict(heads=0), "heads"),
                     (dict(seqs=0), "sequence"), (dict(dtype=5), "dtype"), (dict(max_pages=-1), "max_pages"), (dict(out=p + 2), "aligned"),
                     (dict(mask=p, mask_words=0), "mask_words"), (dict(tokens=-2), "tokens"), (dict(tokens=1 << 40), "tokens")):
        base = dict(q=p, out=p, page_table=p, lengths=p, q_start=p, tokens=1, seqs=1, heads=2, max_pages=1)
        base.update(kw)
        assert lib.pocr_tree_attention(0, None, pages, _native.TreeAttentionArgs(**base)) == 1 and word in _err(), kw
    assert lib.pocr_tree_attention(0, None, pages, None) == 1 and "NULL" in _err()
    for kw, word in ((dict(logits=None), "NULL"), (dict(top=65), "top"), (dict(top=11), "top"), (dict(top=-1), "top"), (dict(classes=0), "classes"),
                     (dict(given=-1), "given"), (dict(dtype=9), "dtype"), (dict(entropy=None), "NULL"), (dict(tokens=p + 2), "aligned"), (dict(rows=-1), "rows")):
        base = dict(logits=p, tokens=p, logprob=p, entropy=p, top_logprob=p, top_index=p, row_stride=10, rows=2, classes=10, given=1, top=2)
        base.update(kw)
        assert lib.pocr_token_logprobs(0, None, _native.TokenLogprobsArgs(**base)) == 1 and word in _err(), kw
    assert lib.pocr_token_logprobs(0, None, None) == 1 and "NULL" in _err()
    # scratch memory that is needed and not given, too small or not aligned
    args = _native.TokenLogprobsArgs(logits=p, tokens=p, logprob=p, entropy=p, top_logprob=p, top_index=p, row_stride=1 << 19, rows=2, classes=1 << 19, given=1, top=2)
    need = lib.pocr_token_logprobs_workspace(args)
    assert need > 0
    for w, n in ((None, need), (p, need - 1), (p + 8, need)):
        args.workspace, args.workspace_bytes = w, n
        assert lib.pocr_token_logprobs(0, None, args) == 1 and "workspace" in _err()
    args = _native.TreeAttentionArgs(q=p, out=p, page_table=p, lengths=p, q_start=p, tokens=1, seqs=1, heads=2, max_pages=4096, q_head_stride=64, q_token_stride=128)
    need = lib.pocr_tree_attention_workspace(pages, args)
    assert need > 0
    for w, n in ((None, need), (p, need - 1), (p + 8, need)):
        args.workspace, args.workspace_bytes = w, n
        assert lib.pocr_tree_attention(0, None, pages, args) == 1 and "workspace" in _err()


def test_c_entries_refuse_more_work_than_a_launch_holds():
    """a grid has fewer than 2^32 threads: said before anything is enqueued"""
    lib, p = _native.load(), 1 << 20
    wide = _fake_pages(head_dim=256)
    for tokens, ok in ((1 << 24, True), ((1 << 24) + 1, False)):           # 2^26 rows of 32 threads
        rows = _native.KvRows(None, p, p, 512, 256, 512, 256, tokens, 1, 1)
        assert lib.pocr_kv_write(0, None, wide, rows) == 1 and ("NULL" if ok else "head_dim") in _err()
        assert lib.pocr_kv_read(0, None, wide, p, 1, tokens, None, p, 1) == 1 and ("NULL" if ok else "head_dim") in _err()
    args = _native.TreeAttentionArgs(q=None, out=p, page_table=p, lengths=p, q_start=p, tokens=1 << 26, seqs=4, heads=2, max_pages=1, q_head_stride=64, q_token_stride=128)
    assert lib.pocr_tree_attention(0, None, _fake_pages(), args) == 1 and "NULL" in _err()
    args.tokens += 1
    assert lib.pocr_tree_attention(0, None, _fake_pages(), args) == 1 and "2^27" in _err()
    for classes, rows in ((512, 1 << 28), (4096, 1 << 26), (32768, 1 << 24), (32769, 1 << 22)):
        args = _native.TokenLogprobsArgs(logits=None, tokens=p, logprob=p, entropy=p, top_logprob=p, top_index=p, row_stride=classes, rows=rows - 16, classes=classes, given=1)
        assert lib.pocr_token_logprobs(0, None, args) == 1 and "NULL" in _err()
        args.rows = rows
        assert lib.pocr_token_logprobs(0, None, args) == 1 and "rows" in _err()


def test_python_refusals_on_cpu_tensors():
    k = torch.zeros(2, 2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.KVPages(k, k.clone())
    with pytest.raises(TypeError):
        ops.KVPages(k.float(), k.float())
    with pytest.raises(TypeError):
        ops.KVPages([1], k)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(TypeError):
        ops.token_logprobs(torch.zeros(2, 5, dtype=torch.int32), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError):
        ops.token_logprobs(torch.zeros(5), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="dtype"):
        ops.kv_pages(2, 2, 16, 64, dtype="int3", device="cpu")


def test_tree_mask():
    with pytest.raises(ValueError):
        ops.tree_mask([0], device="cpu")
    with pytest.raises(ValueError):
        ops.tree_mask([-1, 2, 0], device="cpu")
    assert ops.tree_mask([], device="cpu").shape == (0, 0)
    rng = np.random.RandomState(3)
    for n in (1, 2, 63, 64, 65, 130):
        parents = [-1] + [int(rng.randint(-1, i)) for i in range(1, n)]
        mask = ops.tree_mask(parents, device="cpu")
        assert mask.shape == (n, -(-n // 64)) and mask.dtype == torch.int64
        for i in range(n):
            line, p = set(), i
            while p >= 0:
                line.add(p)
                p = parents[p]
            words = [int(w) & (1 << 64) - 1 for w in mask[i]]
            assert {j for j in range(64 * len(words)) if words[j // 64] >> (j % 64) & 1} == line


def test_bad_pages_are_never_followed(tmp_path):
    """The kernels' index arithmetic (csrc/kv_cache.hpp), compiled for the host: whatever a page table holds, a row is either -1 or inside the
    cache; rows agree with the layout, also where offsets pass 32 bits."""
    src = tmp_path / "rows.cpp"
    src.write_text(r'''
#include <cstdio>
#include <cstdlib>
#include "kv_cache.hpp"
using namespace pocr;
#define CHECK(c) do { if (!(c)) { std::printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)
int main() {
    const int32_t table[5] = {3, -1, 2147483647, 4, 0};
    for (int shift = 4; shift <= 8; ++shift)
        for (int heads = 1; heads <= 3; ++heads)
            for (int head = 0; head < heads; ++head)
                for (int pages = 1; pages <= 5; ++pages)
                    for (int64_t pos = -70; pos < (int64_t)6 << shift; ++pos) {
                        const int64_t r = kv_row_base(table, 5, pages, heads, head, shift, pos), e = pos >> shift;
                        const bool good = pos >= 0 && e < 5 && table[e] >= 0 && table[e] < pages;
                        CHECK(good == (r >= 0));
                        if (good) CHECK(r < ((int64_t)pages * heads << shift) && r == (((int64_t)table[e] * heads + head) << shift) + pos - (e << shift));
                        const int64_t s = kv_slot_row(pos, pages, heads, head, shift);
                        CHECK((pos >= 0 && pos < (int64_t)pages << shift) == (s >= 0));
                        if (s >= 0) CHECK(s < ((int64_t)pages * heads << shift));
                    }
    CHECK(kv_row_base(table, 0, 5, 1, 0, 4, 0) == -1);
    const int32_t far[1] = {2000000000};
    CHECK(kv_row_base(far, 1, 2147483647, 64, 63, 10, 1023) == ((2000000000LL * 64 + 63) << 10) + 1023);
    CHECK(kv_slot_row((int64_t)2000000000 << 10, 2147483647, 64, 63, 10) == (2000000000LL * 64 + 63) << 10);
    CHECK(kv_slot_row(INT64_MIN, 5, 1, 0, 4) == -1 && kv_slot_row(INT64_MAX, 5, 1, 0, 4) == -1);
    std::puts("ok");
}
''')
    exe = tmp_path / "rows"
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(REPO, "pero_ocr_amd", "csrc"), "-o", str(exe), str(src)], check=True)
    assert subprocess.run([str(exe)], capture_output=True, text=True).stdout == "ok\n"


def test_oracle_quantiser_on_known_rows():
    codes, exp = oracle.quantise_rows(np.array([[448.0, -1.0], [449.0, 0.0], [0.0, 0.0], [math.inf, 1.0], [2.0 ** -9, 2.0 ** -10 * 3]]))
    assert exp.tolist() == [127, 128, 27, 119, 110]
    assert codes[0].tolist() == [448.0, -1.0] and codes[1][0] == 224.0 and math.isnan(codes[3][0]) and codes[3][1] == 256.0


# ---------------------------------------------------------------------------------------------- GPU
def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _values(pages):
    """what a cache stands for, [pages][heads][rows][dim] in float64"""
    k, v = (t.float().cpu().double().numpy() for t in (pages.k, pages.v))
    if pages.k_exp is None:
        return k, v
    return oracle.cache_values(k, pages.k_exp.cpu().numpy()), oracle.cache_values(v, pages.v_exp.cpu().numpy())


def _same(got, want):
    """equal numbers, NaN in the same places"""
    return np.array_equal(np.asarray(got, np.float64), np.asarray(want, np.float64), equal_nan=True)


def _special_rows(rows, dim, kind, seed):
    """rows of ordinary numbers, rows at the borders of the quantiser, rows with numbers that are not finite"""
    g = _gen(seed)
    x = torch.randn(rows, dim, device="cuda", generator=g) * torch.exp2(torch.randint(-12, 12, (rows, 1), device="cuda", generator=g).float())
    top = 3e38 if kind != torch.float16 else 6e4
    specials = [0.0, 448.0, 448.0 * 2 ** -20, 449.0, 1.75, 1.7578125, 2.0 ** -24, 1e-38, 1e-45, top, -top, 3.0]
    for i, s in enumerate(specials):
        if i < rows:
            x[i] = torch.clamp(x[i], -1, 1) * abs(s)
            x[i, i % dim] = s
    if rows > 20:
        x[13, 3], x[14, 5], x[15, 0], x[16] = math.nan, math.inf, -math.inf, math.nan
        x[17] = -0.0
    return x.to(kind)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [32, 64, 128, 256])
@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
def test_gpu_cache_round_trip(kind, cache, dim):
    heads, page, num = 3, 16, 9
    tokens = 41
    pages = ops.kv_pages(num, heads, page, dim, dtype=cache)
    for t in (pages.k, pages.v):
        t.view(torch.uint8).random_(0, 127, generator=_gen(5))
    before = _values(pages)
    dt = TYPES[kind]
    k, v = (_special_rows(tokens * heads, dim, dt, s).view(tokens, heads, dim) for s in (1, 2))
    slots = torch.randperm(num * page, device="cuda", generator=_gen(3))[:tokens]
    slots[7], slots[20], slots[21], slots[33] = -1, num * page, 1 << 40, -(1 << 50)
    ops.kv_write(pages, k, v, slots)
    got = _values(pages)
    sl = slots.cpu().numpy()
    for name, x, was, now, codes, exps in (("k", k, before[0], got[0], pages.k, pages.k_exp), ("v", v, before[1], got[1], pages.v, pages.v_exp)):
        x64 = x.float().cpu().double().numpy()
        if cache == "fp8":
            want, e = oracle.quantise_rows(x64)
            value = oracle.cache_values(want, e)
        else:
            value = oracle.round_to(x64, 8, -126)
        flat_was, flat_now = (t.transpose(0, 2, 1, 3).reshape(-1, heads, dim) for t in (was, now))
        touched = np.zeros(num * page, bool)
        for t, s in enumerate(sl):
            if 0 <= s < num * page:
                touched[s] = True
                assert _same(flat_now[s], value[t]), (name, t)
                if cache == "fp8":
                    assert np.array_equal(exps.cpu().numpy().transpose(0, 2, 1).reshape(-1, heads)[s], e[t])
        assert _same(flat_now[~touched], flat_was[~touched])              # rows that no slot names are left as they were
    for out_kind in ("fp32", "bf16", "fp16"):
        rk, rv = ops.kv_read(pages, slots.clamp(-5, num * page + 5).to(torch.int32), dtype=TYPES[out_kind])
        for r, now in ((rk, got[0]), (rv, got[1])):
            flat = now.transpose(0, 2, 1, 3).reshape(-1, heads, dim)
            want = np.stack([flat[s] if 0 <= s < num * page else np.zeros((heads, dim)) for s in sl])
            if out_kind == "fp16":
                want = oracle.round_to(want, 11, -14)
                want = np.where(np.abs(want) > 65504, np.copysign(np.inf, want), want)
            elif out_kind == "bf16":
                want = oracle.round_to(want, 8, -126)
            assert _same(r.float().cpu().numpy(), want), out_kind


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [0, 1, 3])
@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_gpu_write_strided_inputs(kind, shift):
    """slices of a fused projection, at offsets that are and are not multiples of 16 bytes"""
    heads, dim, tokens = 2, 64, 19
    pages, whole = ops.kv_pages(4, heads, 16, dim), ops.kv_pages(4, heads, 16, dim)
    base = torch.randn(tokens, 5 * heads * dim + 8, device="cuda", generator=_gen(1)).to(TYPES[kind])
    k = base[:, shift:shift + heads * dim].unflatten(1, (heads, dim))
    v = base[:, 2 * heads * dim + shift:3 * heads * dim + shift].unflatten(1, (heads, dim))
    slots = torch.arange(40, 40 + tokens, device="cuda")
    ops.kv_write(pages, k, v, slots)
    ops.kv_write(whole, k.contiguous(), v.contiguous(), slots)
    for a, b in zip((pages.k, pages.v), (whole.k, whole.v)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert torch.equal(pages.k_exp, whole.k_exp) and torch.equal(pages.v_exp, whole.v_exp)
    # heads before tokens
    kt = k.transpose(0, 1).contiguous().transpose(0, 1)
    again = ops.kv_pages(4, heads, 16, dim)
    ops.kv_write(again, kt, v, slots)
    assert torch.equal(again.k.view(torch.uint8), whole.k.view(torch.uint8))


def _filled(num, heads, page, dim, cache, seed, spread=True):
    g = _gen(seed)
    pages = ops.kv_pages(num, heads, page, dim, dtype=cache)
    slots = torch.arange(num * page, device="cuda")
    k, v = (torch.randn(num * page, heads, dim, device="cuda", generator=g) for _ in range(2))
    if spread:
        k *= torch.exp2(torch.randint(-3, 2, (num * page, heads, 1), device="cuda", generator=g).float())
        v *= torch.exp2(torch.randint(-6, 6, (num * page, heads, 1), device="cuda", generator=g).float())
    ops.kv_write(pages, k, v, slots)
    return pages


def _problem(lengths, counts, heads, kv_heads, dim, page, kind, cache, seed, mask="chain", tail=0, extra_pages=2):
    need = [-(-n // page) for n in lengths]
    pages = _filled(sum(need) + extra_pages, kv_heads, page, dim, cache, seed)
    g = _gen(seed + 1)
    ids = torch.randperm(sum(need) + extra_pages, device="cuda", generator=g).to(torch.int32).cpu()
    table, at = torch.full((len(lengths), max(max(need), 1)), -1, dtype=torch.int32), 0
    for s, n in enumerate(need):
        table[s, :n] = ids[at:at + n]
        at += n
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    total = starts[-1] + tail
    q = torch.randn(total, heads, dim, device="cuda", generator=g).to(TYPES[kind])
    bits = None
    if mask != "chain":
        rows, rng = [], np.random.RandomState(seed)
        words = max(1, -(-max(counts + [1]) // 64))
        for n in counts:
            if mask == "tree":
                m = ops.tree_mask([-1] + [int(rng.randint(-1, i)) for i in range(1, n)] if n else [], device="cpu")
                m = torch.nn.functional.pad(m, (0, words - m.shape[1]))
            else:                                     # any bits at all, some rows empty
                m = torch.from_numpy(rng.randint(-2 ** 63, 2 ** 63 - 1, (n, words), dtype=np.int64))
                m[::3] = 0
            rows.append(m)
        bits = torch.cat(rows + [torch.full((tail, words), -1, dtype=torch.int64)]).cuda()
    return dict(q=q, pages=pages, page_table=table.cuda(), lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                q_start=torch.tensor(starts, dtype=torch.int32, device="cuda"), mask=bits)


def _planes(kind):
    """how the probabilities enter the second product: as two bfloat16 numbers (2^-17 of the value), three for float32 (2^-24)"""
    return 2.0 ** -24 if kind == "fp32" else 2.0 ** -16


def _check(p, kind, got, **kw):
    k, v = _values(p["pages"])
    out, lse, tol, lse_tol = oracle.attention(p["q"].double().cpu().numpy(), k, v, p["page_table"].cpu().numpy(), p["lengths"].cpu().numpy(),
                                              p["q_start"].cpu().numpy(), None if p["mask"] is None else p["mask"].cpu().numpy(), out_type=kind,
                                              planes=_planes(kind), **kw)
    o, l = got[0].double().cpu().numpy(), got[1].double().cpu().numpy()
    assert np.array_equal(np.isnan(o), np.isnan(out)) and np.array_equal(np.isnan(l), np.isnan(lse))
    fine = np.isfinite(out)
    worst = (np.abs(o - out)[fine] / np.maximum(tol[fine], 1e-30)).max(initial=0)
    assert worst <= 1, f"out: {worst} of what the arithmetic allows"
    assert np.array_equal(np.isneginf(l), np.isneginf(lse))
    fine = np.isfinite(lse)
    worst = (np.abs(l[fine] - lse[fine]) / np.maximum(lse_tol[fine], 1e-30)).max(initial=0)
    assert worst <= 1, f"lse: {worst} of what the arithmetic allows"


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("dim", [32, 64, 128, 256])
def test_gpu_attention_types_and_dims(dim, cache, kind):
    p = _problem([37, 1, 16, 33, 0, 70], [3, 1, 16, 0, 0, 17], 4, 2, dim, 16, kind, cache, 7, mask="tree")
    _check(p, kind, ops.tree_attention(**p, want_lse=True))


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 32, 64, 256])
@pytest.mark.parametrize("heads, kv_heads", [(1, 1), (5, 1), (6, 3), (16, 2), (40, 2)])
def test_gpu_attention_heads_and_pages(heads, kv_heads, page):
    p = _problem([1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129], [1, 2, 1, 3, 1, 2, 1, 1, 7, 1, 1, 2], heads, kv_heads, 64, page, "bf16", "fp8", 11, mask="tree")
    for hint in (0, 1, 7, 1000):
        _check(p, "bf16", ops.tree_attention(**p, max_queries=hint, want_lse=True))


@pytest.mark.gpu
@pytest.mark.parametrize("mask", ["chain", "tree", "any"])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 63, 64, 65, 100])
def test_gpu_attention_masks(n, mask):
    """trees of every size against the tiles' borders; masks of any bits, rows of which see nothing but the context, or nothing at all"""
    p = _problem([n, n + 1, n + 40], [n, n, n], 2, 1, 32, 16, "fp32", "fp8", 13 + n, mask=mask)
    _check(p, "fp32", ops.tree_attention(**p, want_lse=True))


@pytest.mark.gpu
@pytest.mark.parametrize("length", [1000, 2047, 4100])
@pytest.mark.parametrize("cache", ["fp8", "bf16"])
def test_gpu_attention_long(cache, length):
    """a cache much longer than a tile, few rows: the work is split over the positions"""
    p = _problem([length, 5], [2, 1], 2, 1, 64, 64, "fp32", cache, 17, mask="chain")
    _check(p, "fp32", ops.tree_attention(**p, want_lse=True))


@pytest.mark.gpu
def test_gpu_attention_short_mask_words():
    """drafted tokens beyond the mask's words are seen by nobody; a mask without words is refused"""
    p = _problem([80, 90], [70, 66], 2, 2, 32, 16, "fp32", "bf16", 23, mask="tree")
    p["mask"] = p["mask"][:, :1]
    _check(p, "fp32", ops.tree_attention(**p, want_lse=True))
    with pytest.raises(ValueError):
        ops.tree_attention(**dict(p, mask=p["mask"][:, :0]))


@pytest.mark.gpu
def test_gpu_attention_bad_pages_and_lengths():
    """page ids outside the cache are absent, lengths beyond the table are cut to it, negative ones are zero"""
    p = _problem([64, 64, 64, 64], [2, 3, 1, 2], 4, 2, 64, 16, "fp32", "fp8", 29)
    t = p["page_table"]
    t[0, 1], t[0, 3], t[1, :], t[2, 0] = -1, 2 ** 31 - 1, -7, p["pages"].k.shape[0]
    p["lengths"] = torch.tensor([64, 64, 70000, -5], dtype=torch.int32, device="cuda")
    got = ops.tree_attention(**p, want_lse=True)
    assert (got[0][2:5] == 0).all() and torch.isneginf(got[1][2:5]).all() and (got[0][6:] == 0).all()
    q = dict(p, lengths=torch.tensor([64, 64, 64, 0], dtype=torch.int32, device="cuda"))
    # sequence 2: cut to the table's 64 positions (sequence 3: nothing is cached)
    _check(q, "fp32", got)


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["fp8", "bf16"])
def test_gpu_attention_not_a_number_stays_where_it_is_seen(cache):
    """NaN keys / values in drafted tokens, behind the last position and in absent pages reach only the rows that see them"""
    p = _problem([40, 21], [6, 5], 2, 1, 64, 16, "fp32", cache, 31, mask="tree")
    p["mask"] = torch.cat([ops.tree_mask([-1, 0, 0, 1, 2, -1]), ops.tree_mask([-1, 0, 1, 2, 3])])
    pages, table = p["pages"], p["page_table"].cpu()
    bad = torch.full((1, 1, 64), math.nan, device="cuda")
    one = torch.ones((1, 1, 64), device="cuda")

    def slot(s, j):
        return torch.tensor([int(table[s, j // 16]) * 16 + j % 16], device="cuda")
    ops.kv_write(pages, one, bad, slot(0, 34 + 1))                      # drafted token 1 of sequence 0: seen by 1 and 3
    ops.kv_write(pages, bad, one, slot(0, 34 + 5))                      # token 5: seen by itself
    for j in range(40, 48):
        ops.kv_write(pages, bad, bad, slot(0, j))                       # behind the last position, same page
    for j in range(21, 32):
        ops.kv_write(pages, bad, bad, slot(1, j))
    out, lse = ops.tree_attention(**p, want_lse=True)
    nan_rows = torch.isnan(out).any(-1).any(-1).tolist()
    assert nan_rows == [False, True, False, True, False, True] + [False] * 5
    _check(p, "fp32", (out, lse))


@pytest.mark.gpu
def test_gpu_attention_infinite_values_and_scores():
    """an infinite value in a bfloat16 cache reaches the rows that see it, and no others; an infinite query makes its own row NaN"""
    p = _problem([20], [4], 1, 1, 32, 16, "fp32", "bf16", 37, mask="tree")
    p["mask"] = ops.tree_mask([-1, 0, -1, 2])
    table = p["page_table"].cpu()
    x = torch.ones((1, 1, 32), device="cuda")
    y = x.clone()
    y[0, 0, 5] = math.inf
    ops.kv_write(p["pages"], x, y, torch.tensor([int(table[0, 1]) * 16 + 1], device="cuda"))      # drafted token 1
    out = ops.tree_attention(**p)
    assert torch.isinf(out[1, 0, 5]) and torch.isfinite(out[[0, 2, 3]]).all() and torch.isfinite(out[1, 0, :5]).all()
    p["q"][2, 0, 0] = math.inf
    out = ops.tree_attention(**p)
    assert torch.isnan(out[2]).all() and torch.isfinite(out[[0, 3]]).all()


@pytest.mark.gpu
def test_gpu_attention_padded_batch():
    """rows behind the last sequence: zeros in a fresh tensor, left alone in a given one"""
    p = _problem([20, 50], [2, 3], 4, 2, 64, 32, "bf16", "fp8", 41, mask="tree", tail=4)
    out, lse = ops.tree_attention(**p, want_lse=True)
    assert (out[5:] == 0).all() and torch.isneginf(lse[5:]).all()
    given = torch.full_like(out, 7.0)
    same = ops.tree_attention(**p, out=given)
    assert same is given and (given[5:] == 7).all() and torch.equal(given[:5], out[:5])
    _check(p, "bf16", (out, lse))


@pytest.mark.gpu
@pytest.mark.parametrize("kv_heads", [1, 3, 8])
@pytest.mark.parametrize("seqs", [1, 2, 63, 65, 300])
def test_gpu_attention_ragged_batches(seqs, kv_heads):
    """every row of a ragged batch is somebody's, whatever the caller says of the longest sequence, and the rows behind the last one are zeros"""
    rng = np.random.RandomState(seqs)
    counts = [int(rng.choice([0, 0, 1, 1, 2, 3, 9])) for _ in range(seqs)]
    counts[seqs // 2] = 41
    lengths = [n + int(rng.randint(0, 60)) for n in counts]
    p = _problem(lengths, counts, 4 * kv_heads, kv_heads, 32, 16, "fp32", "bf16", seqs + kv_heads, mask="tree", tail=70)
    for most in (0, 1, 41, 10 ** 6):
        _check_dense(p, ops.tree_attention(**p, max_queries=most, want_lse=True))


@pytest.mark.gpu
def test_gpu_attention_thousands_of_sequences():
    """more sequences than one step of the search tells apart twice over, of lengths that nobody names; most of them are empty"""
    seqs, rng = 5000, np.random.RandomState(7)
    counts = [0] * seqs
    for s in rng.choice(seqs, 90, replace=False):
        counts[s] = int(rng.randint(1, 12))
    counts[0] = counts[-1] = 3
    lengths = [n + (int(rng.randint(0, 20)) if n else 0) for n in counts]
    p = _problem(lengths, counts, 16, 8, 32, 16, "fp32", "fp8", 71, mask="tree", tail=3)
    for most in (0, 1, 11):
        _check_dense(p, ops.tree_attention(**p, max_queries=most, want_lse=True))


@pytest.mark.gpu
def test_gpu_attention_many_tokens_without_a_hint():
    """2100 sequences of 8 tokens: rows and workgroups by the rows that there are (every sequence has room for all tokens: a launch that HIP refuses)"""
    seqs = 2100
    p = _problem([16] * seqs, [8] * seqs, 64, 8, 32, 16, "bf16", "fp8", 72)
    out = ops.tree_attention(**p)
    assert torch.equal(out, ops.tree_attention(**p, max_queries=8))
    few = dict(p, q=p["q"][:24].clone(), page_table=p["page_table"][:3], lengths=p["lengths"][:3], q_start=p["q_start"][:4])
    got = ops.tree_attention(**few, want_lse=True)
    _check(few, "bf16", got)
    assert torch.equal(got[0], out[:24])


@pytest.mark.gpu
def test_gpu_attention_in_place_and_without_pages():
    """the outputs may take the queries' place, split or not; sequences without any page see nothing"""
    for lengths, counts in (([40, 70], [3, 2]), ([3000, 2100], [3, 2])):
        p = _problem(lengths, counts, 4, 2, 64, 16, "bf16", "fp8", 45, mask="tree")
        want = ops.tree_attention(**p)
        q = p["q"].clone()
        assert ops.tree_attention(**dict(p, q=q, out=q)) is q and torch.equal(q, want)
    out, lse = ops.tree_attention(**dict(p, page_table=p["page_table"][:, :0]), want_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    empty = ops.tree_attention(p["q"][:0], p["pages"], p["page_table"][:0], none, torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert empty.shape == (0, 4, 64)
    with pytest.raises(RuntimeError, match="without a sequence"):
        ops.tree_attention(p["q"], p["pages"], p["page_table"][:0], none, torch.zeros(1, dtype=torch.int32, device="cuda"))


@pytest.mark.gpu
def test_gpu_attention_split_extremes():
    """sequences of very different lengths that share one cut into splits: empty splits, splits that see nothing, one long sequence"""
    p = _problem([9000, 1, 33, 2000, 0], [1, 1, 2, 3, 0], 2, 1, 64, 64, "fp32", "fp8", 49, mask="tree", tail=2)
    p["page_table"][3, 5:20] = -1                                    # 960 positions that are absent
    _check_dense(p, ops.tree_attention(**p, want_lse=True))
    p["page_table"][0, :-2] = -1
    _check_dense(p, ops.tree_attention(**p, want_lse=True))


def _check_dense(p, got):
    """against the oracle on the rows of the sequences; the rows behind them are zeros"""
    n = int(p["q_start"][-1])
    _check(dict(p, q=p["q"][:n], mask=p["mask"][:n]), "fp32", [t[:n] for t in got])
    assert (got[0][n:] == 0).all() and torch.isneginf(got[1][n:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [0, 1])
def test_gpu_attention_strided_queries(shift):
    p = _problem([20, 50], [2, 3], 4, 2, 64, 16, "bf16", "fp8", 43)
    base = torch.randn(5, 3 * 4 * 64 + 8, device="cuda", generator=_gen(2)).to(torch.bfloat16)
    p["q"] = base[:, 4 * 64 + shift:2 * 4 * 64 + shift].unflatten(1, (4, 64))
    got = ops.tree_attention(**p, want_lse=True)
    want = ops.tree_attention(**dict(p, q=p["q"].contiguous()), want_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    p["q"] = p["q"].transpose(0, 1).contiguous().transpose(0, 1)         # heads before tokens
    assert torch.equal(ops.tree_attention(**p), want[0])
    wide = torch.full((2, p["page_table"].shape[1] + 3), -1, dtype=torch.int32, device="cuda")
    wide[:, :-3] = p["page_table"]
    assert torch.equal(ops.tree_attention(**dict(p, page_table=wide[:, :-3])), want[0])
    _check(p, "bf16", want)


@pytest.mark.gpu
def test_gpu_attention_scale():
    p = _problem([30], [3], 2, 1, 64, 16, "fp32", "fp8", 47)
    _check(p, "fp32", ops.tree_attention(**p, scale=0.5, want_lse=True), scale=0.5)
    _check(p, "fp32", ops.tree_attention(**p, scale=-0.25, want_lse=True), scale=-0.25)
    _check(p, "fp32", ops.tree_attention(**p, scale=0.0, want_lse=True), scale=0.0)


@pytest.mark.gpu
def test_gpu_far_slots():
    """rows whose offset passes 32 bits: writing, reading and attending at the end of a cache of 5 GB"""
    num, heads, page, dim = 20000, 8, 128, 256
    k, v = (torch.empty((num, heads, page, dim), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
    ke, ve = (torch.full((num, heads, page), 127, dtype=torch.uint8, device="cuda") for _ in range(2))
    pages = ops.KVPages(k, v, ke, ve)
    rows = 40
    slots = num * page - rows + torch.arange(rows, device="cuda")
    x, y = (torch.randn(rows, heads, dim, device="cuda", generator=_gen(s)) for s in (1, 2))
    small = ops.kv_pages(2, heads, page, dim)
    ops.kv_write(pages, x, y, slots)
    ops.kv_write(small, x, y, torch.arange(page - rows, page, device="cuda"))
    assert torch.equal(k[-1, :, page - rows:].view(torch.uint8), small.k[0, :, page - rows:].view(torch.uint8))
    for a, b in zip(ops.kv_read(pages, slots), ops.kv_read(small, torch.arange(page - rows, page, device="cuda"))):
        assert torch.equal(a, b)
    ops.kv_write(small, x, y, torch.arange(rows, device="cuda"))
    q = torch.randn(3, heads, dim, device="cuda", generator=_gen(3))
    t = dict(lengths=torch.tensor([page], dtype=torch.int32, device="cuda"), q_start=torch.tensor([0, 3], dtype=torch.int32, device="cuda"))
    k[-1].view(torch.uint8).zero_()
    v[-1].view(torch.uint8).zero_()
    small.k[0].view(torch.uint8).zero_()
    small.v[0].view(torch.uint8).zero_()
    ops.kv_write(pages, x, y, slots)
    ops.kv_write(small, x, y, torch.arange(page - rows, page, device="cuda"))
    small.k_exp[0], small.v_exp[0] = ke[-1], ve[-1]
    a = ops.tree_attention(q, pages, torch.tensor([[num - 1]], dtype=torch.int32, device="cuda"), **t)
    b = ops.tree_attention(q, small, torch.tensor([[0]], dtype=torch.int32, device="cuda"), **t)
    assert torch.equal(a, b)


def _check_scores(x, tokens, top, got):
    t2 = tokens if tokens.dim() == 2 else tokens[:, None]
    lp, ent, tlp, tid, lp_tol, ent_tol = oracle.logprobs(x.double().cpu().numpy(), t2.cpu().numpy(), top)
    g = [t.double().cpu().numpy() for t in got]
    assert got[0].shape == tokens.shape and got[3].dtype == torch.int32
    assert np.array_equal(g[3], tid), "alternatives"
    for name, a, b, tol in (("logprob", g[0].reshape(lp.shape), lp, lp_tol[:, None]), ("entropy", g[1], ent, ent_tol), ("top", g[2], tlp, lp_tol[:, None])):
        assert np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(np.isinf(a), np.isinf(b)), name
        fine = np.isfinite(b)
        with np.errstate(invalid="ignore"):
            worst = (np.abs(a - b) / (tol + 4 * oracle.U32 * np.abs(b) + 1e-30))[fine].max(initial=0)
        assert worst <= 1, f"{name}: {worst} of what the arithmetic allows"


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("classes", [1, 2, 3, 63, 64, 65, 232, 256, 257, 511, 513, 1000, 1025, 4096, 4099, 33001, 70007])
def test_gpu_logprobs_sizes(classes, kind):
    rows = 5 if classes > 2000 else 13
    g = _gen(classes)
    x = (torch.randn(rows, classes, device="cuda", generator=g) * 3).to(TYPES[kind])
    tokens = torch.randint(0, classes, (rows, 3), device="cuda", generator=g)
    tokens[0, 0], tokens[1, 1], tokens[2, 2] = -1, -100, classes
    for top in sorted({0, 1, min(5, classes), min(64, classes)}):
        _check_scores(x, tokens, top, ops.token_logprobs(x, tokens, top=top))
    _check_scores(x, tokens[:, 0].contiguous(), 1, ops.token_logprobs(x, tokens[:, 0].int().contiguous(), top=1))


@pytest.mark.gpu
@pytest.mark.parametrize("classes", [40, 300, 700, 9000, 40000])
def test_gpu_logprobs_special_rows(classes):
    """ties, masks of -inf and of the lowest number, rows without anything, NaN and infinities, numbers at the ends of the range"""
    low = torch.finfo(torch.float32).min
    x = torch.zeros(16, classes, device="cuda")
    g = _gen(3)
    x[1] = -math.inf
    x[2, 1:] = -math.inf
    x[3] = low
    x[4, ::2] = low
    x[5, 7] = math.nan
    x[6, 3] = math.inf
    x[7] = torch.arange(classes, device="cuda") % 5
    x[8] = torch.randn(classes, device="cuda", generator=g) * 30
    x[8, ::3] = -math.inf
    x[9, 5], x[9, 6] = 3e38, low
    x[10] = -0.0
    x[10, 4::7] = 0.0
    x[11] = torch.arange(classes, device="cuda").float()
    x[12] = -torch.arange(classes, device="cuda").float()
    x[13, 30], x[13, 20], x[13, 8] = math.nan, math.nan, math.inf
    x[14] = 1e-40
    x[15, classes - 1] = 88.0
    tokens = torch.stack([torch.arange(16, device="cuda"), torch.full((16,), classes - 1, device="cuda"), torch.zeros(16, dtype=torch.int64, device="cuda")], 1)
    for top in (0, 1, 3, 33):
        _check_scores(x, tokens, top, ops.token_logprobs(x, tokens, top=top))
    for shift in (1, 2, 3):                                          # rows at addresses that are not multiples of 16 bytes
        wide = torch.full((16, classes + 8), 50.0, device="cuda")
        wide[:, shift:shift + classes] = x
        _check_scores(x, tokens, 3, ops.token_logprobs(wide[:, shift:shift + classes], tokens, top=3))


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["rising", "falling", "equal", "blocks", "few"])
@pytest.mark.parametrize("rows", [1, 300])
def test_gpu_logprobs_hard_orders(rows, order):
    """orders that make a running list of the best ones change all the time"""
    classes = 20011
    c = torch.arange(classes, device="cuda").float()
    row = {"rising": c / 1000, "falling": -c / 1000, "equal": torch.full_like(c, 2.5), "blocks": torch.floor(c / 256) % 7, "few": (c % 4001 == 17).float()}[order]
    x = (row[None] + torch.zeros(rows, 1, device="cuda")).contiguous()
    tokens = torch.arange(rows, device="cuda")
    got = ops.token_logprobs(x, tokens, top=50)
    assert all((t == t[:1]).all() for t in got[1:])
    _check_scores(x[:1], tokens[:1], 50, [t[:1] for t in got])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("rows, classes, top", [(1, 32769, 64), (1, 600000, 3), (2, 140003, 16), (9, 400009, 64), (127, 200001, 7), (128, 200001, 7), (9, 500001, 0)])
def test_gpu_logprobs_few_long_rows(rows, classes, top, kind):
    """rows that are cut into slices: special rows among ordinary ones, the alternatives in one slice or in several, given tokens in any"""
    g = _gen(rows)
    x = (torch.randn(rows, classes, device="cuda", generator=g) * 2).to(TYPES[kind])
    for r in range(min(rows, 9)):
        if r == 1:
            x[r, 50:] = -math.inf
        elif r == 2:
            x[r] = -math.inf
        elif r == 3:
            x[r, classes - 3] = math.nan
        elif r == 4:
            x[r, 20000:20100] = 11.0
        elif r == 5:
            x[r] = 1.5
        elif r == 6:
            x[r, 8] = math.inf
        elif r == 7:
            x[r, :30000] = math.nan
    tokens = torch.randint(0, classes, (rows, 2), device="cuda", generator=g)
    tokens[0, 1] = classes - 1
    at = list(range(min(rows, 9)))
    got = ops.token_logprobs(x, tokens, top=top)
    _check_scores(x[at], tokens[at], top, [t[at] for t in got])


@pytest.mark.gpu
def test_gpu_logprobs_many_rows():
    x = torch.randn(70000, 40, device="cuda", generator=_gen(9))
    tokens = torch.randint(0, 40, (70000,), device="cuda", generator=_gen(10))
    got = ops.token_logprobs(x, tokens, top=2)
    at = torch.randperm(70000, device="cuda", generator=_gen(11))[:200]
    _check_scores(x[at], tokens[at], 2, [t[at] for t in got])
    assert ops.token_logprobs(x[:0], tokens[:0], top=2)[2].shape == (0, 2)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("classes", [5, 63, 256, 257, 300, 512, 1500, 2047])
def test_gpu_logprobs_special_rows_among_many(classes, kind):
    """the same special rows where rows are many (other kernels than for few): each block of 16 answers as the first"""
    low, g = torch.finfo(TYPES[kind]).min, _gen(classes)
    x = torch.randn(16, classes, device="cuda", generator=g) * 4
    x[1] = -math.inf
    x[2, 1:] = -math.inf
    x[3] = low
    x[4, ::2] = low
    x[5, 2] = math.nan
    x[6, 3] = math.inf
    x[7] = torch.arange(classes, device="cuda") % 5
    x[8, ::3] = -math.inf
    x[9] = torch.arange(classes, device="cuda").float() / 50          # (in bfloat16: many equal ones)
    x[10] = -x[9]
    x[11] = 2.5
    x[12, :: max(classes // 9, 1)] = 9.0
    x[13, 1], x[13, 4] = math.nan, math.nan
    x[14, ::64] = torch.arange(-(-classes // 64), device="cuda") + 20.0   # all of the best in one lane's share
    x = x.to(TYPES[kind])
    tokens = torch.stack([torch.arange(16, device="cuda") % classes, torch.full((16,), classes - 1, device="cuda")], 1)
    for top in sorted({0, 1, 3, min(9, classes), min(64, classes)} & set(range(classes + 1))):
        got = ops.token_logprobs(x.repeat(260, 1), tokens.repeat(260, 1), top=top)
        _check_scores(x, tokens, top, [t[:16] for t in got])
        for t in got:
            block = t.view(260, 16, -1)
            assert torch.equal(block.view(torch.int32), block[:1].expand_as(block).contiguous().view(torch.int32))


@pytest.mark.gpu
def test_gpu_logprobs_millions_of_rows():
    """more rows than the first axis of a grid holds: the last ones answer as they do alone"""
    rows, classes = (1 << 21) + 3000, 270
    x = torch.randn(3000, classes, device="cuda", generator=_gen(21)).bfloat16()
    many = torch.zeros(rows, classes, device="cuda", dtype=torch.bfloat16)
    many[-3000:] = x
    tokens = torch.randint(0, classes, (3000,), device="cuda", generator=_gen(22))
    all_tokens = torch.zeros(rows, dtype=torch.int64, device="cuda")
    all_tokens[-3000:] = tokens
    for a, b in zip(ops.token_logprobs(many, all_tokens, top=9), ops.token_logprobs(x, tokens, top=9)):
        assert torch.equal(a[-3000:], b)


@pytest.mark.gpu
def test_gpu_python_refusals():
    pages = ops.kv_pages(4, 2, 16, 64)
    k, v, slots = torch.zeros(3, 2, 64, device="cuda"), torch.zeros(3, 2, 64, device="cuda"), torch.arange(3, device="cuda")
    for bad in (lambda: ops.kv_write(pages, k[:2], v, slots), lambda: ops.kv_write(pages, k[:, :1], v[:, :1], slots), lambda: ops.kv_write(pages, k, v, slots[None]),
                lambda: ops.kv_write(pages, k.transpose(1, 2), v.transpose(1, 2), slots), lambda: ops.kv_write(pages, k, v, torch.arange(6, device="cuda")[::2]),
                lambda: ops.kv_pages(4, 2, 24, 64), lambda: ops.kv_pages(4, 2, 16, 80), lambda: ops.kv_pages(0, 2, 16, 64),
                lambda: ops.KVPages(pages.k, pages.v[:2], pages.k_exp, pages.v_exp), lambda: ops.KVPages(pages.k, pages.v, pages.k_exp[:2], pages.v_exp),
                lambda: ops.kv_write(pages, k, v, slots.cpu())):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ops.kv_write(pages, k.double(), v.double(), slots), lambda: ops.kv_write(pages, k, v.bfloat16(), slots),
                lambda: ops.kv_write(pages, k, v, slots.float()), lambda: ops.kv_read(pages, slots, dtype=torch.float64),
                lambda: ops.KVPages(pages.k, pages.v, None, None), lambda: ops.KVPages(pages.k.float(), pages.v.float())):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(RuntimeError, match="gradient"):
        ops.kv_write(pages, k.clone().requires_grad_(), v, slots)
    with torch.no_grad():
        ops.kv_write(pages, k.clone().requires_grad_(), v, slots)
    p = _problem([20], [2], 4, 2, 64, 16, "fp32", "fp8", 1)
    for kw in (dict(q=p["q"][:, :3]), dict(q=p["q"][..., :32]), dict(lengths=p["lengths"][:0]), dict(q_start=p["q_start"][:1]), dict(mask=torch.zeros(3, 1, dtype=torch.int64, device="cuda")),
               dict(out=torch.zeros(1, 4, 64, device="cuda")), dict(page_table=torch.zeros(2, 2, dtype=torch.int32, device="cuda"))):
        with pytest.raises(ValueError):
            ops.tree_attention(**dict(p, **kw))
    for kw in (dict(lengths=p["lengths"].long()), dict(page_table=p["page_table"].long()), dict(out=torch.zeros(2, 4, 64, device="cuda", dtype=torch.bfloat16))):
        with pytest.raises(TypeError):
            ops.tree_attention(**dict(p, **kw))
    x = torch.zeros(2, 5, device="cuda")
    for bad in (lambda: ops.token_logprobs(x, torch.zeros(3, dtype=torch.int64, device="cuda")), lambda: ops.token_logprobs(x, torch.zeros(2, dtype=torch.int64, device="cuda"), top=6),
                lambda: ops.token_logprobs(x.t(), torch.zeros(5, dtype=torch.int64, device="cuda")), lambda: ops.token_logprobs(x, torch.zeros(2, dtype=torch.int64, device="cuda"), top=-1)):
        with pytest.raises(ValueError):
            bad()


def _step(pages, k, v, slots, q, table, lengths, starts, mask, head, drafted):
    """one verification step: the drafted tokens' keys and values, their attention, a projection to the vocabulary, their scores"""
    ops.kv_write(pages, k, v, slots)
    x, lse = ops.tree_attention(q, pages, table, lengths, starts, mask=mask, want_lse=True)
    logits = (x.flatten(1).float() @ head).to(torch.bfloat16)
    return (x, lse) + ops.token_logprobs(logits, drafted, top=5)


def _step_inputs(seed):
    g = _gen(seed)
    heads, kv_heads, dim, page = 8, 2, 64, 16
    lengths, counts = [90, 33, 260], [12, 1, 30]
    need = [-(-n // page) for n in lengths]
    pages = _filled(sum(need), kv_heads, page, dim, "fp8", seed, spread=False)
    table = torch.full((3, max(need)), -1, dtype=torch.int32)
    at, slots = 0, []
    for s, n in enumerate(need):
        table[s, :n] = torch.arange(at, at + n)
        slots += [int(table[s, j // page]) * page + j % page for j in range(lengths[s] - counts[s], lengths[s])]
        at += n
    total = sum(counts)
    k, v = (torch.randn(total, kv_heads, dim, device="cuda", generator=g) for _ in range(2))
    rng = np.random.RandomState(seed)
    mask = torch.cat([ops.tree_mask([-1] + [int(rng.randint(-1, i)) for i in range(1, n)]) for n in counts])
    starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    return dict(pages=pages, k=k, v=v, slots=torch.tensor(slots, device="cuda"), q=torch.randn(total, heads, dim, device="cuda", generator=g).to(torch.bfloat16),
                table=table.cuda(), lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"), starts=torch.from_numpy(starts).cuda(), mask=mask,
                head=torch.randn(heads * dim, 777, device="cuda", generator=g) * 0.1, drafted=torch.randint(0, 777, (total,), device="cuda", generator=g))


@pytest.mark.gpu
def test_gpu_one_verification_step():
    """the operators together, as a decoding loop uses them, then the accepted path moved together in the cache"""
    s = _step_inputs(51)
    x, lse, lp, ent, tlp, tid = _step(**s)
    p = dict(q=s["q"], pages=s["pages"], page_table=s["table"], lengths=s["lengths"], q_start=s["starts"], mask=s["mask"])
    _check(p, "bf16", (x, lse))
    logits = (x.flatten(1).float() @ s["head"]).to(torch.bfloat16)
    _check_scores(logits, s["drafted"], 5, (lp, ent, tlp, tid))
    # sequence 0 accepts tokens 0 -> j (a child of 0): written again behind the context, they read as a chain
    path = [0, next(i for i in range(1, 12) if int(s["mask"][i, 0]) == (1 | 1 << i))] if any(int(s["mask"][i, 0]) == (1 | 1 << i) for i in range(1, 12)) else [0]
    ids = torch.tensor(path, device="cuda")
    ops.kv_write(s["pages"], s["k"][ids], s["v"][ids], s["slots"][:len(path)].clone())
    q = s["q"][ids].contiguous()
    chain = ops.tree_attention(q, s["pages"], s["table"][:1], torch.tensor([78 + len(path)], dtype=torch.int32, device="cuda"),
                               torch.tensor([0, len(path)], dtype=torch.int32, device="cuda"))
    assert torch.allclose(chain.float(), x[ids].float(), rtol=2.0 ** -7, atol=2.0 ** -7)     # the same sums in another order, rounded to bfloat16


@pytest.mark.gpu
def test_gpu_streams_and_graphs():
    """two calls at once on two streams; two captured graphs replayed with other inputs between eager work, each replay checked"""
    a, b = _step_inputs(61), _step_inputs(62)
    want_a, want_b = [t.clone() for t in _step(**a)], [t.clone() for t in _step(**b)]
    torch.cuda.synchronize()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(sa):
            got_a = _step(**a)
        with torch.cuda.stream(sb):
            got_b = _step(**b)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got_a, want_a)) and all(torch.equal(x, y) for x, y in zip(got_b, want_b))
    graphs = []
    for s in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _step(**s)
        graphs.append((g, out))
    other = _step_inputs(63)
    want_o = [t.clone() for t in _step(**other)]
    for turn in range(4):
        for (g, out), want in zip(graphs, (want_a, want_b)):
            for t in out:
                t.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(out, want)), turn
            assert all(torch.equal(x, y) for x, y in zip(_step(**other), want_o))
    with torch.cuda.stream(sa):                                     # both graphs at once, on streams of their own
        graphs[0][0].replay()
    with torch.cuda.stream(sb):
        graphs[1][0].replay()
    torch.cuda.synchronize()
    for (g, out), want in zip(graphs, (want_a, want_b)):
        assert all(torch.equal(x, y) for x, y in zip(out, want))
    a["q"].copy_(a["q"].flip(0))                                    # other inputs in the same places
    want = _step(**a)
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(graphs[0][1], want))


@pytest.mark.gpu
def test_gpu_results_repeat():
    """the same call twice gives the same bits"""
    p = _problem([3000, 700], [4, 9], 8, 2, 128, 64, "bf16", "fp8", 71, mask="tree")
    first = ops.tree_attention(**p, want_lse=True)
    x = torch.randn(6, 50021, device="cuda", generator=_gen(1))
    t = torch.randint(0, 50021, (6,), device="cuda", generator=_gen(2))
    scores = ops.token_logprobs(x, t, top=9)
    for _ in range(5):
        again = ops.tree_attention(**p, want_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
        assert all(torch.equal(u, w) for u, w in zip(scores, ops.token_logprobs(x, t, top=9)))


@pytest.mark.gpu
def test_gpu_two_hip_runtimes_are_refused():
    """a process that loads the library before torch holds two HIP runtimes: a device pointer of one means nothing to the other"""
    code = ("from pero_ocr_amd import _native; _native.load()\nfrom pero_ocr_amd import decode_ops\n"
            "try:\n    decode_ops._lib()\nexcept RuntimeError as e:\n    print('refused' if 'two HIP runtimes' in str(e) else e)\n")
    import sys
    r = subprocess.run([sys.executable, "-c", code], cwd=REPO, capture_output=True, text=True, timeout=100)
    assert r.stdout.strip() == "refused", r.stdout + r.stderr
