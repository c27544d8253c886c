"""Decoding operators (pero_ocr_amd/decode_ops.py) at the edges of what their documentation allows: outputs beside a padded batch, finite values
near the top of the range, scratch memory, tensors with tangents, a cache whose memory has moved."""
import math
import os
import re
import subprocess
import sys
import tempfile
import threading

import pytest
import torch

from pero_ocr_amd import _native, decode_ops as ops
from test_decode_ops import REPO, TYPES, _check, _fake_pages, _gen, _problem


@pytest.mark.gpu
@pytest.mark.parametrize("lengths, counts", [([20, 50], [2, 3]), ([3000, 2100], [2, 3])])
def test_gpu_padded_lse_beside_a_given_out(lengths, counts):
    """lse is made by the call also where out is the caller's: -inf behind the last sequence, whatever its memory held before, while
    the rows of out stay as they were; split over the positions or not"""
    p = _problem(lengths, counts, 4, 2, 64, 32, "bf16", "fp8", 41, mask="tree", tail=11)
    want, want_lse = ops.tree_attention(**p, want_lse=True)
    given = torch.full_like(want, 7.0)
    for _ in range(4):
        held = [torch.full((16, 4), 7.0, device="cuda") for _ in range(8)]          # what the allocator hands out next
        del held
        out, lse = ops.tree_attention(**p, out=given, want_lse=True)
        assert out is given and (given[5:] == 7).all() and torch.equal(given[:5], want[:5])
        assert torch.isneginf(lse[5:]).all() and torch.equal(lse, want_lse)


def _large(cache, kind, lengths, counts, value, seed, heads=2, kv_heads=1, dim=32, page=16):
    p = _problem(lengths, counts, heads, kv_heads, dim, page, kind, cache, seed, mask="tree")
    pages = p["pages"]
    num = pages.k.shape[0] * page
    k = torch.randn(num, kv_heads, dim, device="cuda", generator=_gen(seed)) * 0.25
    v = torch.full((num, kv_heads, dim), value, device="cuda")
    v[:, :, 1::2] = -value
    v[:, :, 5] = 1.0
    v[::3, :, 7] = value / 3
    ops.kv_write(pages, k, v, torch.arange(num, device="cuda"))
    return p


@pytest.mark.gpu
@pytest.mark.parametrize("cache, value", [("bf16", 3e38), ("bf16", 3.3895313892515355e38), ("fp8", 2.9e38)])
@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("lengths, counts", [([2], [1]), ([40, 9], [3, 1]), ([300, 33], [2, 17]), ([3000, 5], [1, 2])])
def test_gpu_attention_of_values_near_the_top_of_the_range(lengths, counts, kind, cache, value):
    """an average is no larger than the largest value: its sums do not pass the range on the way, in a wave, between waves or between splits"""
    p = _large(cache, kind, lengths, counts, value, 91)
    out, lse = ops.tree_attention(**p, want_lse=True)
    assert torch.isfinite(out).all()
    _check(p, kind, (out, lse))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_gpu_attention_of_large_values_all_widths(dim):
    for cache in ("bf16", "fp8"):
        p = _large(cache, "fp32", [70, 18], [20, 3], 2.9e38, 92, heads=4, kv_heads=2, dim=dim)
        _check(p, "fp32", ops.tree_attention(**p, want_lse=True))


def test_workspace_does_not_grow_with_padding():
    """scratch memory follows the rows that a batch can have by its own max_queries, not the rows it is padded to"""
    lib, p = _native.load(), 1 << 20

    def need(tokens, seqs, heads, kv_heads, dim, max_pages, most):
        pages = _fake_pages(num_pages=1 << 20, kv_heads=kv_heads, head_dim=dim)
        args = _native.TreeAttentionArgs(q=p, out=p, page_table=p, lengths=p, q_start=p, tokens=tokens, seqs=seqs, heads=heads, max_pages=max_pages, max_queries=most,
                                         q_head_stride=dim, q_token_stride=heads * dim, dtype=1)
        return lib.pocr_tree_attention_workspace(pages, args)
    for seqs, heads, kv_heads, dim, most in ((4, 64, 8, 128, 1), (1, 8, 8, 256, 1), (3, 32, 8, 64, 5), (16, 8, 8, 128, 1)):
        alone, padded = (need(n, seqs, heads, kv_heads, dim, 8192, most) for n in (seqs * most, 1024))
        rows = heads // kv_heads * most
        tile = 16 if rows <= 16 else 32                                # (padded, every sequence and key head has whole tiles of rows)
        assert 0 < alone <= padded <= alone * tile * -(-rows // tile) // rows
        for tokens in (8192, 100000):
            assert need(tokens, seqs, heads, kv_heads, dim, 8192, most) == padded
    # whatever is said of them, never more than 32 MB
    for tokens in (1, 7, 64, 1000, 30000, 1 << 20):
        for seqs in (1, 2, 30, 500):
            for heads, kv_heads, dim in ((1, 1, 32), (8, 8, 256), (64, 8, 128), (40, 2, 64)):
                for most in (0, 1, 33, tokens):
                    assert need(tokens, seqs, heads, kv_heads, dim, 1 << 16, most) <= 32 << 20


@pytest.mark.gpu
@pytest.mark.parametrize("counts", [[1, 1, 1], [1, 0, 1], [3, 2, 5]])
def test_gpu_padded_batch_costs_no_scratch_memory(counts):
    """the same rows, padded or not, and no more memory than outputs and zeros.  (Not always the same bits: padding may leave other tiles and
    splits, so sums in another order; what that may change is in the oracle's bounds.)"""
    p = _problem([9000, 2000, 40], counts, 16, 2, 64, 64, "bf16", "fp8", 95, mask="tree")
    n = sum(counts)
    for most in (max(counts), 1):
        want = ops.tree_attention(**p, max_queries=most, want_lse=True)
        _check(p, "bf16", want)
        tail = 5000
        wide = dict(p, q=torch.cat([p["q"], torch.ones(tail, 16, 64, device="cuda", dtype=torch.bfloat16)]), mask=torch.cat([p["mask"], torch.full((tail, 1), -1, device="cuda")]))
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        out, lse = ops.tree_attention(**wide, max_queries=most, want_lse=True)
        used = torch.cuda.max_memory_allocated() - before
        assert used <= out.numel() * 2 + lse.numel() * 4 + (32 << 20)
        _check(p, "bf16", (out[:n], lse[:n]))
        assert (out[n:] == 0).all() and torch.isneginf(lse[n:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("classes", [520, 1000, 2048])
def test_gpu_many_alternatives_do_not_cost_a_pass_each(classes, kind):
    """rows by the thousand: 64 alternatives take the time of 24 times a few, not of a pass over the row for each"""
    x = (torch.randn(16384, classes, device="cuda", generator=_gen(5)) * 3).to(kind)
    tokens = torch.zeros(16384, dtype=torch.int64, device="cuda")

    def time(top):
        ops.token_logprobs(x, tokens, top=top)
        best = math.inf
        for _ in range(5):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(5):
                ops.token_logprobs(x, tokens, top=top)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best
    few = time(24)
    for top in (28, 32, 64):
        assert time(top) <= 5 * few, top


def _dual_calls(device):
    from torch.autograd import forward_ad
    x = torch.ones(3, 2, 64, device=device)
    ids = torch.zeros(3, dtype=torch.int64, device=device)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        rows = forward_ad.make_dual(x[:, 0], torch.ones_like(x[:, 0]))
        half = torch.zeros(2, 2, 16, 64, dtype=torch.bfloat16, device=device)
        with pytest.raises(RuntimeError, match="derivative"):
            ops.token_logprobs(rows, ids)
        with pytest.raises(RuntimeError, match="derivative"):
            ops.KVPages(forward_ad.make_dual(half, half.clone()), half.clone())
        if device == "cuda":
            pages = ops.kv_pages(2, 2, 16, 64)
            plain = x.clone()
            for k, v in ((dual, plain), (plain, dual)):
                with pytest.raises(RuntimeError, match="derivative"):
                    ops.kv_write(pages, k, v, ids)
            p = _problem([20], [3], 2, 2, 64, 16, "fp32", "fp8", 1)
            with pytest.raises(RuntimeError, match="derivative"):
                ops.tree_attention(**dict(p, q=dual))
            with pytest.raises(RuntimeError, match="derivative"):
                ops.tree_attention(**p, out=dual)
            cache = ops.kv_pages(2, 2, 16, 64, dtype="bf16")
            cache.k.copy_(forward_ad.make_dual(half, torch.ones_like(half)))          # (the tangent comes with the numbers)
            for call in (lambda: ops.kv_read(cache, ids), lambda: ops.tree_attention(**dict(p, pages=cache))):
                with pytest.raises(RuntimeError, match="derivative"):
                    call()
            ops.tree_attention(**p)                                    # (tensors without a tangent, inside the level)
            ops.token_logprobs(x[:, 0], ids)


def test_tangents_are_refused():
    """forward-mode derivatives: refused as gradients are, not dropped in silence"""
    _dual_calls("cpu")


@pytest.mark.gpu
def test_gpu_tangents_are_refused():
    _dual_calls("cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp8", "bf16"])
def test_gpu_cache_tensors_stay(dtype):
    """the tensors of a cache cannot be exchanged"""
    pages = ops.kv_pages(4, 2, 16, 64, dtype=dtype)
    for name in ("k", "v", "k_exp", "v_exp", "index", "native"):
        with pytest.raises(AttributeError):
            setattr(pages, name, getattr(pages, name))
        with pytest.raises(AttributeError):
            delattr(pages, name)


def _as_if(monkeypatch, dtype):
    """a KVPages of CPU tensors, past the check of the device: what is looked at before anything is enqueued"""
    monkeypatch.setattr(ops.KVPages, "_refuse", staticmethod(lambda *a: None))
    shape = (4, 2, 16, 64)
    if dtype == "bf16":
        return ops.KVPages(*(torch.zeros(shape, dtype=torch.bfloat16) for _ in range(2)))
    return ops.KVPages(*(torch.zeros(shape, dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2)), *(torch.zeros(shape[:3], dtype=torch.uint8) for _ in range(2)))


@pytest.mark.parametrize("dtype, name", [("bf16", "k"), ("bf16", "v"), ("fp8", "k"), ("fp8", "v"), ("fp8", "k_exp"), ("fp8", "v_exp")])
def test_cache_that_has_moved_is_refused(monkeypatch, dtype, name):
    """other storage under a tensor of the cache: every call raises before the library sees a pointer"""
    def never(*a):
        raise AssertionError("the library was called")
    monkeypatch.setattr(ops, "_lib", never)
    for how in ("data", "set_", "freed"):
        pages = _as_if(monkeypatch, dtype)
        assert pages.plan() is pages.native
        t = getattr(pages, name)
        keep = t.untyped_storage()                                     # (its memory stays taken: the new one lies elsewhere)
        if how == "data":
            t.data = torch.empty_like(t)
        elif how == "set_":
            t.set_(torch.empty_like(t))
        else:
            keep.resize_(0)
        x = torch.zeros(3, 2, 64)
        ids = torch.zeros(3, dtype=torch.int64)
        one = torch.ones(1, dtype=torch.int32)
        for call in (pages.plan, lambda: ops.kv_write(pages, x, x, ids), lambda: ops.kv_read(pages, ids),
                     lambda: ops.tree_attention(x, pages, one[:, None], one, torch.tensor([0, 3], dtype=torch.int32))):
            with pytest.raises(RuntimeError, match="other memory"):
                call()


def test_no_kernel_of_any_unit_spills():
    """test_host.py's rule for the whole library: scratch memory per lane is 0 for every kernel of every translation unit"""
    sys.path.insert(0, os.path.join(REPO, "tools"))
    try:
        from codeobj_hash import code_objects
    finally:
        sys.path.pop(0)
    tool = "/opt/rocm/lib/llvm/bin/llvm-readelf"
    if not os.path.exists(tool):
        pytest.skip("llvm-readelf is not here")
    seen = {}
    for elf in code_objects(_native.lib_path()):
        with tempfile.NamedTemporaryFile(suffix=".co") as f:
            f.write(elf)
            f.flush()
            notes = subprocess.run([tool, "--notes", f.name], capture_output=True, text=True, check=True).stdout
        for block in notes.split("- .agpr_count:")[1:]:
            seen[re.search(r"\.symbol:\s*(\S+)", block).group(1)] = int(re.search(r"\.private_segment_fixed_size:\s*(\d+)", block).group(1))
    for kernel in ("tree_attention_kernel", "token_logprobs_kernel", "kv_write_kernel", "ctc"):
        assert any(kernel in name for name in seen), kernel
    assert [name for name, size in seen.items() if size] == []


def test_tools_see_every_code_object():
    """the tools that read the built library's kernels read those of every translation unit"""
    tool = "/opt/rocm/lib/llvm/bin/llvm-readelf"
    if not os.path.exists(tool):
        pytest.skip("llvm-readelf is not here")
    tools = os.path.join(REPO, "tools")
    hashes = subprocess.run([sys.executable, os.path.join(tools, "codeobj_hash.py")], capture_output=True, text=True, check=True).stdout
    assert len(hashes.splitlines()) == len(__import__("__graft_entry__").SOURCES)
    names = subprocess.run([sys.executable, "-c", "import codeobj_hash as c, sys; print(*c.kernels(sys.argv[1]))", _native.lib_path()], cwd=tools, capture_output=True,
                           text=True, check=True).stdout
    meta = subprocess.run([sys.executable, os.path.join(tools, "kernel_meta.py")], capture_output=True, text=True, check=True).stdout
    for kernel in ("tree_attention_kernel", "token_logprobs_kernel", "kv_write_kernel", "ctc"):
        assert kernel in names and kernel in meta, kernel


@pytest.mark.gpu
@pytest.mark.parametrize("kind, cache", [("fp32", "bf16"), ("bf16", "fp8"), ("fp16", "fp8")])
@pytest.mark.parametrize("heads, kv_heads, dim", [(2, 1, 64), (4, 1, 128), (2, 2, 32)])
def test_gpu_long_chains(heads, kv_heads, dim, kind, cache):
    """prompts: hundreds of new tokens, each up to itself, with and without older positions, at the borders of tiles and blocks"""
    for lengths, counts in (([300], [300]), ([129, 417, 33], [129, 150, 1]), ([700], [257])):
        p = _problem(lengths, counts, heads, kv_heads, dim, 32, kind, cache, 101)
        _check(p, kind, ops.tree_attention(**p, want_lse=True))
        _check(p, kind, ops.tree_attention(**p, max_queries=max(counts), want_lse=True))


@pytest.mark.gpu
@pytest.mark.parametrize("over", [1, 40, 1 << 20])
def test_gpu_lengths_beyond_the_table(over):
    """a length beyond the page table counts as the positions that the table has: the new tokens are the last of these"""
    p = _problem([64, 64], [5, 2], 2, 1, 64, 16, "fp32", "fp8", 103, mask="tree")
    want = ops.tree_attention(**p, want_lse=True)
    _check(p, "fp32", want)
    got = ops.tree_attention(**dict(p, lengths=p["lengths"] + over), want_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_gpu_expanded_arguments():
    """one table, query, mask row, key, value, or row of logits for all: strides of zero"""
    p = _problem([70, 70, 70], [2, 2, 2], 4, 2, 64, 16, "bf16", "fp8", 105, mask="tree")
    p["page_table"], p["q"], p["mask"] = p["page_table"][:1].expand(3, -1), p["q"][:1].expand(6, -1, -1), p["mask"][1:2].expand(6, -1)
    whole = dict(p, page_table=p["page_table"].contiguous(), q=p["q"].contiguous(), mask=p["mask"].contiguous())
    assert torch.equal(ops.tree_attention(**p), ops.tree_attention(**whole))
    _check(whole, "bf16", ops.tree_attention(**p, want_lse=True))
    pages, same = ops.kv_pages(2, 2, 16, 64), ops.kv_pages(2, 2, 16, 64)
    row, ids = torch.randn(1, 2, 64, device="cuda", generator=_gen(7)), torch.arange(9, device="cuda")
    ops.kv_write(pages, row.expand(9, -1, -1), row[:, :1].expand(9, 2, -1), ids)
    ops.kv_write(same, row.expand(9, -1, -1).contiguous(), row[:, :1].expand(9, 2, -1).contiguous(), ids)
    for a, b in ((pages.k, same.k), (pages.v, same.v), (pages.k_exp, same.k_exp), (pages.v_exp, same.v_exp)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    for a, b in zip(ops.kv_read(pages, torch.zeros(5, dtype=torch.int64, device="cuda")), ops.kv_read(pages, ids[:1])):
        assert torch.equal(a, b.expand_as(a))                            # the same slot again and again
    x, t = torch.randn(1, 700, device="cuda", generator=_gen(8)), torch.arange(20, device="cuda")
    for a, b in zip(ops.token_logprobs(x.expand(20, -1), t, top=5), ops.token_logprobs(x.expand(20, -1).contiguous(), t, top=5)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_gpu_offset_integer_arguments():
    """lengths, q_start, slots, tokens and mask rows that start in the middle of a tensor: aligned to an element, no more"""
    p = _problem([70, 45], [3, 2], 4, 2, 64, 16, "bf16", "fp8", 107, mask="tree")
    want = ops.tree_attention(**p)
    moved = {k: torch.cat([p[k][:1], p[k]])[1:] for k in ("lengths", "q_start", "mask")}
    wide = torch.full((2, p["page_table"].shape[1] + 1), 7, dtype=torch.int32, device="cuda")
    wide[:, 1:] = p["page_table"]
    assert torch.equal(ops.tree_attention(**dict(p, page_table=wide[:, 1:], **moved)), want)
    x = torch.randn(6, 300, device="cuda", generator=_gen(9))
    for kind in (torch.int32, torch.int64):
        t = torch.arange(7, device="cuda", dtype=kind)
        assert torch.equal(ops.token_logprobs(x, t[1:])[0], ops.token_logprobs(x, t[1:].clone())[0])
        for a, b in zip(ops.kv_read(p["pages"], t[1:]), ops.kv_read(p["pages"], t[1:].clone())):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_gpu_threads():
    """calls from several threads at once, each on a stream of its own"""
    problems = [_problem([300 + 7 * i, 2100], [3, 2], 8, 2, 64, 16, "bf16", "fp8", 110 + i, mask="tree") for i in range(4)]
    x = torch.randn(5, 120000, device="cuda", generator=_gen(11))
    t = torch.arange(5, device="cuda")
    want = [[u.clone() for u in ops.tree_attention(**p, want_lse=True)] for p in problems]
    scores = [u.clone() for u in ops.token_logprobs(x, t, top=4)]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got, again = ops.tree_attention(**problems[i], want_lse=True), ops.token_logprobs(x, t, top=4)
                stream.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])) or not all(torch.equal(a, b) for a, b in zip(again, scores)):
                    bad.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not bad


@pytest.mark.gpu
def test_gpu_inference_mode():
    with torch.inference_mode():
        p = _problem([40, 21], [6, 5], 2, 1, 64, 16, "fp32", "fp8", 115, mask="tree")
        _check(p, "fp32", ops.tree_attention(**p, want_lse=True))
        x = torch.randn(3, 50, device="cuda")
        assert ops.token_logprobs(x, torch.arange(3, device="cuda"), top=2)[2].shape == (3, 2)


@pytest.mark.gpu
def test_gpu_first_calls_of_a_process_may_be_captured():
    """nothing has to run eagerly before a capture: the first calls of a process, recorded, replayed and compared with eager ones"""
    code = """
import torch
from pero_ocr_amd import decode_ops as ops
pages = ops.kv_pages(40, 2, 16, 64)
k, v = (torch.randn(600, 2, 64, device="cuda") for _ in range(2))
slots = torch.arange(600, device="cuda")
q = torch.randn(3, 4, 64, device="cuda")
table = torch.arange(38, device="cuda", dtype=torch.int32)[None]
lengths, starts = torch.tensor([600], device="cuda", dtype=torch.int32), torch.tensor([0, 3], device="cuda", dtype=torch.int32)
x, t = torch.randn(3, 120000, device="cuda"), torch.arange(3, device="cuda")
def step():
    ops.kv_write(pages, k, v, slots)
    return ops.kv_read(pages, slots) + ops.tree_attention(q, pages, table, lengths, starts, want_lse=True) + ops.token_logprobs(x, t, top=3)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = step()
for turn in range(3):
    for o in out:
        o.zero_()
    g.replay()
    torch.cuda.synchronize()
    print("same" if all(torch.equal(a, b) for a, b in zip(out, step())) else "different", flush=True)
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=REPO, capture_output=True, text=True, timeout=100)
    assert r.stdout.split() == ["same"] * 3, r.stdout + r.stderr


@pytest.mark.parametrize("dtype", ["bf16", "fp8"])
@pytest.mark.parametrize("name", ["k", "v"])
def test_cache_that_requires_a_gradient_is_refused(monkeypatch, dtype, name):
    """also where it came to require one behind the making of the KVPages, or was made while none was recorded"""
    def reached(*a):
        raise ZeroDivisionError("the library was called")
    monkeypatch.setattr(ops, "_lib", reached)
    monkeypatch.setattr(ops, "_stream", lambda index: 0)
    x = torch.zeros(3, 2, 64)
    ids = torch.zeros(3, dtype=torch.int64)
    pages = _as_if(monkeypatch, dtype)
    with torch.no_grad():
        getattr(pages, name).requires_grad_()
    calls = (lambda: ops.kv_read(pages, ids), lambda: ops.kv_write(pages, x, x, ids),
             lambda: ops.tree_attention(x, pages, *(torch.ones(s, dtype=torch.int32) for s in ((1, 1), (1,), (2,)))))
    for call in calls:
        with pytest.raises(RuntimeError, match="gradient"):
            call()
    with torch.no_grad():
        monkeypatch.setattr(ops, "_need", lambda *a: None)              # (past the device: without recording a call goes on to the library)
        for call in calls:
            with pytest.raises(ZeroDivisionError):
                call()


@pytest.mark.gpu
def test_gpu_rounding_at_the_end_of_the_range():
    """half a step below 2^128 an 8-bit element is rounded to it, by the rule for all others: it reads as infinity.  Below that finite numbers stay finite"""
    edge = 2.0 ** 128 * (1 - 2.0 ** -5)                                  # between codes 240 and 256, of which the latter is even
    x = torch.ones(4, 1, 32, device="cuda")
    x[0, 0, 3], x[1, 0, 3], x[2, 0, 3], x[3, 0, 3] = edge, -edge, 3.296e38, torch.finfo(torch.float32).max
    pages = ops.kv_pages(1, 1, 16, 32)
    ops.kv_write(pages, x, x, torch.arange(4, device="cuda"))
    k, _v = ops.kv_read(pages, torch.arange(4, device="cuda"))
    assert k[:, 0, 3].tolist() == [math.inf, -math.inf, 240 * 2.0 ** 120, math.inf]
    assert pages.k_exp[0, 0, :4].tolist() == [247] * 4 and pages.k[0, 0, :4, 3].float().tolist() == [256.0, -256.0, 240.0, 256.0]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("cache", ["fp8", "bf16"])
@pytest.mark.parametrize("dim", [32, 64, 128, 256])
def test_gpu_attention_many_rows_all_types(dim, cache, kind):
    """trees with more rows than one tile, in every type: two tiles a wave where they fit; in splits, in one piece, and with waves alone"""
    p = _problem([37, 90, 33, 70], [33, 17, 20, 41], 4, 2, dim, 16, kind, cache, 121, mask="tree")
    _check(p, kind, ops.tree_attention(**p, max_queries=41, want_lse=True))
    p = _problem([700, 20], [33, 18], 2, 1, dim, 32, kind, cache, 122, mask="any")
    for most in (0, 33):
        _check(p, kind, ops.tree_attention(**p, max_queries=most, want_lse=True))
    n = 2050                                                            # (more workgroups than two waves a SIMD: a wave each)
    p = _problem([9] * n, [1] * n, 1, 1, dim, 16, kind, cache, 123)
    got = ops.tree_attention(**p, max_queries=1, want_lse=True)
    few = dict(p, q=p["q"][:40], page_table=p["page_table"][:40], lengths=p["lengths"][:40], q_start=p["q_start"][:41])
    _check(few, kind, [t[:40] for t in got])
    for a, b in zip(got, ops.tree_attention(**dict(p, max_queries=0), want_lse=True)):
        assert torch.allclose(a.float(), b.float(), rtol=2 ** -7, atol=2 ** -7)          # the same sums in another order


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_gpu_probabilities_keep_seventeen_bits(kind):
    """The weight of one key against values that take it away again.  Three keys with scores c < 0, 0, 0 and values 1, -x1, -x2, where x1 + x2 is e^c as
    two bfloat16 numbers: out (2 + e^c) = e^c (1 + d) - x1 - x2, small enough for its own rounding not to hide d.  The kernel's e^c is
    off by 4 u (1 + |c|) and as two planes by 2^-17; sums, divisions and the remaining roundings by a few u: |d| <= 2^-17 + 16 u (1 + |c|), and half a
    step of the output's type on top."""
    dim, tokens = 32, 400
    dt = TYPES[kind]
    c = (-torch.rand(tokens, device="cuda", generator=_gen(131)) * 4 - 2.0 ** -6).bfloat16()
    want = torch.exp(c.double())
    x1 = want.bfloat16()
    x2 = (want - x1.double()).bfloat16()
    pages = ops.kv_pages(tokens, 1, 16, dim, dtype="bf16")
    pages.k[:, 0, 0, 0] = 1
    for at, x in ((0, torch.ones_like(x1)), (1, -x1), (2, -x2)):
        pages.v[:, 0, at] = x[:, None]
    q = torch.zeros(tokens, 1, dim, device="cuda", dtype=dt)
    q[:, 0, 0] = c.to(dt)
    c = q[:, 0, 0].double()                                             # (float16 holds these eight bits too, or what it holds is the score)
    want = torch.exp(c)
    out = ops.tree_attention(q, pages, torch.arange(tokens, dtype=torch.int32, device="cuda")[:, None], torch.full((tokens,), 3, dtype=torch.int32, device="cuda"),
                             torch.arange(tokens + 1, dtype=torch.int32, device="cuda"), scale=1.0, max_queries=1)
    assert (out == out[:, :, :1]).all()
    exact = (want - x1.double() - x2.double()) / (2 + want)
    off = (out[:, 0, 0].double() - exact).abs()
    allowed = want / (2 + want) * (2.0 ** -17 + 16 * 2.0 ** -24 * (1 + c.abs()))
    half = torch.finfo(dt).eps / 2 * (exact.abs() + allowed) + (2.0 ** -25 if kind == "fp16" else 0)          # (float16 has fixed steps of 2^-24 below 2^-14)
    assert (off <= allowed + half).all(), (off / (allowed + half)).max()
