"""Decoding operators (pero_ocr_amd/decode_ops.py) at the edges of what their documentation allows: outputs beside a padded batch, finite values
near the top of the range, scratch memory, tensors with tangents, a cache whose memory has moved."""
import pytest
import torch

from pero_ocr_amd import decode_ops as ops
from test_decode_ops import _check, _gen, _problem


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
