"""The norm of query and key heads fused with the rotation (and with the paged-cache write), against fp64.

Tolerance. The output is one rounding (half a step: eps / 2 relative) of an fp32 value. That value's own error: the sum of
squares of a head of D <= 512 (all terms positive) is off by at most the 16 + log2(32) = 21 additions of the vector form,
or 2 D / 64 + 5 = 21 of the scalar form, each 2^-24, halved by the square root; the division, rsqrtf (2 steps), three
products and the sum add 7: 18 * 2^-24 of the sum's magnitude |y_i cos| + |y_j sin| at most. In sincos mode the angle is
exact by definition (fp32) and sincosf is off by 2 steps of 1, which is counted on the magnitude too (22 in all, taken as
24). fp16 outputs below the normal range step by 2^-24: half of that is added."""

import pytest
import torch

from ckb200 import rope
from helpers import CANARY, bits_equal, misaligned_copy
from oracle import rope as orope
from oracle import serving

pytestmark = pytest.mark.gpu


def assert_near(got, want, size, what):
    bound = torch.finfo(got.dtype).eps / 2 * (want.abs() + 24 * 2.0 ** -24 * size) + 24 * 2.0 ** -24 * size + 2.0 ** -25
    err = (got.cpu().double() - want).abs()
    assert not got.isnan().any(), what
    assert (err <= bound).all(), f"{what}: {(err / bound).max().item():.3f} of the bound"


def heads(layout, g, dtype, b, s, hq, hkv, d):
    """q, k, v on the GPU in a layout: of their own, views of one projection, or with the heads before the tokens."""
    sizes = (hq, hkv, hkv)
    if layout == "fused":
        x = torch.randn(b, s, sum(sizes) * d, generator=g).to(dtype).cuda()
        return [t.view(b, s, n, d) for t, n in zip(x.split([n * d for n in sizes], -1), sizes)]
    if layout == "heads_first":
        return [torch.randn(b, n, s, d, generator=g).to(dtype).cuda().transpose(1, 2) for n in sizes]
    x = [torch.randn(b, s, n, d, generator=g).to(dtype).cuda() for n in sizes]
    return [misaligned_copy(t) for t in x] if layout == "misaligned" else x


SHAPES = [  # dtype, weight dtype, cache dtype, B, S, Hq, Hkv, D, layout
    (torch.bfloat16, torch.bfloat16, torch.float32, 2, 37, 32, 8, 128, "fused"),
    (torch.bfloat16, torch.float32, torch.float32, 64, 1, 32, 8, 128, "fused"),
    (torch.float16, torch.float16, torch.bfloat16, 3, 19, 12, 2, 64, "plain"),
    (torch.float16, torch.float32, torch.float16, 1, 1, 1, 1, 256, "plain"),
    (torch.bfloat16, torch.bfloat16, torch.bfloat16, 2, 5, 7, 7, 80, "heads_first"),  # 5 of 8 lanes
    (torch.bfloat16, torch.float16, torch.float32, 1, 301, 5, 1, 96, "fused"),
    (torch.float16, torch.bfloat16, torch.float32, 2, 3, 3, 1, 512, "plain"),
    (torch.bfloat16, torch.bfloat16, torch.float32, 2, 9, 4, 2, 40, "plain"),  # the scalar form: D
    (torch.float16, torch.float16, torch.float32, 2, 9, 4, 2, 2, "plain"),
    (torch.bfloat16, torch.bfloat16, torch.float32, 2, 9, 6, 2, 128, "misaligned"),  # and the alignment
    (torch.bfloat16, torch.bfloat16, torch.float32, 1, 4096, 40, 8, 128, "fused"),  # many tokens: five heads a thread
]


@pytest.mark.parametrize("dtype,w_dtype,c_dtype,b,s,hq,hkv,d,layout", SHAPES)
def test_matches_fp64(dtype, w_dtype, c_dtype, b, s, hq, hkv, d, layout):
    g = torch.Generator().manual_seed(d + s)
    q, k, v = heads(layout, g, dtype, b, s, hq, hkv, d)
    qw, kw = ((1 + 0.3 * torch.randn(d, generator=g)).to(w_dtype) for _ in range(2))
    cos, sin = orope.cos_sin_cache(10000.0, d, 4096, c_dtype)
    ids = torch.randint(0, 4096, (b, s), generator=g)
    args = [t.cuda() for t in (qw, kw, cos, sin)]
    wq, sq = serving.norm_rotate(q.cpu(), qw, cos[ids], sin[ids], 1e-5)
    wk, sk = serving.norm_rotate(k.cpu(), kw, cos[ids], sin[ids], 1e-5)
    before = [t.clone() for t in (q, k, v)]
    q_out, k_out = rope.qk_norm_rope(q, k, ids.cuda(), *args, eps=1e-5)
    assert_near(q_out, wq, sq, "q")
    assert_near(k_out, wk, sk, "k")
    assert bits_equal(q, before[0]) and bits_equal(k, before[1]), "the inputs stay"

    slots = torch.randperm(b * s + 40, generator=g)[:b * s].view(b, s)
    slots[0, 0] = -1
    slots[-1, -1] = b * s + 48  # beyond the cache: not written either
    caches = [torch.full((b * s + 48, 1, hkv, d), CANARY[dtype], dtype=dtype, device="cuda") for _ in range(2)]
    q2, k2 = rope.qk_norm_rope_kv_cache(q, k, v, ids.cuda(), *args, *caches, slots.cuda(), eps=1e-5, inplace=False)
    assert bits_equal(q2, q_out) and bits_equal(k2, k_out)
    keep = ((slots >= 0) & (slots < b * s + 48)).view(-1)
    rows = slots.view(-1)[keep].cuda()
    for cache, new in zip(caches, (k_out, v)):
        want = torch.full_like(cache, CANARY[dtype])
        want.view(-1, hkv, d)[rows] = new.reshape(-1, hkv, d)[keep.cuda()]
        assert bits_equal(cache, want), "cache rows"
    q3, k3 = rope.qk_norm_rope_kv_cache(q, k, v, ids.cuda(), *args, *caches, slots.cuda(), eps=1e-5, write_k=False)
    assert k3 is None and q3.data_ptr() == q.data_ptr()
    assert bits_equal(q, q_out) and bits_equal(k, before[1]) and bits_equal(v, before[2]), "q in place, k and v stay"


def test_in_place_through_a_fused_projection_writes_nothing_else():
    g = torch.Generator().manual_seed(5)
    x = torch.randn(2, 33, 12 * 64 + 24, generator=g).to(torch.bfloat16).cuda()  # 24 columns of something else
    before = x.clone()
    q, k, v = (t.unflatten(-1, (-1, 64)) for t in x[..., : 12 * 64].split([8 * 64, 2 * 64, 2 * 64], -1))
    w = torch.ones(64, device="cuda")
    ids = torch.arange(33, device="cuda").repeat(2, 1)
    want_q, want_k = rope.qk_norm_rope(q, k, ids, w, w, theta=10000.0)
    q_out, k_out = rope.qk_norm_rope(q, k, ids, w, w, theta=10000.0, inplace=True)
    assert q_out.data_ptr() == x.data_ptr()
    assert bits_equal(q_out, want_q) and bits_equal(k_out, want_k)
    assert bits_equal(x[..., 10 * 64:], before[..., 10 * 64:])


def test_sincos_mode_and_far_positions():
    g = torch.Generator().manual_seed(6)
    q, k = (torch.randn(2, 17, n, 128, generator=g).to(torch.bfloat16) for n in (4, 2))
    w = 1 + 0.1 * torch.randn(128, generator=g)
    ids = torch.randint(0, 1 << 20, (2, 17), generator=g)
    angle = (ids.float()[..., None] * rope.inv_freq(1e6, 128, "cpu")).double()
    cos, sin = (torch.cat([f(angle)] * 2, -1) for f in (torch.cos, torch.sin))
    got = rope.qk_norm_rope(q.cuda(), k.cuda(), ids.cuda(), w.cuda(), w.cuda(), theta=1e6)
    for o, x, what in zip(got, (q, k), "qk"):
        assert_near(o, *serving.norm_rotate(x, w, cos, sin, 1e-6), what)


def test_rows_of_zeros_huge_and_not_finite_values():
    d = 64
    q = torch.ones(1, 4, 2, d)
    q[0, 0] = 0.0
    q[0, 1] = 65504.0  # squares reach 4.3e9 and their sum 2.7e11: within fp32
    q[0, 2, 0, 5] = float("nan")
    q[0, 3, 1, 7] = float("inf")
    q = q.half().cuda()
    w = torch.ones(d, device="cuda")
    ids = torch.zeros(1, 4, dtype=torch.int64, device="cuda")
    cos, sin = (t.cuda() for t in orope.cos_sin_cache(10000.0, d, 8))
    out, _ = rope.qk_norm_rope(q, q.clone(), ids, w, w, cos, sin)
    assert (out[0, 0] == 0).all()
    assert_near(out[0, 1], torch.ones(2, d, dtype=torch.float64), torch.ones(2, d, dtype=torch.float64), "huge")
    assert out[0, 2, 0].isnan().all() and (out[0, 2, 1] == 1).all(), "a NaN stays in its head"
    assert out[0, 3, 1, 7].isnan() and (out[0, 3, 0] == 1).all()


def test_positions_outside_the_cache_take_the_nearest_row_and_empty_batches_pass():
    g = torch.Generator().manual_seed(7)
    q = torch.randn(1, 3, 2, 64, generator=g).to(torch.bfloat16).cuda()
    w = torch.ones(64, device="cuda")
    cos, sin = (t.cuda() for t in orope.cos_sin_cache(10000.0, 64, 16))
    far = rope.qk_norm_rope(q, q.clone(), torch.tensor([[-3, 16, 1 << 40]], device="cuda"), w, w, cos, sin)[0]
    near = rope.qk_norm_rope(q, q.clone(), torch.tensor([[0, 15, 15]], device="cuda"), w, w, cos, sin)[0]
    assert bits_equal(far, near)
    none = torch.empty(0, 5, 2, 64, dtype=torch.bfloat16, device="cuda")
    out, _ = rope.qk_norm_rope(none, none, torch.empty(0, 5, dtype=torch.int64, device="cuda"), w, w, cos, sin)
    assert out.shape == none.shape


def test_other_stream_and_graph_replay():
    g = torch.Generator().manual_seed(8)
    q, k = (torch.randn(4, 1, n, 128, generator=g).to(torch.bfloat16).cuda() for n in (8, 2))
    w = torch.ones(128, device="cuda")
    ids = torch.randint(0, 64, (4, 1), generator=g).cuda()
    cos, sin = (t.cuda() for t in orope.cos_sin_cache(10000.0, 128, 64))
    want = rope.qk_norm_rope(q, k, ids, w, w, cos, sin)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = rope.qk_norm_rope(q, k, ids, w, w, cos, sin)
    q.add_(1)
    want2 = rope.qk_norm_rope(q, k, ids, w, w, cos, sin)
    graph.replay()
    torch.cuda.synchronize()
    assert bits_equal(got[0], want2[0]) and bits_equal(got[1], want[1])


@pytest.mark.parametrize("d,layout", [(128, "fused"), (40, "plain")])  # the vector and the scalar form
def test_sincos_mode_with_the_cache_write(d, layout):
    """theta in place of the cos/sin cache: the caches get what the call without them gives."""
    g = torch.Generator().manual_seed(9)
    q, k, v = heads(layout, g, torch.bfloat16, 3, 21, 8, 2, d)
    w = (1 + 0.1 * torch.randn(d, generator=g)).cuda()
    ids = torch.randint(0, 1 << 17, (3, 21), generator=g).cuda()
    slots = torch.randperm(80, generator=g)[:63].view(3, 21).cuda()
    caches = [torch.zeros(5, 16, 2, d, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    want_q, want_k = rope.qk_norm_rope(q, k, ids, w, w, theta=5e5)
    got_q, got_k = rope.qk_norm_rope_kv_cache(q, k, v, ids, w, w, None, None, *caches, slots, theta=5e5, inplace=False)
    assert bits_equal(got_q, want_q) and bits_equal(got_k, want_k)
    for cache, new in zip(caches, (want_k, v)):
        assert bits_equal(cache.view(-1, 2, d)[slots.flatten()], new.reshape(-1, 2, d))
        assert (cache.view(-1, 2, d).abs().amax((1, 2)) > 0).sum() == 63
