"""Paged attention, with and without a shared prefix, against fp64.

Tolerance, relative to `size`, the weighted mean of |v| (at least |out|). The output's rounding is half a step of its type,
and so is that of each weight exp(x - m) that multiplies a v: eps / 2 each. A score is a sum of D products in fp32, taken
16 at a time (D / 16 additions, at most 16 more within a step), then a scaling, a subtraction and an exponential (4 more,
2^-23 each): off by (D / 16 + 20) 2^-23 of A = max scale sum |q_d k_d|, which changes a weight, and twice that a quotient.
Joining and summing the pieces adds 2^-18 at most (64 additions of 2^-24). fp16 weights below 2^-14 are off by half of
2^-24 each, n of them by n 2^-25 of the largest |v|."""

import pytest
import torch

from ckb200 import attention, rope, softmax, verify
from helpers import bits_equal, guarded_empty
from oracle import rope as orope
from oracle import serving

pytestmark = pytest.mark.gpu


def problem(seed, dtype, t, hq, hkv, d, block_size, lens, prefix=0, spare=0, scale=1.0):
    """CPU tensors of a batch whose unused cache rows, and rows behind each length, hold NaN."""
    g = torch.Generator().manual_seed(seed)
    b = len(lens)
    width = max(1, -(-max([prefix + 1, *lens]) // block_size)) + spare
    shared = prefix // block_size
    blocks = shared + b * (width - shared) + 3
    ids = torch.randperm(blocks, generator=g)
    tables = torch.cat([ids[:shared].expand(b, shared), ids[shared:shared + b * (width - shared)].view(b, -1)], 1).contiguous()
    q = (scale * torch.randn(b, t, hq, d, generator=g)).to(dtype)
    caches = [torch.full((blocks, block_size, hkv, d), float("nan"), dtype=dtype) for _ in range(2)]
    for cache in caches:
        for i, n in enumerate(lens):
            new = torch.randn(width * block_size, hkv, d, generator=g).to(dtype)
            for j in range(shared, -(-n // block_size)):
                rows = min(block_size, n - j * block_size)
                cache[tables[i, j], :rows] = new[j * block_size:j * block_size + rows]
        for j in range(shared):
            cache[tables[0, j]] = torch.randn(block_size, hkv, d, generator=g).to(dtype)
    return q, *caches, tables, torch.tensor(lens)


def assert_near(got, q, kc, vc, tables, lens, prefix, scale=None):
    d = q.shape[3]
    scale = d ** -0.5 if scale is None else scale
    want, size = serving.attend(q, kc, vc, tables, lens, scale, prefix)
    eps, n = torch.finfo(q.dtype).eps, tables.shape[1] * kc.shape[1]
    k = kc[kc.isfinite()].double().abs().max().item() if kc.isfinite().any() else 0.0
    v = vc[vc.isfinite()].double().abs().max().item() if vc.isfinite().any() else 0.0
    a = scale * q.double().abs().sum(-1).max().item() * k  # at least max scale sum |q_d k_d|
    bound = eps / 2 * (want.abs() + size) + 2 * size * ((d / 16 + 20) * 2.0 ** -23 * a + 2.0 ** -18)
    if q.dtype == torch.float16:
        bound = bound + n * 2.0 ** -25 * v + 2.0 ** -25
    got = got.cpu().double()
    assert torch.equal(got.isnan(), want.isnan()), "NaN pattern"
    fine = want.isfinite()
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()]), "infinities"
    err = (got - want).abs()
    assert (err[fine] <= bound[fine] + 1e-30).all(), f"{(err / (bound + 1e-30))[fine].max().item():.3f} of the bound"


def check(q, kc, vc, tables, lens, prefix=0, **kw):
    got = attention.paged_attention(q.cuda(), kc.cuda(), vc.cuda(), tables.cuda(), lens.cuda(), shared_prefix=prefix, **kw)
    assert_near(got, q, kc, vc, tables, lens, prefix, kw.get("scale"))
    return got


BF, HF = torch.bfloat16, torch.float16
OWN = [  # dtype, T, Hq, Hkv, D, block size, lengths
    (BF, 1, 32, 8, 128, 16, [1]),
    (BF, 1, 32, 8, 128, 16, [64, 63, 65, 0, 1, 1000]),
    (HF, 1, 8, 8, 64, 32, [5, 130, 17]),
    (BF, 4, 8, 2, 128, 16, [4, 5, 3, 0, 200, 128]),  # 16 rows; the third has fewer tokens than queries
    (HF, 5, 8, 2, 64, 7, [70, 69, 500]),  # 20 rows; an odd block size
    (BF, 8, 14, 2, 80, 16, [300, 9]),  # 56 rows
    (BF, 6, 24, 2, 96, 128, [129, 6]),  # 72 rows: two row tiles
    (BF, 1, 4, 1, 256, 16, [333, 64]),
    (HF, 9, 4, 2, 256, 16, [100]),  # 18 rows
    (HF, 17, 4, 2, 200, 64, [100, 18]),  # 34 rows
    (BF, 1, 3, 3, 8, 1, [70, 2]),
    (HF, 2, 2, 1, 40, 48, [49, 1]),
    (BF, 1, 8, 2, 128, 16, [4000]),  # a row cut into many pieces
    (BF, 1, 2, 1, 64, 16, [17] * 200),  # many sequences of one tile
    (HF, 3, 8, 4, 128, 16, list(range(0, 190, 3))),
    (BF, 1, 8, 2, 128, 8, [100, 9, 64]),
    (HF, 2, 8, 2, 64, 256, [300, 65, 513]),
    (BF, 1, 8, 2, 136, 24, [100, 9]),
    (BF, 1, 4, 2, 192, 32, [100, 9, 65]),  # three of four blocks of columns
    (BF, 1, 2, 2, 64, 16, [i % 130 for i in range(600)]),  # more sequences than threads
]


@pytest.mark.parametrize("dtype,t,hq,hkv,d,bs,lens", OWN)
def test_own_tokens(dtype, t, hq, hkv, d, bs, lens):
    check(*problem(d + t, dtype, t, hq, hkv, d, bs, lens, spare=1))


SHARED = [  # dtype, T, Hq, Hkv, D, block size, prefix, lengths in all
    (BF, 1, 32, 8, 128, 16, 256, [257, 300, 400, 256, 0, 321]),
    (BF, 1, 8, 2, 128, 16, 48, [49, 64, 112]),  # a prefix shorter than a tile
    (HF, 5, 16, 16, 64, 32, 160, [165, 300, 0, 0]),
    (BF, 4, 8, 1, 80, 16, 1008, [1012] * 5 + [1500]),
    (HF, 1, 4, 4, 128, 16, 320, list(range(320, 520, 2))),  # 100 rows a key head
    (BF, 2, 6, 2, 256, 16, 96, [100, 101, 98]),
    (BF, 3, 4, 2, 64, 16, 128, [40, 129, 2, 130, 0, 131, 300]),  # some end inside the prefix
    (BF, 1, 8, 2, 128, 16, 2048, [2049]),  # a batch of one shares with nobody
    (HF, 2, 64, 1, 64, 64, 4096, [4100, 4098]),
    (BF, 1, 16, 2, 128, 128, 1024, [1024 + 7 * i for i in range(40)]),  # 320 rows a key head
    (BF, 8, 32, 4, 128, 64, 640, [648 + i for i in range(9)]),  # 576 rows a key head
    (BF, 1, 8, 2, 128, 8, 328, [330 + i for i in range(50)]),  # boxes of 8 rows
    (HF, 1, 16, 2, 64, 8, 1000, [1001 + i for i in range(40)]),
    (BF, 1, 8, 2, 96, 16, 272, [280, 300]),
    (BF, 1, 160, 160, 64, 16, 144, [145, 160]),  # more units than CTAs
    (BF, 300, 8, 2, 64, 16, 128, [500, 428]),  # many tokens each
]


@pytest.mark.parametrize("dtype,t,hq,hkv,d,bs,prefix,lens", SHARED)
def test_shared_prefix(dtype, t, hq, hkv, d, bs, prefix, lens):
    p = problem(d + t + 1, dtype, t, hq, hkv, d, bs, lens, prefix)
    check(*p, prefix)
    check(*p)  # the same batch without the word that its prefix is shared


def test_peaked_scores_scale_and_guarded_output():
    q, kc, vc, tables, lens = problem(3, BF, 2, 8, 2, 128, 16, [300, 70, 2], scale=3.0)
    out, check_guard = guarded_empty(q.shape, q.dtype)
    got = check(q, kc, vc, tables, lens, scale=0.5, out=out)
    assert got.data_ptr() == out.data_ptr()
    check_guard()


def test_strided_and_misaligned_queries():
    q, kc, vc, tables, lens = problem(4, BF, 3, 8, 2, 64, 16, [100, 33], 32)
    wide = torch.randn(2, 3, 12 * 64).to(BF).cuda()  # a fused projection: q, then k and v
    wide[..., :512] = q.cuda().flatten(2)
    rest = [t.cuda() for t in (kc, vc, tables, lens)]
    want = attention.paged_attention(q.cuda(), *rest, shared_prefix=32)
    views = [wide[..., :512].view(2, 3, 8, 64), q.cuda().transpose(1, 2).contiguous().transpose(1, 2),
             torch.cat([torch.zeros(1, dtype=BF), q.flatten()]).cuda()[1:].view(q.shape),  # 2 bytes off
             q.cuda().transpose(2, 3).contiguous().transpose(2, 3)]
    for view in views:
        assert bits_equal(attention.paged_attention(view, *rest, shared_prefix=32), want)
    tables_wide = torch.cat([rest[2], rest[2]], 1)[:, :tables.shape[1]]  # rows with a stride
    assert bits_equal(attention.paged_attention(q.cuda(), rest[0], rest[1], tables_wide, rest[3], shared_prefix=32), want)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("prefix", [0, 64])
def test_values_that_a_row_must_not_see(dtype, prefix):
    """NaN and infinities at positions that only later tokens (or longer sequences) see stay with those."""
    q, kc, vc, tables, lens = problem(5, dtype, 4, 8, 2, 64, 16, [64 + 70, 64 + 9], prefix)
    want = check(q, kc, vc, tables, lens, prefix)
    for b, n in enumerate(lens.tolist()):
        block, at = tables[b, (n - 2) // 16], (n - 2) % 16  # seen by tokens 2 and 3
        vc[block, at, 0, 3], kc[block, at, 1, 5] = float("inf"), float("nan")
    got = check(q, kc, vc, tables, lens, prefix)
    assert bits_equal(got[:, :2], want[:, :2])
    assert not got[:, 2:, :4, 3].isfinite().any() and got[:, 2:, 4:].isnan().all()


def test_rows_that_end_inside_a_shared_prefix_do_not_see_its_rest():
    q, kc, vc, tables, lens = problem(6, BF, 1, 8, 2, 128, 16, [300, 100, 290], 256)
    vc[tables[0, 10], 3] = float("nan")  # position 163
    got = check(q, kc, vc, tables, lens, 256)
    assert got[0].isnan().all() and got[1].isfinite().all()


def test_scores_that_are_infinite():
    q, kc, vc, tables, lens = problem(7, BF, 1, 2, 1, 64, 16, [40, 40, 40])
    q.fill_(1.0)
    kc[tables[0, 0], 5] = float("-inf")  # a score of -inf: no weight
    kc[tables[1, :3]] = float("-inf")  # every score: 0 / 0
    kc[tables[2, 1], 2] = float("inf")  # inf - inf
    got = check(q, kc, vc, tables, lens)
    assert got[0].isfinite().all() and got[1:].isnan().all()


def test_bad_blocks_read_as_zeros_and_lengths_are_clamped():
    q, kc, vc, tables, lens = problem(8, HF, 2, 4, 2, 64, 16, [100, 80, 50])
    tables[0, 2], tables[1, 1], tables[2, 0] = -1, kc.shape[0], 1 << 40
    kc.nan_to_num_()
    vc.nan_to_num_()
    check(q, kc, vc, tables, lens)
    check(q, kc, vc, tables, torch.tensor([1 << 40, -5, tables.shape[1] * 16 + 1]))
    tables[0, :2] = -7
    check(q, kc, vc, tables, lens, 32)
    empty = torch.empty(0, 16, 2, 64, dtype=HF)  # a cache of no blocks
    assert (attention.paged_attention(q.cuda(), empty.cuda(), empty.cuda(), tables.cuda(), lens.cuda()) == 0).all()
    none = attention.paged_attention(q[:0].cuda(), kc.cuda(), vc.cuda(), tables[:0].cuda(), lens[:0].cuda())
    assert none.shape == (0, 2, 4, 64)


@pytest.mark.parametrize("bs", [16, 24])  # a whole page as a box, and copies of 16 bytes
def test_offsets_beyond_32_bits(bs):
    """A cache of 2^31 + elements; the sequence's blocks are its last ones. The shared prefix's too."""
    hkv, d = 8, 128
    blocks = (1 << 31) // (hkv * d * bs) + 40
    caches = [torch.empty(blocks, bs, hkv, d, dtype=BF, device="cuda") for _ in range(2)]
    g = torch.Generator().manual_seed(9)
    small = [torch.randn(20, bs, hkv, d, generator=g).to(BF) for _ in range(2)]
    for c, s in zip(caches, small):
        c[-20:] = s.cuda()
    tables = torch.stack([torch.arange(10), torch.cat([torch.arange(4), torch.arange(10, 16)])])
    q, lens = torch.randn(2, 1, 16, d, generator=g).to(BF), torch.tensor([150, 145])
    for prefix in (0, 4 * bs):
        got = attention.paged_attention(q.cuda(), *caches, (tables + blocks - 20).cuda(), lens.cuda(), shared_prefix=prefix)
        assert_near(got, q, *small, tables, lens, prefix)


@pytest.mark.parametrize("bs", [16, 24])
@pytest.mark.parametrize("t,hq,hkv,d", [(1, 2, 2, 64), (17, 2, 1, 256), (9, 2, 1, 256), (1, 4, 1, 128)])
def test_the_largest_batch(t, hq, hkv, d, bs):
    """4096 sequences of up to 40 tokens: the lengths and tile counts of all lie in shared memory, whose limit the wide heads
    with many rows come nearest to."""
    g = torch.Generator(device="cuda").manual_seed(t)
    b, n = 4096, 48
    width = n // bs
    tables = torch.randperm(b * width, generator=g, device="cuda").view(b, width)
    caches = [torch.randn(b * width, bs, hkv, d, generator=g, device="cuda").to(BF) for _ in range(2)]
    lens = torch.randint(0, 41, (b,), generator=g, device="cuda")
    q = torch.randn(b, t, hq, d, generator=g, device="cuda").to(BF)
    got = attention.paged_attention(q, *caches, tables, lens)
    k, v = (c[tables].view(b, n, hkv, d).permute(0, 2, 1, 3).double() for c in caches)
    x = q.double().view(b, t, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, -1, d) @ k.transpose(2, 3) * d ** -0.5
    limit = (lens[:, None] - t + torch.arange(1, t + 1, device="cuda")).repeat_interleave(hq // hkv, 1)
    seen = torch.arange(n, device="cuda") < limit[:, None, :, None]
    p = torch.softmax(x.masked_fill(~seen, float("-inf")), -1).nan_to_num()

    def back(y):
        return y.view(b, hkv, t, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b, t, hq, d)

    want, size = back(p @ v), back(p @ v.abs())
    a = d ** -0.5 * q.double().abs().sum(-1).max() * k.abs().max()
    bound = 2.0 ** -8 * (want.abs() + size) + 2 * size * ((d / 16 + 20) * 2.0 ** -23 * a + 2.0 ** -18)
    assert ((got.double() - want).abs() <= bound + 1e-30).all()


def test_streams_repeats_and_graphs_that_share_a_pool():
    """The same bits in every call; two graphs captured into one pool replay in either order."""
    a = [t.cuda() for t in problem(10, BF, 1, 8, 2, 128, 16, [700, 64, 300], 64)]
    b = [t.cuda() for t in problem(11, BF, 2, 8, 2, 128, 16, [90, 164, 3000], 64)]
    want_a, want_b = (attention.paged_attention(*x, shared_prefix=64) for x in (a, b))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = attention.paged_attention(*b, shared_prefix=64)
    assert bits_equal(attention.paged_attention(*a, shared_prefix=64), want_a)
    torch.cuda.synchronize()
    assert bits_equal(again, want_b)
    pool = torch.cuda.graph_pool_handle()
    graphs, outs = [], []
    for x in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(attention.paged_attention(*x, shared_prefix=64))
        graphs.append(graph)
    for order in ((0, 1), (1, 0), (0, 0, 1)):
        for i in order:
            graphs[i].replay()
    torch.cuda.synchronize()
    assert bits_equal(outs[1], want_b)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert bits_equal(outs[0], want_a)
    # the lengths are read at replay: a graph serves growing sequences
    a[4].fill_(64)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert bits_equal(outs[0], attention.paged_attention(*a, shared_prefix=64))


def test_calls_one_upon_another():
    """Calls of different sizes back to back on one stream (which recycle each other's workspace while the one before still
    joins), with the queries and the cache rewritten by other kernels in between, and on two streams at once: every
    output has the bits of a call alone."""
    sizes = [(20, BF, 1, 8, 2, 128, 16, [300 + 37 * i for i in range(24)], 256), (21, HF, 3, 8, 4, 64, 16, [90, 164, 1200], 64),
             (22, BF, 1, 4, 4, 128, 16, [513] * 40, 512), (23, BF, 2, 16, 2, 128, 16, [5, 40, 900, 77], 0)]
    cases = [([t.cuda() for t in problem(*c)], c[8]) for c in sizes]
    wants = []
    for x, prefix in cases:
        wants.append(attention.paged_attention(*x, shared_prefix=prefix))
        torch.cuda.synchronize()
    got = []
    for _ in range(12):
        for x, prefix in cases:
            q, kc = x[0].clone(), x[1].clone()  # written just before, freed just after
            got.append(attention.paged_attention(q, kc, *x[2:], shared_prefix=prefix))
            kc.fill_(float("nan"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    beside = []
    for _ in range(12):
        for x, prefix in cases:
            got.append(attention.paged_attention(*x, shared_prefix=prefix))
            with torch.cuda.stream(side):
                beside.append(attention.paged_attention(*x, shared_prefix=prefix))
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert bits_equal(out, wants[i % 4]), i
    for i, out in enumerate(beside):
        assert bits_equal(out, wants[i % 4]), i


def test_no_wait_has_given_up():
    from ckb200 import _native

    assert _native.load("attention").ckb_attention_status(0) == 0


def test_a_drafted_decoding_step():
    """qkv -> norms, rotation and append -> attention behind a shared prefix -> logits -> softmax -> verification, eagerly
    and as one replayed graph, against the same chain in fp64 (the cache's own rounding taken from the GPU's)."""
    g = torch.Generator().manual_seed(12)
    b, t, hq, hkv, d, bs, prefix, vocab = 6, 4, 8, 2, 64, 16, 96, 1000
    lens = [prefix + n for n in (4, 30, 77, 5, 64, 19)]
    _, kc, vc, tables, lens = problem(13, BF, t, hq, hkv, d, bs, lens, prefix)
    ids = lens[:, None] - t + torch.arange(t)
    slots = torch.gather(tables, 1, ids // bs) * bs + ids % bs
    qkv = torch.randn(b, t, (hq + 2 * hkv) * d, generator=g).to(BF).cuda()
    qw, kw = ((1 + 0.1 * torch.randn(d, generator=g)).to(BF).cuda() for _ in range(2))
    cos, sin = (c.cuda() for c in orope.cos_sin_cache(10000.0, d, 512))
    proj = (torch.randn(hq * d, vocab, generator=g) / 8).cuda()
    drafts = torch.randint(0, vocab, (b, t - 1), generator=g).cuda()
    draft_probs = torch.softmax(2 * torch.randn(b, t - 1, vocab, generator=g), -1).cuda()
    u = torch.rand(b, t, generator=g).cuda()
    kc_d, vc_d, tables_d, lens_d, ids_d, slots_d = (x.cuda() for x in (kc, vc, tables, lens, ids, slots))

    def step():
        q, k, v = (x.unflatten(-1, (-1, d)) for x in qkv.split([hq * d, hkv * d, hkv * d], -1))
        q, _ = rope.qk_norm_rope_kv_cache(q, k, v, ids_d, qw, kw, cos, sin, kc_d, vc_d, slots_d, inplace=False, write_k=False)
        out = attention.paged_attention(q, kc_d, vc_d, tables_d, lens_d, shared_prefix=prefix)
        probs = softmax.softmax(out.flatten(2).float() @ proj)
        return q, out, probs, *verify.verify_drafts(probs, drafts, u, draft_probs)

    q, out, probs, tokens, accepted = (x.clone() for x in step())
    q_in, k_in, v_in = (x.unflatten(-1, (-1, d)).cpu() for x in qkv.split([hq * d, hkv * d, hkv * d], -1))
    wq, _ = serving.norm_rotate(q_in, qw.cpu(), cos.cpu()[ids], sin.cpu()[ids], 1e-6)
    wk, _ = serving.norm_rotate(k_in, kw.cpu(), cos.cpu()[ids], sin.cpu()[ids], 1e-6)
    assert ((q.cpu().double() - wq).abs() <= 2.0 ** -7 * wq.abs() + 1e-4).all()
    flat = kc_d.cpu().view(-1, hkv, d)[slots.flatten()].view(b, t, hkv, d)
    assert ((flat.double() - wk).abs() <= 2.0 ** -7 * wk.abs() + 1e-4).all()
    assert bits_equal(vc_d.cpu().view(-1, hkv, d)[slots.flatten()].view(b, t, hkv, d), v_in)
    assert_near(out, q.cpu(), kc_d.cpu(), vc_d.cpu(), tables, lens, prefix)
    want = serving.verify(probs.cpu(), drafts.cpu(), u.cpu(), draft_probs.cpu())
    assert torch.equal(tokens.cpu(), want[0]) and torch.equal(accepted.cpu(), want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    kc_d.copy_(kc)
    graph.replay()
    torch.cuda.synchronize()
    assert bits_equal(got[1], out) and torch.equal(got[3], tokens)


@pytest.mark.parametrize("d,bs", [(128, 16), (64, 8), (64, 24), (256, 16)])  # tcgen05 with boxes of 16 and 8 rows; copies
@pytest.mark.parametrize("before", [1, 40])  # within and beyond the first 32 sequences
def test_the_prefix_is_found_behind_padded_rows_and_short_sequences(d, bs, before):
    """The rows in front are padding or end inside the prefix, and what their tables hold behind their lengths is anything."""
    lens = [0] * (before - 1) + [bs + 1, 4 * bs + 5, 4 * bs, 4 * bs + 70]  # with two tokens each, 4 bs is one too short
    q, kc, vc, tables, lens = problem(24 + before, BF, 2, 4, 2, d, bs, lens, 4 * bs)
    want = check(q, kc, vc, tables, lens, 4 * bs)
    for i, n in enumerate(lens.tolist()):
        tables[i, -(-n // bs):] = torch.tensor([-1, 1 << 40, kc.shape[0]])[i % 3]
    assert bits_equal(check(q, kc, vc, tables, lens, 4 * bs), want)
    tables[:, :4] = tables[before, :4]  # nobody sees it all: the tables' first rows are not used for others either
    tables[0] = -1
    check(q, kc, vc, tables, lens.clamp_max(4 * bs), 4 * bs)


@pytest.mark.parametrize("bs", [16, 24])
@pytest.mark.parametrize("prefix,sink", [(0, 0), (0, 2000), (16320, 5), (16320, 8000)])
def test_many_small_weights_beside_a_large_one(prefix, sink, bs):
    """One position takes nearly all the weight and thousands have 2^-26 of it each, which is less than half of fp16's
    smallest step, but 0.00006 and more together: all that the output is made of where the large one's value is zero. Heads
    and sequences enough that a CTA meets many of the positions in one piece.
    The bound is assert_near's, with the small weights off by half of 2^-24 of a weight that is lifted by 2^15, or by 2^7
    where that is all that the shared work does: n 2^-32 of the largest |v|, not n 2^-25."""
    prefix, heads = prefix // bs * bs, 16
    n = prefix + 41 if prefix else 4000
    q, kc, vc, tables, lens = problem(25, HF, 1, heads, heads, 64, bs, [n] * (2 if prefix else 24), prefix)
    q.fill_(1.0)
    kc[kc.isfinite()] = 0.0
    vc[:] = vc.abs() + 0.5
    rows = tables[:, sink // bs] * bs + sink % bs
    kc.view(-1, heads, 64)[rows] = 2.25  # a score of 64 * 2.25 / 8 = 18: exp(-18) = 2^-25.97
    vc.view(-1, heads, 64)[rows] = 0.0
    got = attention.paged_attention(*(t.cuda() for t in (q, kc, vc, tables, lens)), shared_prefix=prefix).cpu().double()
    want, size = serving.attend(q, kc, vc, tables, lens, 64 ** -0.5, prefix)
    v = vc[vc.isfinite()].double().abs().max().item()
    bound = 2.0 ** -11 * (want.abs() + size) + 2 * size * ((64 / 16 + 20) * 2.0 ** -23 * 18 + 2.0 ** -18) + n * 2.0 ** -32 * v + 2.0 ** -25
    assert (want > 2.0 ** -15).all() and ((got - want).abs() <= bound).all(), ((got - want).abs() / bound).max().item()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("prefix", [0, 512])
@pytest.mark.parametrize("shift", [-3e5, 3e5, 1.5e6, -1.5e6])  # to either side of 2^20 in powers of 2
def test_scores_far_from_zero(shift, prefix, dtype):
    """All scores of a row share a large term; what fp32 leaves of their differences has to come out as finite weights that
    add up: with values of 1 the output is 1, but for half a step of the weights and of itself, 2^-18 of the sums and, where
    fp16 weights are not lifted, 2^-25 for each of the 612."""
    q, kc, vc, tables, lens = problem(26, dtype, 1, 2, 1, 64, 16, [512 + 100, 512 + 30], prefix)
    q = 0.5 * torch.randn(q.shape, generator=torch.Generator().manual_seed(27)).to(dtype)
    q[..., 0], seen = 1024.0, kc.isfinite()
    kc[..., 0] = torch.where(seen[..., 0], shift * 8 / 1024 / 64, kc[..., 0])  # scale 64 / 8: shift in all
    vc[vc.isfinite()] = 1.0
    got = attention.paged_attention(*(t.cuda() for t in (q, kc, vc, tables, lens)), scale=8.0, shared_prefix=prefix)
    assert ((got.cpu().double() - 1).abs() <= torch.finfo(dtype).eps + 2.0 ** -18 + 612 * 2.0 ** -25).all()


def test_inputs_that_the_kernel_just_before_wrote():
    """Lengths and tables moved on in place, and the cache written by qk_norm_rope_kv_cache, right before each call behind a
    shared prefix, with no synchronisation: the bits of the same steps with one after each. Steps of 3 tokens over 40 rounds,
    eagerly and as a replayed graph; the tables are turned between two sets of pages that hold different tokens."""
    b, t, hq, hkv, d, bs, prefix, rounds = 24, 3, 8, 2, 64, 16, 128, 40
    g = torch.Generator().manual_seed(28)
    start = [prefix + 3 + 5 * i for i in range(b)]
    q, kc, vc, tables, lens = problem(28, BF, t, hq, hkv, d, bs, start, prefix, spare=10)
    kc, vc = (torch.randn(2 * c.shape[0], *c.shape[1:], generator=g).to(BF) for c in (kc, vc))  # pages of the other set
    shift = torch.zeros_like(tables)
    shift[:, prefix // bs:] = kc.shape[0] // 2
    qkv = torch.randn(rounds, b, t, (hq + 2 * hkv) * d, generator=g).to(BF).cuda()
    cos, sin = (c.cuda() for c in orope.cos_sin_cache(10000.0, d, 1024))
    w = torch.ones(d, device="cuda")
    first = [x.cuda() for x in (kc, vc, tables, lens)]
    shift, step_ids = shift.cuda(), torch.arange(t, device="cuda") - t

    def run(sync, graph=None):
        state = [x.clone() for x in first]
        kc, vc, tables, lens = state
        sign, now, x = torch.ones((), dtype=torch.int64, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda"), None
        outs = []

        def step():
            ids = lens[:, None] + t + step_ids
            slots = torch.gather(tables + sign * shift, 1, ids // bs) * bs + ids % bs
            parts = qkv[now][0].split([hq * d, hkv * d, hkv * d], -1)
            q, k, v = (p.unflatten(-1, (-1, d)) for p in parts)
            now.add_(1)
            tables.add_(sign * shift)
            sign.neg_()
            lens.add_(t)
            q, _ = rope.qk_norm_rope_kv_cache(q, k, v, ids, w, w, cos, sin, kc, vc, slots, inplace=False, write_k=False)
            return attention.paged_attention(q, kc, vc, tables, lens, shared_prefix=prefix)

        if graph is not None:
            with torch.cuda.graph(graph):
                x = step()
        for _ in range(rounds):
            if graph is None:
                outs.append(step())
            else:
                graph.replay()
                outs.append(x.clone())
            if sync:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        return outs, state

    want, kept = run(True)
    for _ in range(3):
        got, state = run(False)
        assert all(bits_equal(x, y) for x, y in zip(got, want))
        assert all(torch.equal(x, y) for x, y in zip(state[2:], kept[2:]))
    got, _ = run(False, torch.cuda.CUDAGraph())
    assert all(bits_equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("t,heads,lens", [(1, 320, [129, 140]), (1, 150, [128 + i % 20 for i in range(130)])])
@pytest.mark.parametrize("prefix", [128, 112])
def test_short_prefixes_of_more_units_than_ctas(t, heads, lens, prefix):
    """A CTA has several units of one tile one after the other: of 2 rows, and of 130."""
    check(*problem(29, BF, t, heads, heads, 64, 16, lens, prefix), prefix)


@pytest.mark.parametrize("op", ["attention", "softmax", "topk"])
def test_reading_the_status_waits_for_every_stream(op):
    """torch's streams are non-blocking: a copy on the legacy stream does not wait for them, the status has to."""
    from ckb200 import _native

    status = getattr(_native.load(op), f"ckb_{op}_status")
    assert status(0) == 0  # a first call waits for everything anyway, while the library is loaded
    side, done = torch.cuda.Stream(), torch.cuda.Event()
    with torch.cuda.stream(side):
        torch.cuda._sleep(400_000_000)  # 0.2 s at 2 GHz
        done.record()
    assert not done.query()
    assert status(0) == 0
    assert done.query()


def test_check_passes_on_either_device_argument():
    p = [t.cuda() for t in problem(30, BF, 1, 4, 2, 64, 16, [100, 70], 32)]
    attention.paged_attention(*p, shared_prefix=32)
    attention.check()
    attention.check("cuda:0")


@pytest.mark.parametrize("bs", [16, 24])  # a TMA box for each page, and copies of 16 bytes
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t", [1, 5, 10, 20])  # 4, 20, 40 and 80 rows a key head: 1, 2 and 4 warps share the rows, or two row tiles
def test_own_tokens_in_every_form(t, d, bs):
    dtype = (BF, HF)[(t + d // 64) % 2]
    check(*problem(31 + t, dtype, t, 8, 2, d, bs, [300, t - 1, 9, 0, 64, 700]))


@pytest.mark.parametrize("bs", [24, 48, 7])  # no box fits a page
@pytest.mark.parametrize("d", [64, 120, 128, 200])
@pytest.mark.parametrize("dtype,t,group,count", [(BF, 2, 4, 20), (HF, 1, 1, 9), (HF, 1, 8, 8), (BF, 7, 4, 5)])  # 160, 9, 64, 140 rows
def test_shared_prefix_without_boxes(dtype, t, group, count, d, bs):
    prefix = {24: 168, 48: 336, 7: 133}[bs]
    lens = [prefix + t + 3 * i for i in range(count)] + [prefix - 3, 0, 10, prefix + t - 1]
    check(*problem(32 + d, dtype, t, 2 * group, 2, d, bs, lens, prefix), prefix)


@pytest.mark.parametrize("bs", [16, 24])
@pytest.mark.parametrize("group", [4, 8, 16])  # 16, 32 and 64 rows a key head
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("shared", [False, True])
def test_values_that_a_row_must_not_see_in_every_form(shared, d, group, bs):
    prefix = 4 * bs if shared else 0
    q, kc, vc, tables, lens = problem(33 + d, (BF, HF)[group // 8 % 2], 4, 2 * group, 2, d, bs, [prefix + 130, prefix + 9], prefix)
    check(q, kc, vc, tables, lens, prefix)
    for b, n in enumerate(lens.tolist()):
        block, at = tables[b, (n - 2) // bs], (n - 2) % bs  # seen by tokens 2 and 3
        vc[block, at, 0, 3], kc[block, at, 1, 5] = float("inf"), float("nan")
    # Tokens 0 and 1 by assert_near's bound, not by bits: the tile that holds the value is then summed one position after the
    # other, not 16 at a time, and two fp32 sums that are each within 2^-18 of the exact one may round to either neighbour.
    got = check(q, kc, vc, tables, lens, prefix)
    assert got[:, :2].isfinite().all()
    assert not got[:, 2:, :group, 3].isfinite().any() and got[:, 2:, group:].isnan().all()
