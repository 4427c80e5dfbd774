"""The serving operators of one drafted-decoding step, as cases with sizes: the norm of queries and keys with their rotation
(and the append to the paged cache), attention over that cache with a prefix that the batch shares, and the check of drafted
tokens against the target's probabilities.

run() computes them in their plain form in torch, or, where `own` is true, by the framework's calls.
"""

import math
import os
import random
import sys

import torch

own = False

PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuda-kernels-optimized-for-rtx5090_b200")
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6
THETA = 10000.0
POSITIONS = 32768  # rows of the cos/sin cache


def _norm(name, batch, seq, q_heads, kv_heads, head_dim, dtype, append, angles="fp32", block_size=16, padding=0):
    return dict(name=name, op="norm_rope", batch=batch, seq=seq, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim,
                dtype=dtype, append=append, angles=angles, block_size=block_size, padding=padding)


def _attend(name, batch, tokens, prefix, own_min, own_max, q_heads, kv_heads, head_dim, dtype, block_size=16, empty=0):
    return dict(name=name, op="attend", batch=batch, tokens=tokens, prefix=prefix, own_min=own_min, own_max=own_max,
                q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, dtype=dtype, block_size=block_size, empty=empty)


def _verify(name, batch, drafts, vocab, dtype, with_probs=True, ragged=False, noise=1.0):
    return dict(name=name, op="verify", batch=batch, drafts=drafts, vocab=vocab, dtype=dtype, with_probs=with_probs,
                ragged=ragged, noise=noise)


def listed():
    return [
        # one decoding step of 64 sequences: latency
        _norm("norm_rope_append_64x1", 64, 1, 32, 8, 128, "bf16", True),
        # prompts of odd length, some tokens of them padding, few heads
        _norm("norm_rope_append_4x1021", 4, 1021, 12, 2, 64, "fp16", True, angles="bf16", padding=37),
        # the rotation's large configuration: 8 x 4096 tokens from a fused projection
        _norm("norm_rope_8x4096", 8, 4096, 32, 8, 128, "bf16", False),
        # one sequence of 8192 tokens, one new token, nothing shared: latency
        _attend("attend_1_own_8192", 1, 1, 0, 8192, 8192, 32, 8, 128, "bf16"),
        # an ordinary serving batch behind one system prompt
        _attend("attend_64_prefix_4096", 64, 1, 4096, 65, 1023, 32, 8, 128, "bf16"),
        # five drafted tokens each, a head for each key head, padded rows, odd lengths
        _attend("attend_18x5_prefix_1536", 18, 5, 1536, 5, 701, 16, 16, 64, "fp16", block_size=32, empty=2),
        # nothing shared and very unequal lengths, four tokens each
        _attend("attend_48x4_ragged", 48, 4, 0, 4, 16001, 32, 8, 128, "bf16"),
        # many answers to one long document
        _attend("attend_256_prefix_16384", 256, 1, 16384, 1, 511, 32, 8, 128, "bf16"),
        # one sequence with four drafted tokens: latency
        _verify("verify_1x4_151936", 1, 4, 151936, "fp32"),
        # drafts of five tokens, probabilities in 16 bits
        _verify("verify_64x5_128256", 64, 5, 128256, "bf16"),
        # drafts without probabilities (looked up in the text), some sequences with fewer, an odd vocabulary
        _verify("verify_16x3_looked_up_50001", 16, 3, 50001, "fp32", with_probs=False, ragged=True),
        # the largest serving batch
        _verify("verify_256x4_151936", 256, 4, 151936, "fp32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm_rope", "attend", "attend", "verify"])
    if op == "norm_rope":
        batch, append = _log(rng, 1, 64), rng.random() < 0.6
        seq = _log(rng, 1, 32768 // batch)
        kv = rng.choice([1, 2, 4, 8])
        heads = min(32, kv * rng.choice([1, 2, 4, 5, 7, 8]) // kv * kv)
        c = _norm("", batch, seq, heads, kv, rng.choice([64, 80, 96, 128]), rng.choice(["bf16", "bf16", "fp16"]), append,
                  angles=rng.choice(["fp32", "fp32", "bf16"]), block_size=rng.choice([16, 32, 64]),
                  padding=rng.randrange(0, batch * seq // 4 + 1) if append else 0)
    elif op == "attend":
        block, tokens = rng.choice([16, 16, 32, 64]), rng.choice([1, 1, 1, 2, 3, 5, 8])
        batch = _log(rng, 1, 256 // tokens)
        prefix = rng.choice([0, 1, 1]) * (_log(rng, 64, 16384) // block * block)
        own_max = _log(rng, tokens, max(tokens, min(16384, 262144 // batch)))
        kv = rng.choice([1, 2, 4, 8])
        c = _attend("", batch, tokens, prefix, rng.randint(tokens, own_max), own_max, kv * rng.choice([1, 2, 3, 4, 4]), kv,
                    rng.choice([64, 80, 128, 128]), rng.choice(["bf16", "bf16", "fp16"]), block_size=block,
                    empty=rng.randrange(0, batch // 4 + 1))
    else:
        probs = rng.random() < 0.7
        c = _verify("", _log(rng, 1, 256), rng.randint(1, 4) if probs else rng.randint(1, 8), _log(rng, 1000, 151936),
                    rng.choice(["fp32", "bf16"]), with_probs=probs, ragged=rng.random() < 0.5, noise=rng.choice([0.3, 1.0, 2.0]))
        if c["batch"] * (c["drafts"] + 1) > 1280:
            c["batch"] = 1280 // (c["drafts"] + 1)
    del c["name"]
    return c


def _lengths(case):
    """The own tokens (behind the prefix) of each sequence: spread evenly over the case's range, in a fixed mixed order."""
    n, lo, hi = case["batch"], case["own_min"], case["own_max"]
    own_len = [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]
    random.Random(n * 7919 + hi).shuffle(own_len)
    return own_len


def _sequences(case):
    """The tokens of each sequence in all; the last `empty` rows are padding of the batch."""
    return [0 if i >= case["batch"] - case["empty"] else case["prefix"] + l for i, l in enumerate(_lengths(case))]


def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "norm_rope":
        tokens = case["batch"] * case["seq"]
        heads = case["q_heads"] + case["kv_heads"] * (2 if case["append"] else 1)
        angles = min(tokens, POSITIONS) if case["append"] else case["seq"]
        moved = tokens * heads * case["head_dim"] * 2 * e + angles * 2 * case["head_dim"] * SIZE[case["angles"]] + tokens * 8 * (2 if case["append"] else 1)
        return {"bytes": moved, "flops": tokens * (case["q_heads"] + case["kv_heads"]) * case["head_dim"] * 8}
    if case["op"] == "attend":
        seqs, t = _sequences(case), case["tokens"]
        kept = sum(s - case["prefix"] for s in seqs if s) + (case["prefix"] if any(seqs) else 0)
        seen = sum(max(0, s - t + i + 1) for s in seqs for i in range(t))
        moved = kept * case["kv_heads"] * case["head_dim"] * 2 * e + 2 * case["batch"] * t * case["q_heads"] * case["head_dim"] * e
        return {"bytes": moved, "flops": 4 * case["q_heads"] * case["head_dim"] * seen}
    # The target's row at the place that the drawing reaches, and the draft's where a token was refused (about 3 of 10
    # drafted tokens are, at these distributions).
    rows = 1 + ((1 - 0.7 ** case["drafts"]) if case["with_probs"] else 0)
    return {"bytes": case["batch"] * (case["vocab"] * e * rows + 8 * (2 * case["drafts"] + 2)), "flops": case["batch"] * case["vocab"] * rows * 2}


def _angles(head_dim, dtype):
    inv = 1.0 / (THETA ** (torch.arange(0, head_dim, 2, device="cuda", dtype=torch.float64) / head_dim))
    a = torch.outer(torch.arange(POSITIONS, device="cuda", dtype=torch.float64), inv)
    a = torch.cat([a, a], -1)
    return a.cos().to(dtype), a.sin().to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = {"case": case}
    dtype = TYPES[case["dtype"]]
    if case["op"] == "norm_rope":
        b, n, hq, hkv, d = (case[k] for k in ("batch", "seq", "q_heads", "kv_heads", "head_dim"))
        qkv = randn(b, n, (hq + 2 * hkv) * d).to(dtype)  # what the fused projection of a layer gives
        s["q"], s["k"], s["v"] = (x.view(b, n, -1, d) for x in qkv.split([hq * d, hkv * d, hkv * d], dim=-1))
        s["qw"], s["kw"] = ((1 + 0.1 * randn(d)).to(dtype) for _ in range(2))
        s["cos"], s["sin"] = _angles(d, TYPES[case["angles"]])
        if not case["append"]:
            s["ids"] = torch.arange(n, device="cuda").repeat(b, 1)
            return s
        first = torch.randint(0, POSITIONS - n + 1, (b, 1), generator=g, device="cuda")
        s["ids"] = first + torch.arange(n, device="cuda")
        blocks = -(-b * n // case["block_size"]) + 8
        s["slots"] = torch.randperm(blocks * case["block_size"], generator=g, device="cuda")[: b * n].view(b, n)
        order = torch.randperm(b * n, generator=g, device="cuda")
        s["kept"] = order[case["padding"]:].sort().values  # the tokens that are not padding
        s["slots"].view(-1)[order[: case["padding"]]] = -1
        s["key_cache"] = randn(blocks, case["block_size"], hkv, d).to(dtype)
        s["value_cache"] = randn(blocks, case["block_size"], hkv, d).to(dtype)
        return s
    if case["op"] == "attend":
        b, t, hq, hkv, d, bs = (case[k] for k in ("batch", "tokens", "q_heads", "kv_heads", "head_dim", "block_size"))
        shared = case["prefix"] // bs
        own_blocks = -(-case["own_max"] // bs)
        blocks = shared + b * own_blocks + 1
        ids = torch.randperm(blocks, generator=g, device="cuda")  # a cache in use: no block beside its neighbour
        s["tables"] = torch.cat([ids[:shared].expand(b, shared), ids[shared:shared + b * own_blocks].view(b, own_blocks)], 1).contiguous()
        s["lens"] = torch.tensor(_sequences(case), device="cuda")
        s["q"] = (2 * randn(b, t, hq, d)).to(dtype)
        s["key_cache"] = torch.empty(blocks, bs, hkv, d, device="cuda", dtype=dtype).normal_(generator=g)
        s["value_cache"] = torch.empty(blocks, bs, hkv, d, device="cuda", dtype=dtype).normal_(generator=g)
        return s
    b, k, v = case["batch"], case["drafts"], case["vocab"]
    logits = 3 * randn(b, k + 1, v)
    s["target"] = torch.softmax(logits, -1).to(dtype)
    logits = logits[:, :k] + case["noise"] * randn(b, k, v)
    draft = torch.softmax(logits, -1)
    s["draft"] = draft.to(dtype) if case["with_probs"] else None
    if case["with_probs"]:  # drawn from the draft's probabilities
        race = draft.div_(torch.empty_like(draft).exponential_(generator=g))
        s["tokens"] = race.argmax(-1)
    else:
        s["tokens"] = draft.argmax(-1)
    s["uniforms"] = torch.rand(b, k + 1, generator=g, device="cuda")
    s["counts"] = torch.randint(0, k + 1, (b,), generator=g, device="cuda") if case["ragged"] else None
    return s


def _calls():
    if PACKAGE not in sys.path:
        sys.path.insert(0, PACKAGE)
    import ckb200

    return ckb200


def _run_own(s):
    op = s["case"]["op"]
    if op == "norm_rope" and s["case"]["append"]:
        q, _ = _calls().rope.qk_norm_rope_kv_cache(s["q"], s["k"], s["v"], s["ids"], s["qw"], s["kw"], s["cos"], s["sin"], s["key_cache"],
                                                   s["value_cache"], s["slots"], eps=EPS, inplace=False, write_k=False)
        return {"q": q, "key_cache": s["key_cache"], "value_cache": s["value_cache"]}
    if op == "norm_rope":
        q, k = _calls().rope.qk_norm_rope(s["q"], s["k"], s["ids"], s["qw"], s["kw"], s["cos"], s["sin"], eps=EPS)
        return {"q": q, "k": k}
    if op == "attend":
        return {"out": _calls().attention.paged_attention(s["q"], s["key_cache"], s["value_cache"], s["tables"], s["lens"],
                                                          shared_prefix=s["case"]["prefix"])}
    tokens, accepted = _calls().verify.verify_drafts(s["target"], s["tokens"], s["uniforms"], s["draft"], s["counts"])
    return {"tokens": tokens, "accepted": accepted}


def _normed_and_turned(x, w, cos, sin):
    x = x.float()
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
    lo, hi = y.chunk(2, -1)
    return y * cos + torch.cat([-hi, lo], -1) * sin


def _norm_rope(s):
    dtype = s["q"].dtype
    cos, sin = (s[n][s["ids"]].float().unsqueeze(2) for n in ("cos", "sin"))
    q = _normed_and_turned(s["q"], s["qw"], cos, sin).to(dtype)
    k = _normed_and_turned(s["k"], s["kw"], cos, sin).to(dtype)
    if not s["case"]["append"]:
        return {"q": q, "k": k}
    rows = s["slots"].view(-1)[s["kept"]]
    for cache, new in (("key_cache", k), ("value_cache", s["v"])):
        s[cache].view(-1, *new.shape[2:])[rows] = new.reshape(-1, *new.shape[2:])[s["kept"]]
    return {"q": q, "key_cache": s["key_cache"], "value_cache": s["value_cache"]}


def _attend_plain(s):
    """The shared prefix's scores for the whole batch in one product, the own tokens' for each sequence, one softmax."""
    q = s["q"].float()
    b, t, hq, d = q.shape
    bs, hkv = s["key_cache"].shape[1:3]
    g, prefix = hq // hkv, s["case"]["prefix"]
    shared, rest = s["tables"][0, : prefix // bs], s["tables"][:, prefix // bs:]
    ks, vs = (s[n][shared].reshape(prefix, hkv, d).permute(1, 0, 2).float() for n in ("key_cache", "value_cache"))  # [hkv, prefix, d]
    ko, vo = (s[n][rest].reshape(b, -1, hkv, d).permute(0, 2, 1, 3).float() for n in ("key_cache", "value_cache"))  # [b, hkv, own, d]
    qh = q.view(b, t, hkv, g, d).permute(2, 0, 1, 3, 4)  # [hkv, b, t, g, d]
    first = torch.matmul(qh.reshape(hkv, -1, d), ks.transpose(1, 2)).view(hkv, b, t * g, prefix)
    then = torch.matmul(qh.transpose(0, 1).reshape(b, hkv, t * g, d), ko.transpose(2, 3)).transpose(0, 1)
    scores = torch.cat([first, then], -1).view(hkv, b, t, g, -1) * d ** -0.5
    limit = s["lens"][:, None] - t + torch.arange(1, t + 1, device=q.device)  # [b, t]: the positions that a query sees
    seen = torch.arange(scores.shape[-1], device=q.device) < limit[..., None]
    scores = scores.masked_fill(~seen[None, :, :, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    p = p.view(hkv, b, t * g, -1)
    out = torch.matmul(p[..., :prefix].reshape(hkv, b * t * g, prefix), vs).view(hkv, b, t, g, d)
    out = out + torch.matmul(p[..., prefix:].transpose(0, 1), vo).view(b, hkv, t, g, d).transpose(0, 1)
    return {"out": out.permute(1, 2, 0, 3, 4).reshape(b, t, hq, d).to(s["q"].dtype)}


def _verify_plain(s):
    """In 64 bits: a drawn number beside a border of the sums decides a whole number."""
    p, tokens, u = s["target"], s["tokens"], s["uniforms"].double()
    b, k = tokens.shape
    n = torch.full((b,), k, device=p.device) if s["counts"] is None else s["counts"]
    at = torch.gather(p[:, :k], 2, tokens[..., None])[..., 0].double()
    drafted = 1.0 if s["draft"] is None else torch.gather(s["draft"], 2, tokens[..., None])[..., 0].double()
    fine = (u[:, :k] * drafted < at) & (torch.arange(k, device=p.device) < n[:, None])
    accepted = fine.long().cumprod(1).sum(1)
    row = p[torch.arange(b, device=p.device), accepted].double()
    refused = accepted.clamp_max(k - 1)
    token = tokens[torch.arange(b, device=p.device), refused]
    if s["draft"] is None:
        less = row.scatter(1, token[:, None], 0.0)
    else:
        less = (row - s["draft"][torch.arange(b, device=p.device), refused].double()).clamp_min(0)
    less = torch.where((less.sum(1, keepdim=True) > 0), less, row)
    w = torch.where((accepted < n)[:, None], less, row)
    sums = w.cumsum(1)
    drawn = (sums <= u[:, k:] * sums[:, -1:]).sum(1)
    place = torch.arange(k + 1, device=p.device)
    out = torch.where(place < accepted[:, None], torch.cat([tokens, tokens[:, :1]], 1), -1)
    out = torch.where(place == accepted[:, None], drawn[:, None], out)
    return {"tokens": out, "accepted": accepted}


def run(state):
    if own:
        return _run_own(state)
    return {"norm_rope": _norm_rope, "attend": _attend_plain, "verify": _verify_plain}[state["case"]["op"]](state)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm_rope":
        h = case["head_dim"] // 2

        def turned(x, w):
            x = x.double()
            y = w.double() * x / (x.pow(2).sum(-1, keepdim=True) / (2 * h) + EPS).sqrt()
            c, z = s["cos"].double()[s["ids"]][:, :, None], s["sin"].double()[s["ids"]][:, :, None]
            out = torch.empty_like(y)
            out[..., :h] = y[..., :h] * c[..., :h] - y[..., h:] * z[..., :h]
            out[..., h:] = y[..., h:] * c[..., h:] + y[..., :h] * z[..., h:]
            return out

        q, k = turned(s["q"], s["qw"]), turned(s["k"], s["kw"])
        if not case["append"]:
            return {"q": q, "k": k}
        caches = {}
        keep = s["slots"] >= 0
        for name, new in (("key_cache", k), ("value_cache", s["v"].double())):
            flat = s[name].double().flatten(0, 1)
            flat[s["slots"][keep]] = new[keep]
            caches[name] = flat.view(s[name].shape)
        return {"q": q, **caches}
    if case["op"] == "attend":
        t, bs, group = case["tokens"], case["block_size"], case["q_heads"] // case["kv_heads"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for b, length in enumerate(_sequences(case)):
            for i in range(t):
                seen = length - t + i + 1
                if seen <= 0:
                    continue
                if i == 0 or length - t <= 0:
                    blocks = s["tables"][b, : -(-length // bs)]
                    keys, values = (s[n][blocks].flatten(0, 1).double().repeat_interleave(group, 1) if group > 1 else s[n][blocks].flatten(0, 1).double()
                                    for n in ("key_cache", "value_cache"))
                z = torch.einsum("hd,lhd->hl", s["q"][b, i].double(), keys[:seen]) / math.sqrt(case["head_dim"])
                out[b, i] = torch.einsum("hl,lhd->hd", torch.softmax(z, 1), values[:seen])
        return {"out": out}
    tokens, accepted = [], []
    drafts, u = s["tokens"].tolist(), s["uniforms"].double().tolist()
    counts = [case["drafts"]] * case["batch"] if s["counts"] is None else s["counts"].tolist()
    for b in range(case["batch"]):
        line, weights = [], None
        for i in range(counts[b]):
            p, d = s["target"][b, i].double(), drafts[b][i]
            q = torch.zeros_like(p).index_fill_(0, torch.tensor([d], device="cuda"), 1.0) if s["draft"] is None else s["draft"][b, i].double()
            if u[b][i] * q[d].item() < p[d].item():
                line.append(d)
                continue
            weights = torch.relu(p - q)
            weights = weights if weights.sum() > 0 else p
            break
        accepted.append(len(line))
        weights = s["target"][b, counts[b]].double() if weights is None else weights
        cum = weights.cumsum(0)
        line.append(int(torch.searchsorted(cum, cum[-1:] * u[b][-1], right=True)))
        tokens.append(line + [-1] * (case["drafts"] + 1 - len(line)))
    return {"tokens": torch.tensor(tokens, device="cuda"), "accepted": torch.tensor(accepted, device="cuda")}
