"""Plain 64-bit forms of the serving operators (test infrastructure only), on CPU tensors: the norm of query and key heads
with the rotation, paged attention behind a shared prefix, and the verification of drafted tokens."""

import torch


def norm_rotate(x, weight, cos, sin, eps):
    """(the normed and rotated heads of x [B, S, H, D], the magnitude |y_i cos_i| + |y_j sin_j| of each sum), in fp64;
    cos / sin [B, S, D]."""
    x, c, s = x.double(), cos.double()[:, :, None], sin.double()[:, :, None]
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()
    h = x.shape[-1] // 2
    lo, hi = y[..., :h], y[..., h:]
    out = torch.cat([lo * c[..., :h] - hi * s[..., :h], hi * c[..., h:] + lo * s[..., h:]], -1)
    size = torch.cat([(lo * c[..., :h]).abs() + (hi * s[..., :h]).abs(),
                      (hi * c[..., h:]).abs() + (lo * s[..., h:]).abs()], -1)
    return out, size


def attend(q, key_cache, value_cache, tables, lens, scale, shared_prefix=0):
    """(out, the weighted mean of |v|) [B, T, Hq, D] in fp64. Where all T tokens of a sequence see shared_prefix tokens,
    these come from the first such sequence's row of tables."""
    b, t, hq, d = q.shape
    block_size, hkv = key_cache.shape[1:3]
    out = torch.zeros(q.shape, dtype=torch.float64)
    size = torch.zeros(q.shape, dtype=torch.float64)
    shared = shared_prefix // block_size
    lengths = [max(0, min(int(n), tables.shape[1] * block_size)) for n in lens]
    sharing = [i for i in range(b) if lengths[i] - t + 1 >= shared_prefix]
    for i in range(b):
        ids = torch.cat([tables[sharing[0] if i in sharing else i, :shared], tables[i, shared:]])
        length = lengths[i]
        ids = ids[: -(-length // block_size)]
        fine = (ids >= 0) & (ids < key_cache.shape[0])
        at = ids.clamp(0, key_cache.shape[0] - 1)
        k = torch.where(fine[:, None, None, None], key_cache[at].double(), 0.0).flatten(0, 1)
        v = torch.where(fine[:, None, None, None], value_cache[at].double(), 0.0).flatten(0, 1)
        for j in range(t):
            n = length - t + j + 1
            if n <= 0:
                continue
            for h in range(hq):
                g = h // (hq // hkv)
                p = torch.softmax(k[:n, g] @ q[i, j, h].double() * scale, 0)
                out[i, j, h] = p @ v[:n, g]
                size[i, j, h] = p @ v[:n, g].abs()
    return out, size


def verify(target, tokens, uniforms, draft=None, counts=None):
    """(tokens [B, K + 1], accepted [B]) by the definition, one sequence and one column after the other. A probability that is
    NaN or negative, the target's or the draft's, counts as 0."""
    b, rows, vocab = target.shape
    k = rows - 1
    out = torch.full((b, rows), -1, dtype=torch.int64)
    accepted = torch.zeros(b, dtype=torch.int64)

    def clean(x):
        x = x.double()
        return torch.where(x > 0, x, 0.0)

    for i in range(b):
        n = k if counts is None else max(0, min(k, int(counts[i])))
        w, a = None, n
        for j in range(n):
            d = int(tokens[i, j])
            u = float(uniforms[i, j])
            inside = 0 <= d < vocab
            q = 1.0 if draft is None else float(clean(draft[i, j, d])) if inside else 0.0
            if inside and u * q < float(clean(target[i, j, d])):
                out[i, j] = d
                continue
            p = clean(target[i, j])
            if draft is None:
                w = p.clone()
                if inside:
                    w[d] = 0.0
            else:
                w = clean(p - clean(draft[i, j]))
            if not w.sum() > 0:
                w = p
            a = j
            break
        accepted[i] = a
        if w is None:
            w = clean(target[i, n])
        cum = w.cumsum(0)
        if cum[-1] > 0:
            over = torch.nonzero(cum > float(uniforms[i, k]) * cum[-1])
            out[i, a] = over[0, 0] if over.numel() else torch.nonzero(w)[-1, 0]
    return out, accepted
