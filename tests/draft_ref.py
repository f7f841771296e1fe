"""Plain 64-bit forms of the operators on drafted tokens, one sequence and one row at a time."""
import math

import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def trees(gen, batch, rows, chain=False):
    """int32 [batch, rows]: a root, then every row under one before it (a chain: under the one before it)."""
    p = torch.full((batch, rows), -1, dtype=torch.int32)
    for b in range(batch):
        for j in range(1, rows):
            p[b, j] = j - 1 if chain else int(torch.randint(0, j, (1,), generator=gen))
    return p


def tree(parents, context, drafted):
    """positions and, as truth values, who sees whom."""
    batch, rows = parents.shape
    pos, sees = torch.full((batch, rows), -1, dtype=torch.int32), torch.zeros((batch, rows, rows), dtype=torch.bool)
    for b in range(batch):
        for i in range(int(drafted[b])):
            path, j = [i], i
            while -1 < int(parents[b, j]) < j:
                j = int(parents[b, j])
                path.append(j)
            if int(parents[b, j]) != -1:
                continue  # the path ends at a parent that is none
            pos[b, i] = int(context[b]) + len(path) - 1
            sees[b, i, path] = True
    return pos, sees


def words(sees):
    batch, rows, _ = sees.shape
    out = torch.zeros((batch, rows, -(-rows // 64)), dtype=torch.int64)
    for j in range(rows):
        bit = 1 << (j % 64)
        out[:, :, j // 64] |= torch.where(sees[:, :, j], bit - (1 << 64) if j % 64 == 63 else bit, 0)
    return out


def rotate(x, positions, inv_freq, factor, interleaved, suffix, inverse=False):
    """x [rows, heads, head_dim] as f64; rows of negative position stay."""
    x = x.double().clone()
    half = inv_freq.numel()
    start = x.shape[2] - 2 * half if suffix else 0
    for r in range(x.shape[0]):
        if int(positions[r]) < 0:
            continue
        for p in range(half):
            i, j = (start + 2 * p, start + 2 * p + 1) if interleaved else (start + p, start + half + p)
            t = int(positions[r]) * float(inv_freq[p])
            c, s = math.cos(t) * factor, (-1 if inverse else 1) * math.sin(t) * factor
            re, im = x[r, :, i].clone(), x[r, :, j].clone()
            x[r, :, i], x[r, :, j] = re * c - im * s, im * c + re * s
    return x


def cache_row(blocks, page, at):
    return int(blocks[at // page]), at % page


def gathered(pages, blocks, n):
    """The first n positions of a sequence: [n, heads, head_dim] as f64."""
    page = pages.shape[1]
    rows = blocks.long()[torch.arange(n, device=blocks.device) // page] * page + torch.arange(n, device=blocks.device) % page
    return pages.reshape(-1, *pages.shape[2:])[rows].double()


def attention(q, k_pages, v_pages, blocks, context, sees, drafted, scale):
    """(out, bound of its error by arithmetic), [batch, rows, heads, head_dim] f64; everything on one device.

    The bound: the result is rounded once, its weights once each (half a step of the type, of a weight below the type's normal range half
    its smallest step); a score is a sum of head_dim products in f32 and off by as much as (head_dim + 4) half steps of their absolute sum, which moves a
    weight by that much, in numerator and denominator."""
    batch, rows, heads, dim = q.shape
    kv, u = k_pages.shape[2], half_step(q.dtype)
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    out, bound = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b in range(batch):
        n, c = int(drafted[b]), int(context[b])
        if n == 0:
            continue
        k, v = gathered(k_pages, blocks[b], c + n), gathered(v_pages, blocks[b], c + n)
        seen = torch.ones((n, c + n), dtype=torch.bool, device=q.device)
        seen[:, c:] = sees[b, :n, :n].to(q.device)
        for h in range(heads):
            x, kh, vh = q[b, :n, h].double(), k[:, h // (heads // kv)], v[:, h // (heads // kv)]
            for i in range(n):
                at = seen[i].nonzero().squeeze(1)
                if at.numel() == 0:
                    continue
                s = kh[at] @ x[i] * scale
                w = torch.exp(s - s.max())
                out[b, i, h] = (w @ vh[at]) / w.sum()
                mean = (w @ vh[at].abs()) / w.sum()
                slack = 2 * (dim + 4) * 2.0 ** -24 * float((kh[at].abs() @ x[i].abs()).max()) * scale
                bound[b, i, h] = u * (out[b, i, h].abs() + mean * (1 + u)) + slack * mean + at.numel() * tiny * vh[at].abs().max() / w.sum() + (2.0 ** -24 if q.dtype == torch.float16 else 0.0)
    return out, bound


def verify(logits, draft, tokens, parents, accept_u, sample_u, temperature, drafted):
    """path, accepted, token of every sequence, by the definition; None in the place of a token whose random number lies within 1e-9 of a border."""
    batch, rows, vocab = logits.shape
    result = []
    for b in range(batch):
        n, heat = int(drafted[b]), float(temperature[b])
        if n == 0:
            result.append(([], 0, -1))
            continue

        def chances(x, i):
            x = x[b, i].double()
            if bool(torch.isnan(x).any()) or not math.isfinite(float(x.max())):
                return None
            if heat == 0:
                p = torch.zeros_like(x)
                p[int((x == x.max()).nonzero()[0])] = 1.0
                return p
            return torch.softmax((x - x.max()) / heat, 0)

        node, path, token = 0, [0], None
        while True:
            children = [j for j in range(node + 1, n) if int(parents[b, j]) == node]
            p = chances(logits, node)
            q = chances(draft, node) if draft is not None and children and heat != 0 else None
            if p is None or (draft is not None and children and heat != 0 and q is None):
                token = -1
                break
            kept = None
            for j in children:
                t = int(tokens[b, j])
                if not 0 <= t < vocab:
                    continue
                one = torch.zeros_like(p)
                one[t] = 1.0
                if float(accept_u[b, j]) * (float(q[t]) if q is not None else 1.0) < float(p[t]):
                    kept = j
                    break
                less = (p - q).clamp(min=0) if q is not None else p * (1 - one)
                if float(less.sum()) > 0:
                    p = less / less.sum()
            if kept is None:
                break
            node = kept
            path.append(kept)
        if token is None:
            sums = torch.cumsum(p, 0)
            target = float(sample_u[b]) * float(sums[-1])
            over = (sums > target).nonzero()
            token = int(over[0]) if over.numel() else int((p > 0).nonzero()[-1])
            near = (sums - target).abs()[p > 0].min()
            if float(near) < 1e-9 and heat != 0:
                token = None
        result.append((path, len(path), token))
    return result
