"""Speculative decoding over a paged cache: what is measured of the operators that a drafted tree of tokens passes through.

One step of a decoder that drafts tokens: the tree's positions and mask (``draft_tree``), for every layer the rotation of its
queries and keys with the keys and values written to the cache (``rope_rows``, ``rope_append``) and the attention over the
cache (``tree_attention``), then the choice of the path that is kept (``verify_draft``) and the cache rows that go with it
(``cache_keep_path``).

``own`` False: plain torch in 32 bits, in 64 where 32 lose what matters (angles of far positions; sums over a vocabulary that
a random number is compared with).  ``own`` True: the framework's operators.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one conversation with a tree of eight drafted tokens
        {"name": "tree_b1_n8", "op": "tree", "batch": 1, "rows": 8, "width": 3},
        # a full batch of wide trees, some of them cut short
        {"name": "tree_b256_n255", "op": "tree", "batch": 256, "rows": 255, "width": 8},
        # the single token of a 1B-class decoder's step (24 heads of 64 over 8), f32 rows as its projections give them
        {"name": "rope_f32_m1", "op": "rope", "batch": 1, "rows": 1, "heads": 24, "kv_heads": 8, "head_dim": 64, "rotary": 64, "interleaved": False, "suffix": False, "yarn": False, "inverse": False, "dtype": "f32", "append": False, "page": 16, "far": 4096},
        # 4096 rows of a scaled long-context model, written to the cache as they are rotated
        {"name": "rope_append_bf16_m4096", "op": "rope", "batch": 64, "rows": 64, "heads": 32, "kv_heads": 8, "head_dim": 128, "rotary": 128, "interleaved": False, "suffix": False, "yarn": True, "inverse": False, "dtype": "bf16", "append": True, "page": 32, "far": 131072},
        # one token of a 1B-class decoder, short context: latency
        {"name": "attn_f16_b1_n1_517", "op": "attn", "batch": 1, "rows": 1, "heads": 24, "kv_heads": 8, "head_dim": 64, "page": 16, "context": 517, "ragged": False, "tree": False, "dtype": "f16"},
        # sixteen conversations of unequal length, trees of up to 13 tokens
        {"name": "attn_bf16_b16_n13_8191", "op": "attn", "batch": 16, "rows": 13, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 32, "context": 8191, "ragged": True, "tree": True, "dtype": "bf16"},
        # a large tree over one long document
        {"name": "attn_bf16_b1_n64_131072", "op": "attn", "batch": 1, "rows": 64, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "context": 131072, "ragged": False, "tree": True, "dtype": "bf16"},
        # plain decode of a large batch
        {"name": "attn_f16_b64_n1_16384", "op": "attn", "batch": 64, "rows": 1, "heads": 40, "kv_heads": 8, "head_dim": 128, "page": 64, "context": 16384, "ragged": True, "tree": False, "dtype": "f16"},
        # one conversation, the children of each node chosen, not drawn
        {"name": "verify_f32_b1_n8", "op": "verify", "batch": 1, "rows": 8, "width": 3, "vocab": 32768, "drawn": False, "greedy": False, "dtype": "f32"},
        # a full batch with the draft's own distributions
        {"name": "verify_bf16_b64_n13", "op": "verify", "batch": 64, "rows": 13, "width": 2, "vocab": 128003, "drawn": True, "greedy": False, "dtype": "bf16"},
        # one layer's cache of one conversation
        {"name": "keep_f16_b1_n8", "op": "keep", "batch": 1, "rows": 8, "layers": 1, "kv_heads": 8, "head_dim": 64, "page": 16, "dtype": "f16"},
        # all layers' caches of a full batch
        {"name": "keep_bf16_b64_n64", "op": "keep", "batch": 64, "rows": 64, "layers": 24, "kv_heads": 8, "head_dim": 128, "page": 32, "dtype": "bf16"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["tree", "rope", "rope", "attn", "attn", "attn", "attn", "verify", "verify", "keep"])
    kv = rng.choice([1, 2, 4, 8])
    group, head_dim, page = rng.choice([1, 2, 3, 4, 5, 8, 16]), rng.choice([32, 64, 80, 96, 128, 128, 192, 256]), rng.choice([8, 16, 32, 64, 128])
    half = rng.choice(["f16", "bf16"])
    if op == "tree":
        return {"op": op, "batch": _log(rng, 1, 256), "rows": _log(rng, 1, 255), "width": rng.randint(1, 8)}
    if op == "rope":
        batch = _log(rng, 1, 64)
        append = rng.random() < 0.5
        rows = _log(rng, 1, max(2, 4096 * 40 * 128 // (batch * kv * (group + 2) * head_dim)))
        return {"op": op, "batch": batch, "rows": min(rows, 2048), "heads": kv * group, "kv_heads": kv, "head_dim": head_dim, "rotary": rng.choice([head_dim, head_dim, head_dim // 2]), "interleaved": rng.random() < 0.5,
                "suffix": rng.random() < 0.3, "yarn": rng.random() < 0.5, "inverse": not append and rng.random() < 0.3, "dtype": half if append else rng.choice(["f32", "f16", "bf16"]), "append": append, "page": page, "far": _log(rng, 2048, 1 << 20)}
    if op == "attn":
        batch, rows = _log(rng, 1, 64), _log(rng, 1, 128)
        # the cache of all sequences and the products stay below the largest listed case
        most = min((1 << 30) // (batch * kv * head_dim * 2), (1 << 34) // (batch * rows * kv * group * head_dim))
        return {"op": op, "batch": batch, "rows": rows, "heads": kv * group, "kv_heads": kv, "head_dim": head_dim, "page": page, "context": _log(rng, 17, max(64, min(131072, most))), "ragged": rng.random() < 0.7,
                "tree": rng.random() < 0.7, "dtype": half}
    if op == "verify":
        batch, rows = _log(rng, 1, 64), _log(rng, 1, 24)
        vocab = _log(rng, 1000, max(2000, min(200000, 64 * 13 * 128003 // (batch * rows))))
        return {"op": op, "batch": batch, "rows": rows, "width": rng.randint(1, 4), "vocab": vocab, "drawn": rng.random() < 0.5, "greedy": rng.random() < 0.2, "dtype": rng.choice(["f32", half])}
    return {"op": op, "batch": _log(rng, 1, 64), "rows": _log(rng, 2, 64), "layers": _log(rng, 1, 24), "kv_heads": kv, "head_dim": rng.choice([64, 96, 128]), "page": page, "dtype": half}


# ---- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(gen, low, high, shape):
    """Whole numbers of [low, high]."""
    return torch.randint(low, high + 1, shape, generator=gen, device="cuda", dtype=torch.int32)


def _randn(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(_DTYPES[dtype])


def _parents(gen, batch, rows, width):
    """Trees whose row 0 is the newest known token: row j hangs under one of the `width` rows before it that can have it, level by level."""
    j = torch.arange(rows, device="cuda", dtype=torch.int32)
    low = torch.clamp((j - 1) // width - (j % 2), min=0)
    p = low + (torch.rand((batch, rows), generator=gen, device="cuda") * (torch.clamp(j - low, min=1, max=2))).to(torch.int32)
    p = torch.minimum(p, torch.clamp(j - 1, min=0))
    p[:, 0] = -1
    return p


def _drafted(gen, batch, rows):
    """Rows of each sequence: all of them for most, fewer for some."""
    n = _ints(gen, max(1, rows // 2), rows, (batch,))
    n[0::2] = rows
    return n


def _blocks(gen, batch, pages):
    return torch.randperm(batch * pages, generator=gen, device="cuda").to(torch.int32).reshape(batch, pages)


def _inv_freq(rotary, base, yarn):
    """Angle per position of each pair; with `yarn` slow pairs turn 8 times slower, fast ones as before, a ramp between them."""
    half = rotary // 2
    f = base ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    if yarn:
        turns = 32768 * f / (2 * math.pi)  # of a pair over the context that it was trained on
        keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
        f = f * keep + f / 8 * (1 - keep)
    return f.to(torch.float32)


def prepare(case, seed):
    gen, op, b, n = _gen(seed), case["op"], case["batch"], case["rows"]
    s = {"case": case}
    if op == "tree":
        s["parents"], s["context"], s["drafted"] = _parents(gen, b, n, case["width"]), _ints(gen, 0, 32768, (b,)), _drafted(gen, b, n)
    elif op == "rope":
        kv, d = case["kv_heads"], case["head_dim"]
        s["q"], s["k"] = _randn(gen, (b * n, case["heads"], d), case["dtype"]), _randn(gen, (b * n, kv, d), case["dtype"])
        s["inv_freq"], s["factor"] = _inv_freq(case["rotary"], 500000.0, case["yarn"]), 1.0 + 0.1 * math.log(8) if case["yarn"] else 1.0
        s["context"] = _ints(gen, 0, case["far"] if not case["append"] else 3 * case["page"], (b,))
        s["positions"] = (_ints(gen, 0, case["far"], (b, 1)) + torch.arange(n, device="cuda", dtype=torch.int32)).reshape(-1)
        if case["append"]:
            pages = 4 + -(-n // case["page"])
            s["v"] = _randn(gen, (b * n, kv, d), case["dtype"])
            s["k_pages"], s["v_pages"] = _randn(gen, (b * pages, case["page"], kv, d), case["dtype"]), _randn(gen, (b * pages, case["page"], kv, d), case["dtype"])
            s["blocks"], s["drafted"] = _blocks(gen, b, pages), _drafted(gen, b, n)
    elif op == "attn":
        kv, d = case["kv_heads"], case["head_dim"]
        pages = -(-(case["context"] + n) // case["page"])
        s["q"] = _randn(gen, (b, n, case["heads"], d), case["dtype"])
        s["k_pages"], s["v_pages"] = _randn(gen, (b * pages, case["page"], kv, d), case["dtype"]), _randn(gen, (b * pages, case["page"], kv, d), case["dtype"])
        s["blocks"] = _blocks(gen, b, pages)
        s["context"] = _ints(gen, case["context"] // 4, case["context"], (b,)) if case["ragged"] else torch.full((b,), case["context"], device="cuda", dtype=torch.int32)
        s["drafted"], s["mask"] = None, None
        if case["tree"]:
            s["drafted"] = _drafted(gen, b, n)
            s["mask"] = _plain_tree(_parents(gen, b, n, 3), s["context"], s["drafted"])["mask"]
    elif op == "verify":
        v = case["vocab"]
        common = -1.1 * torch.log(1.0 + torch.randperm(v, generator=gen, device="cuda").to(torch.float32))  # frequent and rare tokens
        logits = torch.randn((b, n, v), generator=gen, device="cuda").mul_(2.0).add_(common)
        s["parents"], s["drafted"] = _parents(gen, b, n, case["width"]), _drafted(gen, b, n)
        near = torch.randn((b, n, v), generator=gen, device="cuda").mul_(0.5).add_(logits)  # what the draft makes of it
        s["temperature"] = torch.zeros(b, device="cuda") if case["greedy"] else torch.rand(b, generator=gen, device="cuda") * 0.6 + 0.6
        s["logits"] = logits.to(_DTYPES[case["dtype"]])
        s["draft_logits"] = near.to(_DTYPES[case["dtype"]]) if case["drawn"] else None
        # each row's token is drawn at its parent's place: from the draft's distribution there, or one of its likely tokens
        up = s["parents"].clamp(min=0).long().unsqueeze(2).expand(b, n, v)
        near = torch.gather(near, 1, up)
        if not case["greedy"]:
            near.div_(s["temperature"].reshape(b, 1, 1))
        gumbel = torch.rand((b, n, v), generator=gen, device="cuda").clamp_(min=1e-20).log_().neg_().log_()
        s["tokens"] = (near - gumbel * (1.0 if case["drawn"] else 0.5)).argmax(2).to(torch.int32)
        s["accept_u"], s["sample_u"] = torch.rand((b, n), generator=gen, device="cuda"), torch.rand(b, generator=gen, device="cuda")
    else:
        kv, d, pages = case["kv_heads"], case["head_dim"], 4 + -(-n // case["page"])
        shape = (case["layers"], b * pages, case["page"], kv, d)
        s["k_pages"], s["v_pages"] = _randn(gen, shape, case["dtype"]), _randn(gen, shape, case["dtype"])
        s["blocks"], s["context"] = _blocks(gen, b, pages), _ints(gen, 0, 3 * case["page"], (b,))
        # row 0 stays, the kept rows behind it come from further back than any row moves to, as in a tree listed level by level
        most = max(1, min(6, n // 2))
        s["accepted"] = _ints(gen, 1, most, (b,))
        pick = torch.rand((b, n - most), generator=gen, device="cuda").argsort(1)[:, :most - 1].sort(1).values.to(torch.int32) + most
        path = torch.full((b, n), -1, device="cuda", dtype=torch.int32)
        path[:, 0] = 0
        path[:, 1:most] = pick
        s["path"] = torch.where(torch.arange(n, device="cuda") < s["accepted"].unsqueeze(1), path, -1)
    return s


# ---- plain forms
def _plain_tree(parents, context, drafted):
    """Row i sees itself and the rows above it; its position is the sequence's length and how many rows are above it."""
    b, n = parents.shape
    at = torch.arange(n, device="cuda")
    reach = torch.zeros((b, n, n), device="cuda").scatter_(2, parents.clamp(min=0).long().unsqueeze(2), (parents >= 0).float().unsqueeze(2))
    reach[:, at, at] = 1.0
    for _ in range(n.bit_length()):  # twice as many levels up each time
        reach = torch.matmul(reach, reach).clamp(max=1.0)
    sees = reach > 0
    real = at < drafted.unsqueeze(1)
    sees &= real.unsqueeze(2)
    positions = torch.where(real, context.unsqueeze(1) + sees.sum(2) - 1, -1).to(torch.int32)
    words = -(-n // 64)
    bits = torch.zeros((b, n, words * 64), dtype=torch.int64, device="cuda")
    bits[:, :, :n] = sees
    return {"positions": positions, "mask": (bits.reshape(b, n, words, 64) << torch.arange(64, device="cuda")).sum(3)}


def _rotate(x, positions, inv_freq, factor, case):
    """f32 rows [rows, heads, head_dim]; the angles and their sines in 64 bits."""
    rotary, half = case["rotary"], case["rotary"] // 2
    angle = positions.double().unsqueeze(1) * inv_freq.double()
    c, s = (torch.cos(angle) * factor).float().unsqueeze(1), (torch.sin(angle) * factor).float().unsqueeze(1)
    if case["inverse"]:
        s = -s
    start = case["head_dim"] - rotary if case["suffix"] else 0
    part = x[..., start:start + rotary]
    re, im = (part[..., 0::2], part[..., 1::2]) if case["interleaved"] else (part[..., :half], part[..., half:])
    a, b = re * c - im * s, im * c + re * s
    turned = torch.stack([a, b], -1).flatten(-2) if case["interleaved"] else torch.cat([a, b], -1)
    return torch.cat([x[..., :start], turned, x[..., start + rotary:]], -1)


def _cache_rows(blocks, page, at):
    """Numbers of the cache rows at positions `at` [batch, n] of each sequence."""
    return torch.gather(blocks.long(), 1, at.long() // page) * page + at.long() % page


def _plain_rope(s, case):
    b, n = case["batch"], case["rows"]
    q = _rotate(s["q"].float(), s["positions"], s["inv_freq"], s["factor"], case).to(s["q"].dtype)
    k = _rotate(s["k"].float(), s["positions"], s["inv_freq"], s["factor"], case).to(s["k"].dtype)
    if not case["append"]:
        return {"q": q, "k": k}
    at = torch.arange(n, device="cuda")
    real = (at < s["drafted"].unsqueeze(1)).reshape(-1)
    rows = _cache_rows(s["blocks"], case["page"], s["context"].unsqueeze(1) + at).reshape(-1)[real]
    s["k_pages"].flatten(0, 1)[rows] = k[real]
    s["v_pages"].flatten(0, 1)[rows] = s["v"][real]
    return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _visible(s, case, length):
    """[batch, rows, length]: the keys that each row sees."""
    b, n = case["batch"], case["rows"]
    key = torch.arange(length, device="cuda")
    draft = (key.unsqueeze(0) - s["context"].unsqueeze(1)).unsqueeze(1).expand(b, n, length)
    if s["mask"] is None:
        return draft <= torch.arange(n, device="cuda").unsqueeze(1)
    j = draft.clamp(0, n - 1)
    bit = (torch.gather(s["mask"], 2, j // 64) >> (j % 64)) & 1
    return ((draft < 0) | ((draft < n) & (bit == 1))) & (torch.arange(n, device="cuda") < s["drafted"].unsqueeze(1)).unsqueeze(2)


def _plain_attention(s, case):
    b, n, h, kv, d = case["batch"], case["rows"], case["heads"], case["kv_heads"], case["head_dim"]
    length = case["context"] + n
    k = s["k_pages"][s["blocks"].long()].flatten(1, 2)[:, :length].permute(0, 2, 1, 3).float()  # [batch, kv, length, d]
    v = s["v_pages"][s["blocks"].long()].flatten(1, 2)[:, :length].permute(0, 2, 1, 3).float()
    q = s["q"].float().reshape(b, n, kv, h // kv, d).permute(0, 2, 1, 3, 4).reshape(b, kv, n * (h // kv), d)
    score = torch.matmul(q, k.transpose(2, 3)).mul_(d ** -0.5).reshape(b, kv, n, h // kv, length)
    seen = _visible(s, case, length)[:, None, :, None, :]
    score.masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = score.sum(-1, keepdim=True)
    y = torch.matmul(score.reshape(b, kv, n * (h // kv), length), v).reshape(b, kv, n, h // kv, d)
    y = torch.where(total > 0, y / total, 0.0)
    return y.permute(0, 2, 1, 3, 4).reshape(b, n, h, d).to(s["q"].dtype)


def _plain_verify(s, case):
    b, n, v = case["batch"], case["rows"], case["vocab"]
    seq = torch.arange(b, device="cuda")
    greedy = (s["temperature"] == 0).unsqueeze(1)
    heat = torch.where(greedy, torch.ones_like(greedy, dtype=torch.float64), s["temperature"].unsqueeze(1).double())

    def chances(logits, node):
        x = logits[seq, node]
        x = (x.double() - x.amax(1, keepdim=True).double()) / heat
        p = torch.exp(x)
        p = p / p.sum(1, keepdim=True)
        best = torch.where(x == 0, torch.arange(v, device="cuda"), v).amin(1, keepdim=True)
        first = torch.zeros_like(p).scatter_(1, best, 1.0)
        return torch.where(greedy, first, p)

    node = torch.zeros(b, dtype=torch.int64, device="cuda")
    path = torch.full((b, n), -1, dtype=torch.int32, device="cuda")
    path[:, 0] = 0
    accepted = torch.ones(b, dtype=torch.int64, device="cuda")
    rest = chances(s["logits"], node)  # what is left of the target's distribution at the node
    draft = chances(s["draft_logits"], node) if s["draft_logits"] is not None else None
    for j in range(1, n):  # rows come after their parents: one walk over the rows tries the children of every node on the path, in order
        tried = (s["parents"][:, j] == node) & (j < s["drafted"])
        token = s["tokens"][:, j].long()
        q = draft[seq, token] if draft is not None else torch.ones(b, dtype=torch.float64, device="cuda")
        q = torch.where(greedy.squeeze(1), torch.ones_like(q), q)
        yes = tried & (s["accept_u"][:, j].double() * q < rest[seq, token])
        no = tried & ~yes
        one = torch.zeros_like(rest).scatter_(1, token.unsqueeze(1), 1.0)
        less = (rest - (torch.where(greedy, one, draft) if draft is not None else one)).clamp(min=0) if draft is not None else rest * (1 - one)
        left = less.sum(1, keepdim=True)
        rest = torch.where((no.unsqueeze(1)) & (left > 0), less / left, rest)
        node = torch.where(yes, j, node)
        path[seq[yes], accepted[yes]] = j
        accepted = accepted + yes
        rest = torch.where(yes.unsqueeze(1), chances(s["logits"], node), rest)
        if draft is not None:
            draft = torch.where(yes.unsqueeze(1), chances(s["draft_logits"], node), draft)
    sums = torch.cumsum(rest, 1)
    token = (sums <= s["sample_u"].double().unsqueeze(1) * sums[:, -1:]).sum(1).clamp(max=v - 1)
    return {"path": path, "accepted": accepted.to(torch.int32), "token": token.to(torch.int32)}


def _plain_keep(s, case):
    at = torch.arange(case["rows"], device="cuda").expand(case["batch"], -1)
    real = at < s["accepted"].unsqueeze(1)
    to = _cache_rows(s["blocks"], case["page"], s["context"].unsqueeze(1) + at)[real]
    src = _cache_rows(s["blocks"], case["page"], s["context"].unsqueeze(1) + s["path"].clamp(min=0))[real]
    for pages in (s["k_pages"], s["v_pages"]):
        rows = pages.flatten(1, 2)
        rows[:, to] = rows[:, src]
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


_context = None


def _ctx():
    """The framework's context on the current stream, made once as a program does."""
    global _context
    if _context is None:
        from zllm_b200.backend import B200Context

        _context = B200Context(0)
    return _context


def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if own:
        ctx = _ctx()
        if op == "tree":
            positions, mask = ctx.draft_tree(s["parents"], s["context"], s["drafted"])
            return {"positions": positions, "mask": mask}
        if op == "rope":
            if case["append"]:
                q = ctx.rope_append(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["blocks"], s["context"], s["positions"], s["inv_freq"], draft_lens=s["drafted"], interleaved=case["interleaved"], suffix=case["suffix"],
                                    factor=s["factor"])
                return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
            q, k = ctx.rope_rows(s["q"], s["k"], s["positions"], s["inv_freq"], interleaved=case["interleaved"], suffix=case["suffix"], factor=s["factor"], inverse=case["inverse"])
            return {"q": q, "k": k}
        if op == "attn":
            return ctx.tree_attention(s["q"], s["k_pages"], s["v_pages"], s["blocks"], s["context"], mask=s["mask"], draft_lens=s["drafted"])
        if op == "verify":
            path, accepted, token = ctx.verify_draft(s["logits"], s["tokens"], s["parents"], s["accept_u"], s["sample_u"], s["temperature"], draft_logits=s["draft_logits"], draft_lens=s["drafted"])
            return {"path": path, "accepted": accepted, "token": token}
        ctx.cache_keep_path(s["k_pages"], s["v_pages"], s["blocks"], s["context"], s["path"], s["accepted"])
        return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if op == "tree":
        return _plain_tree(s["parents"], s["context"], s["drafted"])
    if op == "rope":
        return _plain_rope(s, case)
    if op == "attn":
        return _plain_attention(s, case)
    if op == "verify":
        return _plain_verify(s, case)
    return _plain_keep(s, case)


# ---- what a pass cannot do without
def work(case):
    op, b, n = case["op"], case["batch"], case["rows"]
    size = _SIZE[case["dtype"]] if "dtype" in case else 4
    if op == "tree":
        return {"bytes": b * (8 + n * (8 + -(-n // 64) * 8)), "flops": 0}
    if op == "rope":
        row = (case["heads"] + case["kv_heads"] * (2 if case["append"] else 1)) * case["head_dim"] * size
        return {"bytes": b * n * (2 * row + 4), "flops": 3.0 * b * n * (case["heads"] + case["kv_heads"]) * case["rotary"]}
    if op == "attn":
        mean = (5 * case["context"] / 8 if case["ragged"] else case["context"]) + n  # ragged lengths: a quarter of the longest up to the longest
        return {"bytes": b * (2 * mean * case["kv_heads"] + 2 * n * case["heads"]) * case["head_dim"] * size, "flops": 4.0 * b * n * mean * case["heads"] * case["head_dim"]}
    if op == "verify":
        # the rows of the nodes on the path, the last one's included; a drafted tree keeps two or three of its tokens
        visits = min(n, 3)
        return {"bytes": b * (visits * case["vocab"] * size * (2 if case["drawn"] else 1) + 16 * n), "flops": b * visits * case["vocab"] * (6.0 if case["drawn"] else 3.0)}
    kept = max(0.0, (max(1, min(6, n // 2)) - 1) / 2)  # rows that move, on average
    return {"bytes": b * case["layers"] * kept * 4 * case["kv_heads"] * case["head_dim"] * size + 8.0 * b * n, "flops": 0}


# ---- from the definitions, in 64 bits
def exact(case, seed):
    op = case["op"]
    if op not in ("rope", "attn"):
        return None  # whole numbers, and rows that are moved as they are
    s = prepare(case, seed)
    if op == "rope":
        pairs = torch.arange(case["rotary"] // 2, device="cuda")
        first = case["head_dim"] - case["rotary"] if case["suffix"] else 0
        i, j = (first + 2 * pairs, first + 2 * pairs + 1) if case["interleaved"] else (first + pairs, first + pairs + case["rotary"] // 2)
        turn = torch.polar(torch.full((), s["factor"], dtype=torch.float64, device="cuda"), s["positions"].double()[:, None, None] * s["inv_freq"].double() * (-1 if case["inverse"] else 1))
        done = []
        for x in (s["q"], s["k"]):
            x = x.double()
            z = torch.complex(x[..., i], x[..., j]) * turn
            x[..., i], x[..., j] = z.real, z.imag
            done.append(x)
        if not case["append"]:
            return {"q": done[0], "k": done[1]}
        return {"q": done[0], "k_pages": None, "v_pages": None}
    b, n, h, kv, d = case["batch"], case["rows"], case["heads"], case["kv_heads"], case["head_dim"]
    if 4.0 * b * n * (case["context"] + n) * h * d > 6e11:
        return None
    y = torch.zeros((b, n, h, d), dtype=torch.float64, device="cuda")
    for i in range(b):
        ctx = int(s["context"][i])
        real = n if s["drafted"] is None else int(s["drafted"][i])
        rows = torch.cat([s["blocks"][i].long()[:, None] * case["page"] + torch.arange(case["page"], device="cuda")], 0).reshape(-1)[:ctx + n]
        seen = torch.ones((n, ctx + n), dtype=torch.bool, device="cuda")
        if s["mask"] is None:
            seen[:, ctx:] = torch.ones((n, n), dtype=torch.bool, device="cuda").tril()
        else:
            words = s["mask"][i]
            seen[:, ctx:] = torch.stack([(words[:, t // 64] >> (t % 64)) & 1 for t in range(n)], 1).bool()
        for g in range(kv):
            k, v = s["k_pages"].flatten(0, 1)[rows, g].double(), s["v_pages"].flatten(0, 1)[rows, g].double()
            for m in range(g * (h // kv), (g + 1) * (h // kv)):
                z = (s["q"][i, :real, m].double() @ k.T) / math.sqrt(d)
                z = torch.softmax(z.masked_fill(~seen[:real], -math.inf), 1)
                y[i, :real, m] = z @ v
    return y
