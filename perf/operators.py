"""Timed cases of the language-model operators (kbb200.lm): query/key norms with the position rotation,
attention of a batch over a shared prefix in a paged cache, the cache's page operations, and penalties, biases
and masks on logits.

Each case is one call as a decoding or training program makes it, at sizes from the smallest (where latency
counts) to the largest.  `run` computes it with the library's kernels where `own` is set, and otherwise in its
plain form: elementary torch operations in 32 bits, rounded once at the end.  `exact` computes the same from the
definitions in 64 bits.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6
ROPE_BASE = 10000.0


# ------------------------------------------------------------------ cases
def _rope(name, dtype, direction, tokens, heads_q, heads_kv, dim, rotary, interleaved=False):
    return {"name": name, "op": "qk_norm_rope", "dtype": dtype, "direction": direction, "tokens": tokens,
            "heads_q": heads_q, "heads_kv": heads_kv, "dim": dim, "rotary": rotary, "interleaved": interleaved}


def _attn(name, dtype, batch, queries, heads_q, heads_kv, dim, page, prefix_pages, suffix):
    return {"name": name, "op": "attention", "dtype": dtype, "batch": batch, "queries": queries, "heads_q": heads_q,
            "heads_kv": heads_kv, "dim": dim, "page": page, "prefix_pages": prefix_pages, "suffix": suffix}


def _cache(name, dtype, use, planes, heads_kv, dim, page, parent_len, children, tokens):
    return {"name": name, "op": "cache", "dtype": dtype, "use": use, "planes": planes, "heads_kv": heads_kv,
            "dim": dim, "page": page, "parent_len": parent_len, "children": children, "tokens": tokens}


def _logits(name, dtype, batch, vocab, prompt, output, bias, mask):
    return {"name": name, "op": "logits", "dtype": dtype, "batch": batch, "vocab": vocab, "prompt": prompt,
            "output": output, "bias": bias, "mask": mask}


def listed():
    return [
        # one decoding step of 64 sequences: a few hundred KB, so launch latency
        _rope("qk-decode-bf16", "bf16", "forward", 64, 32, 8, 128, 128),
        # the forward pass of a packed training batch
        _rope("qk-train-bf16", "bf16", "forward", 16384, 32, 8, 128, 128),
        # its backward pass, with the gradients of both weights
        _rope("qk-train-backward-bf16", "bf16", "backward", 16384, 32, 8, 128, 128),
        # odd token count, seven query heads per key head, a partial interleaved rotation, in fp32
        _rope("qk-odd-backward-f32", "f32", "backward", 1001, 14, 2, 80, 40, True),
        # four samples of a short prompt, one new token each: latency
        _attn("attn-few-bf16", "bf16", 4, 1, 32, 8, 128, 16, 32, 64),
        # best of 64 on an 8192-token prompt, ragged continuations
        _attn("attn-best-of-64-bf16", "bf16", 64, 1, 32, 8, 128, 16, 512, 1000),
        # a rollout step: 256 samples on a long prompt
        _attn("attn-rollout-bf16", "bf16", 256, 1, 32, 8, 128, 64, 512, 700),
        # fp32 cache, three draft tokens verified at once, causal among themselves
        _attn("attn-draft-f32", "f32", 16, 3, 16, 4, 64, 16, 130, 200),
        # branching a sequence into 4 drafts of 5 tokens: fork, reserve, append
        _cache("cache-branch-bf16", "bf16", "branch", 4, 8, 128, 16, 1003, 4, 5),
        # one round of a sampler over all layers' pages: fork 64, free every other, compact
        _cache("cache-round-bf16", "bf16", "round", 64, 8, 128, 16, 8200, 64, 0),
        # the logits of one sequence
        _logits("logits-one-f32", "f32", 1, 32000, 500, 200, 0, False),
        # the logits of a large batch with histories, biases and a grammar's masks
        _logits("logits-batch-bf16", "bf16", 256, 131072, 2048, 1000, 300, True),
    ]


def _span(rng, lo, hi):
    """Whole numbers spread over the logarithm of [lo, hi]."""
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    while True:
        c = _draw(rng)
        widths = [c.get("heads_q", 0) * c.get("dim", 0), (c.get("heads_q", 0) + 2 * c.get("heads_kv", 0)) * c.get("dim", 0),
                  c.get("prefix_pages", 0) * c.get("page", 0)]
        if 3072 not in [*c.values(), *widths]:
            return c


def _draw(rng):
    op = rng.choice(["qk_norm_rope", "attention", "attention", "cache", "logits"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "qk_norm_rope":
        heads_kv = rng.choice([1, 2, 4, 8])
        heads_q = heads_kv * rng.choice([1, 2, 4, 7])
        dim = rng.choice([64, 72, 80, 96, 128, 192, 256])
        rotary = dim if rng.random() < 0.6 else 2 * rng.randint(1, dim // 2)
        top = 16384 * 40 * 128 * 2 // ((heads_q + heads_kv) * dim * SIZE[dtype])
        c = _rope("", dtype, rng.choice(["forward", "backward"]), _span(rng, 1, min(top, 20000)), heads_q, heads_kv,
                  dim, rotary, rng.random() < 0.4)
    elif op == "attention":
        heads_kv = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 4, 5, 8])
        dim = rng.choice([64, 80, 96, 128, 128])
        queries = rng.choice([1, 1, 1, 2, 3, 8])
        page = rng.choice([16, 32, 64, 128])
        batch = _span(rng, 1, 256)
        prefix = _span(rng, 1, 32768) // page
        suffix = _span(rng, queries, 1500)
        most = 256 * 32 * 128 * 33468 // (2 if dtype != "f32" else 16)  # row x key x dim products
        while batch > 1 and batch * queries * heads_kv * group * dim * (prefix * page + suffix) > most:
            batch //= 2
        c = _attn("", dtype, batch, queries, heads_kv * group, heads_kv, dim, page, prefix, suffix)
    elif op == "cache":
        use = rng.choice(["branch", "round"])
        c = _cache("", dtype, use, 2 * _span(rng, 1, 32 if dtype != "f32" else 16), rng.choice([1, 2, 4, 8]),
                   rng.choice([64, 80, 128]), rng.choice([8, 16, 32]), _span(rng, 1, 9000), _span(rng, 1, 64),
                   rng.randint(1, 20) if use == "branch" else 0)
        while c["planes"] > 2 and c["planes"] * c["children"] * c["page"] * c["heads_kv"] * c["dim"] * SIZE[dtype] > 130e6:
            c["planes"] = 2 * (c["planes"] // 4)
        c["planes"] = max(2, c["planes"])
    else:
        vocab = _span(rng, 1000, 200000)
        batch = max(1, min(_span(rng, 1, 256), 256 * 131072 * 2 // (vocab * SIZE[dtype])))
        c = _logits("", dtype, batch, vocab, _span(rng, 1, 4000) if rng.random() < 0.8 else 0,
                    _span(rng, 1, 3000) if rng.random() < 0.8 else 0, rng.choice([0, 1, 300]), rng.random() < 0.6)
    c.pop("name")
    return c


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    c, dt = case, DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, device=dev, generator=g, dtype=torch.float32)

    def rand(*shape):
        return torch.rand(shape, device=dev, generator=g, dtype=torch.float32)

    def perm(n):
        return torch.argsort(rand(n)).to(torch.int32)

    s = {"case": dict(c)}
    if c["op"] == "qk_norm_rope":
        T, hq, hkv, d, r = c["tokens"], c["heads_q"], c["heads_kv"], c["dim"], c["rotary"]
        qkv = (randn(T, (hq + 2 * hkv) * d) * 1.5).to(dt)  # the packed projection; q and k are views of it
        s["q"] = qkv[:, : hq * d].view(T, hq, d)
        s["k"] = qkv[:, hq * d: (hq + hkv) * d].view(T, hkv, d)
        s["qw"], s["kw"] = (1 + 0.1 * randn(d)).to(dt), (1 + 0.1 * randn(d)).to(dt)
        longest = 4096
        f = ROPE_BASE ** (-torch.arange(0, r, 2, device=dev, dtype=torch.float64) / r)
        a = torch.arange(longest, device=dev, dtype=torch.float64)[:, None] * f
        s["cos"], s["sin"] = a.cos().float().contiguous(), a.sin().float().contiguous()
        at = int(torch.randint(0, longest, (1,), device=dev, generator=g))
        if T <= 256:  # decoding: every token at its own place
            s["pos"] = torch.randint(0, longest, (T,), device=dev, generator=g)
        else:         # training: sequences packed one after the other
            s["pos"] = (torch.arange(T, device=dev) + at) % 2048
        if c["direction"] == "backward":
            s["dq"], s["dk"] = randn(T, hq, d).to(dt), randn(T, hkv, d).to(dt)
    elif c["op"] == "attention":
        B, Q, hq, hkv, d, page = c["batch"], c["queries"], c["heads_q"], c["heads_kv"], c["dim"], c["page"]
        n_pre, n_suf = c["prefix_pages"], -(-c["suffix"] // page)
        pages = n_pre + B * n_suf + 3
        pool = randn(2, pages, page, hkv, d).to(dt)
        s["k_pages"], s["v_pages"] = pool[0], pool[1]
        s["q"] = (2 * randn(B, Q, hq, d)).to(dt)
        order = perm(pages)
        s["prefix"] = order[:n_pre].contiguous()
        suffix = torch.randint(Q, c["suffix"] + 1, (B,), device=dev, generator=g)
        suffix[0] = c["suffix"]
        table = torch.full((B, n_pre + n_suf), -1, device=dev, dtype=torch.int32)
        table[:, :n_pre] = s["prefix"]
        table[:, n_pre:] = order[n_pre: n_pre + B * n_suf].view(B, n_suf)
        used = torch.arange(n_suf, device=dev)[None] * page < suffix[:, None]
        table[:, n_pre:] = torch.where(used, table[:, n_pre:], torch.full_like(table[:, n_pre:], -1))
        lens = suffix + n_pre * page
        if B >= 8:  # a slot whose sequence has ended
            lens[B // 2] = 0
            table[B // 2] = -1
        s["table"], s["lens"] = table, lens.to(torch.int32)
    elif c["op"] == "cache":
        P, hkv, d, page, n = c["planes"], c["heads_kv"], c["dim"], c["page"], c["children"]
        full = -(-c["parent_len"] // page)
        width = -(-(c["parent_len"] + c["tokens"]) // page)
        extra = width - full
        pages = full + (2 + 2 * extra) * n + 5
        s["pool"] = randn(P, pages, page, hkv, d).to(dt)
        s["table"] = torch.full((n + 1, width), -1, device=dev, dtype=torch.int32)
        order = perm(pages)[:full]
        s["table"][0, :full] = order
        s["lens"] = torch.zeros(n + 1, device=dev, dtype=torch.int32)
        s["lens"][0] = c["parent_len"]
        s["refs"] = torch.zeros(pages, device=dev, dtype=torch.int32)
        s["refs"][order.long()] = 1
        s["parents"] = torch.zeros(n, device=dev, dtype=torch.int32)
        s["children"] = torch.arange(1, n + 1, device=dev, dtype=torch.int32)
        s["ended"] = s["children"][::2].contiguous()
        s["k"], s["v"] = randn(n, c["tokens"], hkv, d).to(dt), randn(n, c["tokens"], hkv, d).to(dt)
    else:
        B, V = c["batch"], c["vocab"]
        s["logits"] = (3 * randn(B, V)).to(dt)

        def history(n):  # some tokens come often, most never; rows of different lengths, filled up with -1
            ids = (V * rand(B, n) ** 4).long().clamp_(0, V - 1)
            keep = (rand(B) * (n + 1)).long()
            keep[-1] = n
            return torch.where(torch.arange(n, device=dev)[None] < keep[:, None], ids, torch.full_like(ids, -1))

        s["prompt"] = history(c["prompt"]) if c["prompt"] else None
        s["output"] = history(c["output"]) if c["output"] else None
        s["repetition"], s["presence"], s["frequency"] = 1 + 0.5 * rand(B), rand(B), 0.5 * rand(B)
        nb = c["bias"]
        s["bias_ids"] = s["bias_values"] = s["mask"] = None
        if nb:
            start = torch.randint(0, V, (B, 1), device=dev, generator=g)
            s["bias_ids"] = (start + torch.arange(nb, device=dev)[None] * (V // nb)) % V
            s["bias_values"] = 5 * randn(B, nb)
        if c["mask"]:
            words = -(-V // 32)
            m = torch.randint(-2 ** 31, 2 ** 31, (B, words), device=dev, generator=g, dtype=torch.int64)
            m &= torch.randint(-2 ** 31, 2 ** 31, (B, words), device=dev, generator=g, dtype=torch.int64)
            m[rand(B) < 0.5] = -1  # half the sequences have no grammar
            if B >= 4:
                m[B // 2] = 0      # one whose grammar has come to its end
            s["mask"] = m.to(torch.int32)
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return _RUN_OWN[op](_lm(), state)
    return _RUN_PLAIN[op](state)


def _lm():
    lm = sys.modules.get("kbb200.lm")
    if lm is None:
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "kernelbench-hip_b200"))
        import kbb200.lm as lm
    return lm


def _own_rope(lm, s):
    c = s["case"]
    if c["direction"] == "forward":
        return lm.qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["cos"], s["sin"], s["pos"], eps=EPS,
                               interleaved=c["interleaved"])
    return lm.qk_norm_rope_backward(s["dq"], s["dk"], s["q"], s["k"], s["qw"], s["kw"], s["cos"], s["sin"], s["pos"],
                                    eps=EPS, interleaved=c["interleaved"])


def _own_attention(lm, s):
    return lm.shared_prefix_attention(s["q"], s["k_pages"], s["v_pages"], s["prefix"], s["table"], s["lens"])


def _own_cache(lm, s):
    c = s["case"]
    granted = lm.cache_fork(s["pool"], s["table"], s["lens"], s["refs"], s["parents"], s["children"])
    if c["use"] == "branch":
        room = lm.cache_reserve(s["table"], s["lens"], s["refs"], s["children"], c["tokens"], c["page"])
        lm.cache_append(s["k"], s["v"], s["pool"][0], s["pool"][1], s["table"], s["lens"], s["children"])
        return granted, room, s["table"], s["lens"], s["refs"], s["pool"]
    lm.cache_free(s["table"], s["lens"], s["refs"], s["ended"])
    live = lm.cache_compact(s["pool"], s["table"], s["refs"])
    return granted, live, s["table"], s["lens"], s["refs"], s["pool"]


def _own_logits(lm, s):
    return lm.penalize_logits(s["logits"], prompt=s["prompt"], output=s["output"], repetition=s["repetition"],
                              presence=s["presence"], frequency=s["frequency"], bias_ids=s["bias_ids"],
                              bias_values=s["bias_values"], mask=s["mask"])


_RUN_OWN = {"qk_norm_rope": _own_rope, "attention": _own_attention, "cache": _own_cache, "logits": _own_logits}


# ------------------------------------------------------------------ plain forms
def _pairs(x, r, interleaved):
    """The two halves of each rotated pair, and the rest."""
    if interleaved:
        return x[..., 0:r:2], x[..., 1:r:2], x[..., r:]
    return x[..., : r // 2], x[..., r // 2: r], x[..., r:]


def _joined(a, b, rest, interleaved):
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, rest), -1)


def _plain_rope(s):
    c = s["case"]
    r, il = c["rotary"], c["interleaved"]
    cos, sin = s["cos"][s["pos"]][:, None], s["sin"][s["pos"]][:, None]

    def forward(x, w):
        x = x.float()
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        a, b, rest = _pairs(y, r, il)
        return _joined(a * cos - b * sin, b * cos + a * sin, rest, il)

    def backward(dz, x, w):
        x, dz = x.float(), dz.float()
        rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        a, b, rest = _pairs(dz, r, il)
        dy = _joined(a * cos + b * sin, b * cos - a * sin, rest, il)
        xhat = x * rstd
        dh = dy * w.float()
        return rstd * (dh - xhat * (dh * xhat).mean(-1, keepdim=True)), (dy * xhat).sum((0, 1))

    dt = s["q"].dtype
    if c["direction"] == "forward":
        return forward(s["q"], s["qw"]).to(dt), forward(s["k"], s["kw"]).to(dt)
    dq, dqw = backward(s["dq"], s["q"], s["qw"])
    dk, dkw = backward(s["dk"], s["k"], s["kw"])
    return dq.to(dt), dk.to(dt), dqw.to(s["qw"].dtype), dkw.to(s["kw"].dtype)


def _plain_attention(s):
    c = s["case"]
    B, Q, hkv, d, page, n_pre = c["batch"], c["queries"], c["heads_kv"], c["dim"], c["page"], c["prefix_pages"]
    G = c["heads_q"] // hkv
    q = (s["q"].float() * d ** -0.5).view(B, Q, hkv, G, d)
    pre, own_rows = s["prefix"].long(), s["table"][:, n_pre:].long().clamp(min=0)
    kp, vp = (x[pre].float().view(-1, hkv, d) for x in (s["k_pages"], s["v_pages"]))
    ks, vs = (x[own_rows].float().flatten(1, 2) for x in (s["k_pages"], s["v_pages"]))
    # each key head's queries against the prefix in one product, and against their own keys
    rows = q.permute(2, 0, 1, 3, 4).reshape(hkv, B * Q * G, d)
    sp = torch.matmul(rows, kp.permute(1, 2, 0)).view(hkv, B, Q, G, -1)
    ss = torch.matmul(q.permute(2, 0, 1, 3, 4).reshape(hkv, B, Q * G, d), ks.permute(2, 0, 3, 1)).view(hkv, B, Q, G, -1)
    sc = torch.cat((sp, ss), -1)
    seen = s["lens"].long()[:, None] - Q + 1 + torch.arange(Q, device=q.device)  # keys that each query sees
    sc = sc.masked_fill(torch.arange(sc.shape[-1], device=q.device) >= seen[:, :, None, None], -math.inf)
    top = sc.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(sc - top)
    total = p.sum(-1, keepdim=True)
    p1, p2 = p[..., : n_pre * page], p[..., n_pre * page:]
    o = torch.matmul(p1.reshape(hkv, B * Q * G, -1), vp.transpose(0, 1)).view(hkv, B, Q, G, d)
    o = o + torch.matmul(p2.reshape(hkv, B, Q * G, -1), vs.permute(2, 0, 1, 3)).view(hkv, B, Q, G, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    lse = (top + torch.log(total)).squeeze(-1)
    return (o.permute(1, 2, 0, 3, 4).reshape(B, Q, -1, d).to(s["q"].dtype),
            lse.permute(1, 2, 0, 3).reshape(B, Q, -1).contiguous())


def _plain_cache(s):
    c = s["case"]
    pool, table, lens, refs, page = s["pool"], s["table"], s["lens"], s["refs"], c["page"]
    parents, children = s["parents"].long(), s["children"].long()
    one = torch.ones((), device=pool.device, dtype=torch.int32)

    def count(rows, by):  # refs[p] += by for every page p of the rows
        rows = rows.flatten().long()
        refs.index_add_(0, rows.clamp(min=0), torch.where(rows >= 0, by, torch.zeros_like(by)).to(torch.int32))

    # fork: a child takes its parent's full pages and a copy of the last one where that is not full
    rows, n_keys = table[parents].clone(), lens[parents]
    need = n_keys % page != 0
    free = torch.argsort(refs != 0, stable=True).to(torch.int32)
    rank = torch.cumsum(need.int(), 0) - 1
    granted = ~need | (rank < (refs == 0).sum())
    old = torch.where(granted[:, None], table[children], torch.full_like(rows, -1))
    last = (n_keys // page).long()[:, None].clamp(max=table.shape[1] - 1)
    src, dst = rows.gather(1, last)[:, 0], free[rank.clamp(0, free.numel() - 1).long()]
    moved = need & granted
    rows = torch.where(moved[:, None], rows.scatter(1, last, dst[:, None]), rows)
    to = torch.where(moved, dst, src).long()[moved]
    pool[:, to] = pool[:, src.long()[moved]]
    table[children] = torch.where(granted[:, None], rows, table[children])
    lens[children] = torch.where(granted, n_keys, lens[children])
    count(torch.where(granted[:, None], rows, torch.full_like(rows, -1)), one)
    count(old, -one)
    granted = granted.to(torch.int32)
    if c["use"] == "branch":
        # reserve: as many pages more as the new tokens need, the lowest free ones, in order
        T = c["tokens"]
        have = (lens[children] + page - 1) // page
        want = (lens[children] + T + page - 1) // page - have
        ends = torch.cumsum(want, 0)
        room = (ends <= (refs == 0).sum()) & ((lens[children] + T) <= table.shape[1] * page)
        free = torch.argsort(refs != 0, stable=True).to(torch.int32)
        at = torch.arange(table.shape[1], device=pool.device)[None] - have[:, None]
        new = (at >= 0) & (at < want[:, None]) & room[:, None]
        pick = free[(at + (ends - want)[:, None]).clamp(0, free.numel() - 1).long()]
        table[children] = torch.where(new, pick, table[children])
        count(torch.where(new, pick, torch.full_like(pick, -1)), one)
        lens[children] = torch.where(room, lens[children] + T, lens[children])
        # append
        pos = lens[children].long()[:, None] - T + torch.arange(T, device=pool.device)
        pages = table[children].gather(1, pos // page).long()
        pool[0, pages, pos % page], pool[1, pages, pos % page] = s["k"], s["v"]
        return granted, room.to(torch.int32), table, lens, refs, pool
    # free
    ended = s["ended"].long()
    count(table[ended], -one)
    table[ended] = -1
    lens[ended] = 0
    # compact: the live pages past the live count go to the holes below it, in order
    live = (refs > 0).sum()
    index = torch.arange(refs.numel(), device=pool.device)
    src, dst = index[(refs > 0) & (index >= live)], index[(refs == 0) & (index < live)]
    pool[:, dst] = pool[:, src]
    to = index.to(torch.int32)
    to[src] = dst.to(torch.int32)
    refs[dst] = refs[src]
    refs[src] = 0
    table.copy_(torch.where(table >= 0, to[table.long().clamp(min=0)], table))
    return granted, live.to(torch.int32).view(1), table, lens, refs, pool


def _plain_logits(s):
    c = s["case"]
    x = s["logits"].float()
    B, V = x.shape

    def counts(ids):
        if ids is None:
            return torch.zeros(B, V, device=x.device)
        n = torch.zeros(B, V + 1, device=x.device)
        return n.scatter_add_(1, torch.where(ids < 0, V, ids), torch.ones_like(ids, dtype=torch.float32))[:, :V]

    made = counts(s["output"])
    seen = (made > 0) | (counts(s["prompt"]) > 0)
    rep = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * made - s["presence"][:, None] * (made > 0)
    if s["bias_ids"] is not None:
        x = x.scatter_add(1, s["bias_ids"], s["bias_values"])
    if s["mask"] is not None:
        bits = (s["mask"][:, :, None] >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
        x = x.masked_fill(bits.view(B, -1)[:, :V] == 0, -math.inf)
    return x.to(s["logits"].dtype)


_RUN_PLAIN = {"qk_norm_rope": _plain_rope, "attention": _plain_attention, "cache": _plain_cache,
              "logits": _plain_logits}


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    return _EXACT[case["op"]](case, prepare(case, seed))


def _exact_rope(c, s):
    r, d = c["rotary"], c["dim"]
    turn = torch.complex(s["cos"][s["pos"]].double(), s["sin"][s["pos"]].double())[:, None]
    at = torch.arange(r, device="cuda")
    first, second = (at[0::2], at[1::2]) if c["interleaved"] else (at[: r // 2], at[r // 2:])

    def forward(x, w):
        y = w * x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / d + EPS)
        z = torch.complex(y[..., first], y[..., second]) * turn
        out = y.clone()
        out[..., first], out[..., second] = z.real, z.imag
        return out

    leaves = [s[n].double().requires_grad_(c["direction"] == "backward") for n in ("q", "k", "qw", "kw")]
    zq, zk = forward(leaves[0], leaves[2]), forward(leaves[1], leaves[3])
    if c["direction"] == "forward":
        return zq, zk
    return torch.autograd.grad([zq, zk], leaves, [s["dq"].double(), s["dk"].double()])


def _exact_attention(c, s):
    B, Q, hq, d, page, n_pre = c["batch"], c["queries"], c["heads_q"], c["dim"], c["page"], c["prefix_pages"]
    G = hq // c["heads_kv"]
    out = torch.zeros(B, Q, hq, d, device="cuda", dtype=torch.float64)
    lse = torch.full((B, Q, hq), -math.inf, device="cuda", dtype=torch.float64)
    lens = s["lens"].tolist()
    for h in range(c["heads_kv"]):
        kh, vh = s["k_pages"][:, :, h].double(), s["v_pages"][:, :, h].double()
        pre = s["prefix"].long()
        kp, vp = kh[pre].view(-1, d), vh[pre].view(-1, d)
        for b, n in enumerate(lens):
            own_pages = s["table"][b, n_pre: max(n_pre, -(-n // page))].long()
            keys = torch.cat((kp, kh[own_pages].view(-1, d)))[:n]
            values = torch.cat((vp, vh[own_pages].view(-1, d)))[:n]
            for t in range(Q):
                m = n - Q + 1 + t
                if m <= 0:
                    continue
                x = s["q"][b, t, h * G: (h + 1) * G].double() @ keys[:m].T / math.sqrt(d)
                out[b, t, h * G: (h + 1) * G] = torch.softmax(x, -1) @ values[:m]
                lse[b, t, h * G: (h + 1) * G] = torch.logsumexp(x, -1)
    return out, lse


def _exact_cache(c, s):
    """The page operations one sequence at a time, on lists."""
    pool, page = s["pool"].double(), c["page"]
    rows = [[p for p in row if p >= 0] for row in s["table"].tolist()]
    lens, refs = s["lens"].tolist(), s["refs"].tolist()
    children = s["children"].tolist()
    before = [(list(rows[p]), lens[p]) for p in s["parents"].tolist()]
    held = [list(rows[k]) for k in children]

    def take():
        p = refs.index(0)
        refs[p] = 1
        return p

    for k, (row, n) in zip(children, before):
        row = list(row)
        shared = row[: n // page]
        if n % page:
            p = take()
            pool[:, p] = pool[:, row[n // page]]
            row[n // page] = p
        for p in shared:
            refs[p] += 1
        rows[k], lens[k] = row, n
    for row in held:
        for p in row:
            refs[p] -= 1
    if c["use"] == "branch":
        for i, k in enumerate(children):
            for t in range(c["tokens"]):
                if lens[k] % page == 0:
                    rows[k].append(take())
                for plane, x in ((0, s["k"]), (1, s["v"])):
                    pool[plane, rows[k][lens[k] // page], lens[k] % page] = x[i, t].double()
                lens[k] += 1
        last = torch.ones(len(children))
    else:
        for k in s["ended"].tolist():
            for p in rows[k]:
                refs[p] -= 1
            rows[k], lens[k] = [], 0
        live = sum(r > 0 for r in refs)
        holes = [p for p in range(live) if not refs[p]]
        to = {}
        for p in range(live, len(refs)):
            if refs[p]:
                to[p] = holes.pop(0)
                pool[:, to[p]] = pool[:, p]
                refs[to[p]], refs[p] = refs[p], 0
        rows = [[to.get(p, p) for p in row] for row in rows]
        last = torch.tensor([live])
    width = s["table"].shape[1]
    table = torch.tensor([row + [-1] * (width - len(row)) for row in rows])
    return torch.ones(len(children)).int(), last.int(), table.int(), torch.tensor(lens).int(), torch.tensor(refs).int(), pool


def _exact_logits(c, s):
    x = s["logits"].double()
    V = x.shape[1]
    for b in range(x.shape[0]):
        row = x[b]
        made = torch.zeros(V, device="cuda", dtype=torch.int64)
        seen = torch.zeros(V, device="cuda", dtype=torch.bool)
        for ids, is_output in ((s["prompt"], False), (s["output"], True)):
            if ids is None:
                continue
            ids = ids[b][ids[b] >= 0]
            seen[ids] = True
            if is_output:
                made = torch.bincount(ids, minlength=V)
        rep = s["repetition"][b].double()
        row[seen] = torch.where(row[seen] > 0, row[seen] / rep, row[seen] * rep)
        row -= s["frequency"][b].double() * made + s["presence"][b].double() * (made > 0)
        if s["bias_ids"] is not None:
            row[s["bias_ids"][b]] += s["bias_values"][b].double()
        if s["mask"] is not None:
            words = s["mask"][b].long() & 0xFFFFFFFF
            at = torch.arange(V, device="cuda")
            row[((words[at // 32] >> (at % 32)) & 1) == 0] = -math.inf
    return x


_EXACT = {"qk_norm_rope": _exact_rope, "attention": _exact_attention, "cache": _exact_cache, "logits": _exact_logits}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c, e = case, SIZE[case["dtype"]]
    if c["op"] == "qk_norm_rope":
        n = c["tokens"] * (c["heads_q"] + c["heads_kv"]) * c["dim"]
        table = min(c["tokens"], 4096) * c["rotary"] * 4
        passes, ops = (2, 10) if c["direction"] == "forward" else (3, 24)
        return {"bytes": passes * n * e + table + 8 * c["tokens"], "flops": ops * n}
    if c["op"] == "attention":
        keys, rows = c["prefix_pages"] * c["page"], c["batch"] * c["queries"] * c["heads_q"]
        mean = (c["suffix"] + c["queries"]) / 2
        kv = 2 * c["heads_kv"] * c["dim"] * e
        return {"bytes": kv * (keys + c["batch"] * mean) + rows * (2 * c["dim"] * e + 4),
                "flops": 4 * rows * c["dim"] * (keys + mean)}
    if c["op"] == "cache":
        one = c["page"] * c["heads_kv"] * c["dim"] * e
        n, part = c["children"], bool(c["parent_len"] % c["page"])
        table = 4 * n * -(-(c["parent_len"] + c["tokens"]) // c["page"])
        if c["use"] == "branch":
            return {"bytes": 2 * c["planes"] * one * n * part + 4 * c["tokens"] * n * one // c["page"] + 2 * table,
                    "flops": 0}
        # the children's last pages are copied, and in the steady state those of the half that stays move into holes
        return {"bytes": 2 * c["planes"] * one * (n + n // 2) * part + 4 * table, "flops": 0}
    n = c["batch"] * c["vocab"]
    return {"bytes": 2 * n * e + (n // 8 if c["mask"] else 0) + c["batch"] * (8 * (c["prompt"] + c["output"]) // 2 + 12 * c["bias"]),
            "flops": 2 * n}
