"""The token-by-token operators: a paged key/value cache and its append, the
attention of one new token over it, log probabilities of given tokens with
their gradient, and Linear products with 4-bit weights.

`listed()` names the measured cases, `draw()` makes more of the same ranges,
`prepare()` makes a case's inputs, `run()` is one pass (in plain torch, or
through haelixe_b200 where `own` is true), `work()` what a pass cannot do
without, and `exact()` the results in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
ROPE_BASE = 500000.0


def listed():
    return [
        # One sequence's new token entering a 32-head layer: launch latency alone.
        dict(name="append_one_token", op="append", dtype="bf16", tokens=1, seqs=1, q_heads=32, kv_heads=32,
             dim=128, page=16, far=8192, heads_first=False),
        # A prompt of 8192 tokens written to the cache, its queries rotated in the same call.
        dict(name="append_prompt", op="append", dtype="bf16", tokens=8192, seqs=1, q_heads=32, kv_heads=32,
             dim=128, page=64, far=8192, heads_first=False),
        # One sequence answering from a cache of 8192 positions, every head with its own keys.
        dict(name="attend_one_sequence", op="attend", dtype="bf16", seqs=1, q_heads=32, kv_heads=32, dim=128,
             page=16, longest=8192, ragged=False, heads_first=False),
        # A serving batch: 64 sequences of very different lengths, four query heads to a key head.
        dict(name="attend_ragged_batch", op="attend", dtype="bf16", seqs=64, q_heads=32, kv_heads=8, dim=128,
             page=16, longest=8192, ragged=True, heads_first=False),
        # A few very long contexts, eight query heads to a key head, pages stored head by head.
        dict(name="attend_long_context", op="attend", dtype="bf16", seqs=4, q_heads=64, kv_heads=8, dim=128,
             page=64, longest=131072, ragged=False, heads_first=True),
        # f32 caches, pages that do not divide the tiles.
        dict(name="attend_f32", op="attend", dtype="f32", seqs=16, q_heads=16, kv_heads=16, dim=64, page=24,
             longest=2048, ragged=True, heads_first=False),
        # The decode step's answer: a handful of rows with their top alternatives.
        dict(name="logprobs_decode", op="logprobs", dtype="bf16", rows=8, classes=32000, top=5, masked=False,
             grad=False),
        # A training batch of 2 x 4096 tokens scored and differentiated.
        dict(name="logprobs_train", op="logprobs", dtype="bf16", rows=8192, classes=32000, top=0, masked=False,
             grad=True),
        # Scoring with alternatives over a large odd vocabulary, part of it masked out.
        dict(name="logprobs_score", op="logprobs", dtype="f32", rows=515, classes=131071, top=20, masked=True,
             grad=True),
        # One token through an MLP's first product.
        dict(name="w4_one_token", op="w4", dtype="bf16", rows=1, inner=2048, outer=8192, group=128, bias=True),
        # A decode batch through a large square product.
        dict(name="w4_batch", op="w4", dtype="bf16", rows=16, inner=8192, outer=8192, group=64, bias=False),
        # f32 activations, narrow output and a long inner axis.
        dict(name="w4_f32", op="w4", dtype="f32", rows=5, inner=8192, outer=2048, group=32, bias=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "logprobs", "w4"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op in ("append", "attend"):
        dim = rng.choice([32, 64, 80, 96, 128, 128, 256])
        kv = rng.choice([1, 2, 4, 5, 8, 16, 32])
        q = kv * rng.choice([g for g in (1, 2, 3, 4, 7, 8, 16) if g * kv <= 64])
        page = rng.choice([1, 8, 16, 24, 32, 64, 128])
        c = dict(op=op, dtype=dtype, q_heads=q, kv_heads=kv, dim=dim, page=page, heads_first=rng.random() < 0.5)
        if op == "append":
            tokens = _log(rng, 1, 8192)
            while tokens * (q + 2 * kv) * dim > 8192 * 96 * 128 // 2:
                tokens = max(1, tokens // 2)
            return dict(c, tokens=tokens, seqs=rng.randint(1, min(tokens, 64)), far=_log(rng, 8192, 1048576))
        seqs = _log(rng, 1, 128)
        longest = _log(rng, 1, 131072)
        most = 4 * 131072 * 1024 // (2 if dtype == "f32" else 1)
        while seqs * (longest + page) * kv * dim > most or seqs * longest * q > 1 << 26:
            if seqs > 1:
                seqs = (seqs + 1) // 2
            else:
                longest = (longest + 1) // 2
        return dict(c, seqs=seqs, longest=longest, ragged=rng.random() < 0.7)
    if op == "logprobs":
        classes = _log(rng, 33, 200000)
        rows = _log(rng, 1, max(2, min(16384, 8192 * 32000 // classes // 4)))
        return dict(op=op, dtype=dtype, rows=rows, classes=classes, top=rng.choice([0, 1, 5, 20, 32]),
                    masked=rng.random() < 0.4, grad=rng.random() < 0.5)
    inner = _log(rng, 64, 16384)
    outer = min(_log(rng, 16, 32768), 8192 * 8192 // inner)
    return dict(op=op, dtype=dtype, rows=_log(rng, 1, 16), inner=inner, outer=outer,
                group=rng.choice([32, 64, 128, 256]), bias=rng.random() < 0.5)


def _cache(case, gen, pages):
    """k and v caches indexed [page, slot, head, dim]; heads_first stores each page head by head."""
    dt = DTYPES[case["dtype"]]
    shape = (pages, case["page"], case["kv_heads"], case["dim"])
    if case["heads_first"]:
        shape = (pages, case["kv_heads"], case["page"], case["dim"])
    kv = [torch.randn(shape, generator=gen, device="cuda", dtype=dt) for _ in range(2)]
    return [t.transpose(1, 2) for t in kv] if case["heads_first"] else kv


def _table(gen, pages, seqs, columns):
    return torch.randperm(pages, generator=gen, device="cuda")[:seqs * columns].to(torch.int32).view(seqs, columns)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dt)

    op = case["op"]
    if op == "append":
        # Each sequence gets a run of consecutive positions, ending anywhere up to `far`. Only the pages
        # that hold new tokens are in memory: earlier table columns share page 0.
        T, n, D, page = case["tokens"], case["seqs"], case["dim"], case["page"]
        per = -(-T // n)
        room = max(case["far"], per)
        host = torch.Generator().manual_seed(seed)
        starts = (torch.rand(n, generator=host) * (room - per + 1)).long().clamp_(max=room - per)
        t = torch.arange(T)
        seq, pos = t // per, starts[t // per] + t % per
        columns = -(-room // page)
        used = -(-per // page) + 1
        table = torch.zeros(n, columns, dtype=torch.int32)
        perm = torch.randperm(n * used, generator=host).to(torch.int32).view(n, used) + 1
        cols = starts[:, None] // page + torch.arange(used)
        rows = torch.arange(n)[:, None].expand_as(cols)
        inside = cols < columns
        table[rows[inside], cols[inside]] = perm[inside]
        kc, vc = _cache(case, gen, n * used + 1)
        s = dict(q=normal(T, case["q_heads"], D), k=normal(T, case["kv_heads"], D), v=normal(T, case["kv_heads"], D),
                 seq=seq.to(torch.int32).cuda(), pos=pos.to(torch.int32).cuda(), kc=kc, vc=vc, table=table.cuda())
    elif op == "attend":
        n, page, longest = case["seqs"], case["page"], case["longest"]
        host = torch.Generator().manual_seed(seed)
        lens = torch.full((n,), longest)
        if case["ragged"]:
            lens = torch.exp(torch.rand(n, generator=host) * math.log(longest + 1)).long().clamp_(1, longest)
            lens[int(torch.randint(n, (1,), generator=host))] = longest
        columns = -(-longest // page)
        pages = n * columns + 3
        kc, vc = _cache(case, gen, pages)
        s = dict(q=normal(n, case["q_heads"], case["dim"]), kc=kc, vc=vc, table=_table(gen, pages, n, columns),
                 lens=lens.to(torch.int32).cuda(), longest=int(lens.max()), scale=case["dim"] ** -0.5)
    elif op == "logprobs":
        R, V = case["rows"], case["classes"]
        logits = normal(R, V).mul_(2.5)
        if case["masked"]:
            logits.masked_fill_(torch.rand(1, V, generator=gen, device="cuda") < 0.25, float("-inf"))
            logits[:, 0] = 1.0
        # The given tokens are likely ones, as tokens that were drawn from the model are.
        targets = torch.randint(V, (R, 4), generator=gen, device="cuda")
        best = logits.gather(1, targets).argmax(1, keepdim=True)
        targets = targets.gather(1, best)
        targets = torch.where(logits.gather(1, targets) == float("-inf"), 0, targets)
        s = dict(logits=logits, targets=targets.squeeze(1).to(torch.int32),
                 g_logprob=torch.randn(R, generator=gen, device="cuda"),
                 g_entropy=torch.randn(R, generator=gen, device="cuda"))
    else:
        K, M, G = case["inner"], case["outer"], case["group"]
        # 8 weights of a column, four bits each with the first in the lowest ones, to a word.
        s = dict(x=normal(case["rows"], K), group=G,
                 packed=torch.randint(-2**31, 2**31, (-(-K // 8), M), generator=gen, device="cuda").to(torch.int32),
                 scales=(torch.rand(-(-K // G), M, generator=gen, device="cuda") * 0.01 + 0.002).to(dt),
                 bias=normal(M) if case["bias"] else None)
    s.update(case=case)
    if own and op in ("append", "attend"):
        import haelixe_b200 as hx

        s["cache"] = hx.PagedKVCache(s["kc"], s["vc"], s["table"])
    return s


def _rotate(x, angles):
    c, n = torch.cos(angles).to(torch.float32)[:, None], torch.sin(angles).to(torch.float32)[:, None]
    a, b = x.float()[..., 0::2], x.float()[..., 1::2]
    return torch.stack((a * c - b * n, a * n + b * c), -1).flatten(-2).to(x.dtype)


def _angles(positions, dim):
    i = torch.arange(0, dim, 2, device=positions.device, dtype=torch.float64)
    return positions.double()[:, None] * ROPE_BASE ** (-i / dim)


def _plain_append(s):
    page = s["case"]["page"]
    pos, seq = s["pos"].long(), s["seq"].long()
    angles = _angles(pos, s["case"]["dim"])
    at = s["table"][seq, pos // page].long()
    s["kc"][at, pos % page] = _rotate(s["k"], angles)
    s["vc"][at, pos % page] = s["v"]
    return dict(q=_rotate(s["q"], angles), k_cache=s["kc"], v_cache=s["vc"])


def _plain_attend(s):
    kc, vc, q, page = s["kc"], s["vc"], s["q"].float(), s["case"]["page"]
    n, hq, d = q.shape
    hk = kc.shape[2]
    j = torch.arange(s["longest"], device=q.device)
    at = s["table"][:, j // page].long()
    k, v = kc[at, j % page].float(), vc[at, j % page].float()  # [n, longest, hk, d]
    scores = torch.einsum("nhgd,nlhd->nhgl", q.view(n, hk, hq // hk, d), k) * s["scale"]
    scores = scores.masked_fill((j >= s["lens"][:, None])[:, None, None], float("-inf"))
    lse = torch.logsumexp(scores, -1)
    o = torch.einsum("nhgl,nlhd->nhgd", torch.exp(scores - lse[..., None]), v)
    return dict(o=o.reshape(n, hq, d).to(s["q"].dtype), lse=lse.reshape(n, hq))


def _order(x):
    """Integers in the order of the values, ties to the lower index, in the last axis."""
    b = (x + 0.0).view(torch.int32).long()
    b = torch.where(b < 0, -(b & 0x7FFFFFFF), b)
    return (b << 32) | (0xFFFFFFFF - torch.arange(x.shape[-1], device=x.device))


def _plain_logprobs(s):
    x, t = s["logits"].float(), s["targets"].long()[:, None]
    top = s["case"]["top"]
    lse = torch.logsumexp(x, -1, keepdim=True)
    logp = x - lse
    p = torch.exp(logp)
    plogp = torch.where(p > 0, p * logp, 0.0)
    entropy = -plogp.sum(-1)
    out = dict(logprob=logp.gather(1, t).squeeze(1), entropy=entropy)
    if top:
        ids = 0xFFFFFFFF - (torch.topk(_order(x), top).values & 0xFFFFFFFF)
        out.update(top_ids=ids.to(torch.int32), top_logprobs=logp.gather(1, ids))
    if s["case"]["grad"]:
        gl, gh = s["g_logprob"][:, None], s["g_entropy"][:, None]
        d = -gl * p - gh * (plogp + p * entropy[:, None])
        d.scatter_add_(1, t, gl)
        out.update(dlogits=d.to(s["logits"].dtype))
    return out


def _plain_w4(s):
    K = s["x"].shape[1]
    shifts = torch.arange(0, 32, 4, device="cuda", dtype=torch.int32)[None, :, None]
    q = ((s["packed"][:, None] >> shifts) & 15).flatten(0, 1)[:K]
    w = (q - 8).float() * s["scales"].float().repeat_interleave(s["group"], 0)[:K]
    y = s["x"].float() @ w
    return (y if s["bias"] is None else y + s["bias"].float()).to(s["x"].dtype)


def run(s):
    op = s["case"]["op"]
    if own:
        import haelixe_b200 as hx

        if op == "append":
            q = hx.paged_append(s["cache"], s["k"], s["v"], s["seq"], s["pos"], rope_base=ROPE_BASE, q=s["q"])
            return dict(q=q, k_cache=s["kc"], v_cache=s["vc"])
        if op == "attend":
            o, lse = hx.paged_attention(s["cache"], s["q"], s["lens"], s["scale"])
            return dict(o=o, lse=lse)
        if op == "logprobs":
            x = s["logits"].detach().requires_grad_(s["case"]["grad"])
            r = hx.nn.token_logprobs(x, s["targets"], s["case"]["top"])
            out = dict(logprob=r.logprob, entropy=r.entropy)
            if s["case"]["top"]:
                out.update(top_ids=r.top_ids, top_logprobs=r.top_logprobs)
            if s["case"]["grad"]:
                out.update(dlogits=torch.autograd.grad([r.logprob, r.entropy], [x], [s["g_logprob"], s["g_entropy"]])[0])
            return out
        return hx.nn.linear_w4(s["x"], s["packed"], s["scales"], s["group"], s["bias"])
    return {"append": _plain_append, "attend": _plain_attend, "logprobs": _plain_logprobs, "w4": _plain_w4}[op](s)


def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "append":
        n = case["tokens"] * (case["q_heads"] + 2 * case["kv_heads"]) * case["dim"]
        return {"bytes": 2 * n * es + 12 * case["tokens"], "flops": 3 * n}
    if case["op"] == "attend":
        n, longest = case["seqs"], case["longest"]
        # The mean of a length whose logarithm is uniform, and one sequence at the longest.
        mean = longest / math.log(longest + 1) if case["ragged"] else longest
        keys = longest + (n - 1) * mean
        per_head = 2 * case["dim"] * es + 4
        return {"bytes": int(keys * (2 * case["kv_heads"] * case["dim"] * es + 4 / case["page"]) +
                             n * case["q_heads"] * per_head),
                "flops": int(4 * keys * case["q_heads"] * case["dim"])}
    if case["op"] == "logprobs":
        n = case["rows"] * case["classes"]
        # Forward: one read. Backward: the logits read again, their gradient written.
        return {"bytes": n * es * (3 if case["grad"] else 1) + case["rows"] * (12 + 8 * case["top"]),
                "flops": n * (10 if case["grad"] else 5)}
    K, M = case["inner"], case["outer"]
    return {"bytes": K * M // 2 + -(-K // case["group"]) * M * es + case["rows"] * (K + M) * es,
            "flops": 2 * case["rows"] * K * M}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        pos, dim = s["pos"].double(), case["dim"]
        freq = torch.exp(torch.arange(dim // 2, device="cuda", dtype=torch.float64) * (-2.0 / dim * math.log(ROPE_BASE)))
        turn = torch.polar(torch.ones((), device="cuda", dtype=torch.float64), pos[:, None] * freq)[:, None]

        def spun(x):
            z = torch.view_as_complex(x.double().unflatten(-1, (-1, 2)).contiguous())
            return torch.view_as_real(z * turn).flatten(-2)

        kc, vc = s["kc"].double(), s["vc"].double()
        where = s["table"].long()[s["seq"].long(), s["pos"].long() // case["page"]], s["pos"].long() % case["page"]
        kc.index_put_(where, spun(s["k"]))
        vc.index_put_(where, s["v"].double())
        return dict(q=spun(s["q"]), k_cache=kc, v_cache=vc)
    if case["op"] == "attend":
        n, hq, d = s["q"].shape
        hk = case["kv_heads"]
        o = torch.zeros(n, hq, d, dtype=torch.float64, device="cuda")
        lse = torch.full((n, hq), -math.inf, dtype=torch.float64, device="cuda")
        for i, length in enumerate(s["lens"].tolist()):
            pages = s["table"][i, :-(-length // case["page"])].long()
            for h in range(hk):
                k = s["kc"][pages, :, h].double().flatten(0, 1)[:length]
                v = s["vc"][pages, :, h].double().flatten(0, 1)[:length]
                mine = slice(h * (hq // hk), (h + 1) * (hq // hk))
                scores = s["q"][i, mine].double() @ k.T * s["scale"]
                o[i, mine] = torch.softmax(scores, -1) @ v
                lse[i, mine] = torch.logsumexp(scores, -1)
        return dict(o=o, lse=lse)
    if case["op"] == "logprobs":
        top, parts = case["top"], []
        for r in range(0, case["rows"], 512):
            x = s["logits"][r:r + 512].double()
            t = s["targets"][r:r + 512].long()[:, None]
            x = x - x.amax(1, keepdim=True)
            z = torch.exp(x)
            total = z.sum(1, keepdim=True)
            p = z / total
            surprise = torch.where(p > 0, torch.log(total) - x, 0.0)
            entropy = (p * surprise).sum(1, keepdim=True)
            part = dict(logprob=x.gather(1, t).squeeze(1) - torch.log(total).squeeze(1), entropy=entropy.squeeze(1))
            if top:
                part.update(top_logprobs=x.topk(top).values - torch.log(total))
            if case["grad"]:
                gl, gh = (s[g][r:r + 512].double()[:, None] for g in ("g_logprob", "g_entropy"))
                d = p * (gh * (surprise - entropy) - gl)
                part.update(dlogits=d.scatter_add(1, t, gl))
            parts.append(part)
        out = {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
        return dict(out, top_ids=None) if top else out
    K, G = case["inner"], case["group"]
    y = torch.zeros(case["rows"], case["outer"], dtype=torch.float64, device="cuda")
    x = s["x"].double()
    for j in range(8):  # the weights in nibble j of each word
        x_j = x[:, j::8]
        q = (s["packed"][:x_j.shape[1]].long() >> (4 * j)) & 15
        k = torch.arange(j, K, 8, device="cuda")
        y += x_j @ ((q - 8).double() * s["scales"].double()[k // G])
    return y if s["bias"] is None else y + s["bias"].double()
