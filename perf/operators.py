"""The operators of cached generation and scoring: appending keys and values
to a paged cache, attention of a batch that shares a prefix in that cache, and
the log probabilities of given tokens with their VJP.

`run` computes them in plain torch arithmetic (float32, rounded once at the
end) or, where `own` is true, through the library's C entry points. Sizes are
those of this repository's models (nanoGPT-char: 6 heads of 64, GPT-2-small:
12 heads of 64, 50304 tokens) and generic grouped-query ones (32 query heads
on 8 key heads of 128).
"""
import math

import numpy as np
import torch

own = False

ELEM = {"f32": 0x21000020, "bf16": 0x22000010}
DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16}
ROTARY = {"none": 0, "halves": 1, "pairs": 2}


def listed():
    return [
        # one decode step of four nanoGPT-char answers: call latency
        dict(name="append_step", op="append", dtype="bf16", n=4, seqs=4, hq=6, hkv=6, hd=64, page=16, rotary="none",
             rot=0, base=200, longest=56),
        # the keys and values of one long prompt going into the cache at once
        dict(name="append_prompt", op="append", dtype="bf16", n=16384, seqs=1, hq=32, hkv=8, hd=128, page=64,
             rotary="halves", rot=128, base=0, longest=16384),
        # one decode step of four nanoGPT-char answers to one prompt: call latency
        dict(name="attend_step", op="attend", dtype="bf16", b=4, tq=1, hq=6, hkv=6, hd=64, page=16, prefix=200,
             longest=56, scale=0.125),
        # a few hundred tokens into 64 answers to one long prompt
        dict(name="attend_answers", op="attend", dtype="bf16", b=64, tq=1, hq=32, hkv=8, hd=128, page=16, prefix=8192,
             longest=512, scale=0.08838834764831845),
        # eight answers about a very long document: reading the shared keys bounds it
        dict(name="attend_document", op="attend", dtype="bf16", b=8, tq=1, hq=32, hkv=8, hd=128, page=64,
             prefix=131072, longest=2048, scale=0.08838834764831845),
        # a large batch on one prompt: the products over the shared keys bound it
        dict(name="attend_batch", op="attend", dtype="bf16", b=512, tq=1, hq=32, hkv=8, hd=128, page=16, prefix=16384,
             longest=256, scale=0.08838834764831845),
        # 24 different questions of up to 37 tokens read in one pass behind a common prompt (GPT-2-small's heads,
        # pages that end inside tiles)
        dict(name="attend_questions", op="attend", dtype="bf16", b=24, tq=37, hq=12, hkv=12, hd=64, page=24,
             prefix=777, longest=128, scale=0.125),
        # the same in float32, two tokens a sequence
        dict(name="attend_f32", op="attend", dtype="f32", b=5, tq=2, hq=12, hkv=12, hd=64, page=24, prefix=777,
             longest=130, scale=0.125),
        # scoring one drawn token of each of four answers, with five alternatives
        dict(name="score_step", op="score", dtype="bf16", rows=4, v=50304, ld=50304, k=5, temperature=0.8),
        # scoring a whole GPT-2-small batch (8 x 1024 tokens)
        dict(name="score_batch", op="score", dtype="bf16", rows=8192, v=50304, ld=50304, k=8, temperature=1.0),
        # its VJP for a policy-gradient step on half of that batch
        dict(name="score_grad", op="score_grad", dtype="bf16", rows=4096, v=50304, ld=50304, temperature=1.0),
        # float32 logits of an unpadded vocabulary, odd row count
        dict(name="score_grad_f32", op="score_grad", dtype="f32", rows=1023, v=50257, ld=50264, temperature=0.7),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(case):
    w = work(case)
    rate = 60e12 if case["dtype"] == "f32" else 1.5e15
    return max(w["bytes"] / 6.5e12, w["flops"] / rate)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["append", "attend", "attend", "score", "score_grad"])
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        hkv = rng.choice([1, 2, 4, 6, 8, 12])
        hq = hkv * rng.choice([1, 1, 2, 4, 8])
        hd = rng.choice([32, 64, 64, 128, 128])
        page = rng.choice([8, 16, 24, 32, 64, 128])
        if op == "append":
            n = _log_int(rng, 1, 16384)
            rotary = rng.choice(["none", "halves", "pairs"])
            base = rng.choice([0, _log_int(rng, 1, 8192)])
            seqs = _log_int(rng, 1, n)
            case = dict(op=op, dtype=dtype, n=n, seqs=seqs, hq=hq, hkv=hkv, hd=hd, page=page, rotary=rotary,
                        rot=0 if rotary == "none" else rng.choice([hd, hd, hd // 2]), base=base,
                        longest=n // seqs + 1 + rng.randrange(100))
        elif op == "attend":
            tq = rng.choice([1, 1, 1, 2, _log_int(rng, 3, 200)])
            b = _log_int(rng, 1, 512)
            case = dict(op=op, dtype=dtype, b=b, tq=tq, hq=hq, hkv=hkv, hd=hd, page=page,
                        prefix=rng.choice([0, _log_int(rng, 1, 131072), _log_int(rng, 100, 32768)]),
                        longest=tq + _log_int(rng, 1, 2048), scale=rng.choice([1.0, 0.7]) / math.sqrt(hd))
            keys = case["prefix"] + case["longest"]
            if 4.0 * b * tq * hq * keys > 8e9 or 8.0 * b * case["longest"] * hkv * hd > 8e9:
                continue  # the plain form's scores and gathered keys have to fit the card
        else:
            v = _log_int(rng, 40, 200000)
            rows = _log_int(rng, 1, 8192)
            case = dict(op=op, dtype=dtype, rows=rows, v=v, ld=v + rng.choice([0, 0, rng.randrange(1, 64)]),
                        temperature=rng.choice([1.0, 0.8, 1.3]))
            if op == "score":
                case["k"] = rng.choice([0, 1, 5, 8, 20, 32])
            if rows * v > 4.2e8:
                continue
        if _cost(case) <= most:
            return case


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 17)
    return g


def _randn(shape, dtype, g, scale=1.0):
    return (torch.randn(shape, device="cuda", dtype=torch.float32, generator=g) * scale).to(dtype)


def _pages(count, per_seq, g):
    """`count` sequences' page tables and the number of pages: a shuffled pool, as a cache in use has."""
    n = max(1, count * per_seq)
    return torch.randperm(n, device="cuda", generator=g)[:count * per_seq].to(torch.int32), n


def _lens(case, seed):
    """Ragged lengths between tq and `longest`; in larger batches one slot is idle (-1) and one holds nothing new."""
    r = np.random.default_rng(int(seed) + 101)
    lens = r.integers(min(case["tq"], case["longest"]), case["longest"] + 1, case["b"]).astype(np.int32)
    lens[0] = case["longest"]
    if case["b"] >= 16:
        lens[3] = -1
        lens[5] = 0
    return lens


def _append_tokens(case, seed):
    """Sequence and position of each token: the new tokens of `seqs` sequences in order; with 64 tokens or more the
    last one is padding (sequence -1)."""
    n, seqs = case["n"], case["seqs"]
    r = np.random.default_rng(int(seed) + 202)
    seq = np.sort(np.arange(n) % seqs)
    counts = np.bincount(seq, minlength=seqs)
    start = r.integers(0, case["longest"] - counts.max() + 1, seqs)
    first = np.concatenate([[0], np.cumsum(counts)[:-1]])
    pos = case["base"] + start[seq] + (np.arange(n) - first[seq])
    if n >= 64:
        seq[-1] = -1
    return seq.astype(np.int32), pos.astype(np.int32)


def _angles(n_pos, rot):
    inv = 10000.0 ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)
    a = np.arange(n_pos, dtype=np.float64)[:, None] * inv[None]
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def prepare(case, seed):
    g = _generator(seed)
    dt = DTYPE[case["dtype"]]
    st = dict(case=dict(case))
    if case["op"] == "append":
        per_seq = -(-case["longest"] // case["page"])
        table, n_pages = _pages(case["seqs"], per_seq, g)
        st["table"] = table.view(case["seqs"], per_seq)
        st["k"] = _randn((n_pages, case["page"], case["hkv"], case["hd"]), dt, g)
        st["v"] = _randn((n_pages, case["page"], case["hkv"], case["hd"]), dt, g)
        st["qkv"] = _randn((case["n"], (case["hq"] + 2 * case["hkv"]) * case["hd"]), dt, g)
        seq, pos = _append_tokens(case, seed)
        st["seq"], st["pos"] = torch.from_numpy(seq).cuda(), torch.from_numpy(pos).cuda()
        st["n_pos"] = case["base"] + case["longest"]
        if case["rot"]:
            cos, sin = _angles(st["n_pos"], case["rot"])
            st["cos"], st["sin"] = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()
        st["q_out"] = torch.empty(case["n"], case["hq"] * case["hd"], device="cuda", dtype=dt)
    elif case["op"] == "attend":
        per_seq = -(-case["longest"] // case["page"])
        n_prefix = -(-case["prefix"] // case["page"])
        table, n_pages = _pages(1, case["b"] * per_seq + n_prefix, g)
        st["prefix_table"] = table[:n_prefix].contiguous()
        st["table"] = table[n_prefix:].reshape(case["b"], per_seq).contiguous()
        st["k"] = _randn((n_pages, case["page"], case["hkv"], case["hd"]), dt, g)
        st["v"] = _randn((n_pages, case["page"], case["hkv"], case["hd"]), dt, g)
        # a factor of 2 on the queries: scores that pick some keys out, as trained heads do
        st["q"] = _randn((case["b"] * case["tq"], case["hq"] * case["hd"]), dt, g, 2.0)
        st["lens"] = torch.from_numpy(_lens(case, seed)).cuda()
        st["out"] = torch.empty_like(st["q"])
        st["lse"] = torch.empty(case["b"] * case["tq"], case["hq"], device="cuda", dtype=torch.float32)
    else:
        rows, v, ld = case["rows"], case["v"], case["ld"]
        x = torch.empty(rows, ld, device="cuda", dtype=dt)
        for r0 in range(0, rows, 1024):
            x[r0:r0 + 1024] = _randn((min(1024, rows - r0), ld), dt, g, 2.0)
        # a model that is sure of some rows, and a few tokens that decoding has banned
        hot = torch.randint(0, v, (rows,), device="cuda", generator=g)
        x[torch.arange(rows, device="cuda"), hot] += (torch.arange(rows, device="cuda") % 5 * 3).to(dt)
        x[::7, torch.randint(0, v, (min(3, v - 1),), device="cuda", generator=g)] = -math.inf
        st["x"] = x
        target = torch.randint(0, v, (rows,), device="cuda", generator=g)
        target = torch.where(torch.arange(rows, device="cuda") % 2 == 0, hot, target).float()
        if rows >= 16:
            target[3] = -1.0  # a padded position
        st["target"] = target
        f = dict(device="cuda", dtype=torch.float32)
        if case["op"] == "score":
            st["logp"], st["entropy"], st["lse"] = (torch.empty(rows, **f) for _ in range(3))
            if case["k"]:
                st["top_ids"] = torch.empty(rows, case["k"], device="cuda", dtype=torch.int32)
                st["top_logp"] = torch.empty(rows, case["k"], **f)
        else:
            z = torch.empty(rows, **f)
            ent = torch.empty(rows, **f)
            for r0 in range(0, rows, 1024):
                zz = x[r0:r0 + 1024, :v].double() / case["temperature"]
                l = torch.logsumexp(zz, 1)
                lp = zz - l[:, None]
                ent[r0:r0 + 1024] = -(lp.exp() * lp.clamp_min(-1e4)).sum(1).float()
                z[r0:r0 + 1024] = l.float()
            st["lse"], st["entropy"] = z, ent
            st["dlogp"] = torch.randn(rows, generator=g, **f)
            st["dentropy"] = torch.randn(rows, generator=g, **f) * 0.1
            st["dx"] = torch.zeros(rows, ld, device="cuda", dtype=dt)
    return st


# ---- the library's calls ---------------------------------------------------


def _cache(st):
    """The cache's description, which a program makes once beside the cache."""
    if "cache" not in st:
        from sheaf_b200 import KvCache

        c = st["case"]
        st["cache"] = KvCache(st["k"].data_ptr(), st["v"].data_ptr(), st["k"].stride(0), st["k"].stride(1),
                              st["k"].stride(2), st["k"].shape[0], c["page"], c["hkv"], c["hd"], ELEM[c["dtype"]])
    return st["cache"]


def _own(st):
    import sheaf_b200

    L = sheaf_b200.lib()
    c = st["case"]
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "append":
        cos, sin = (st["cos"].data_ptr(), st["sin"].data_ptr()) if c["rot"] else (None, None)
        rc = L.sb_op_kv_append(_cache(st), st["qkv"].data_ptr(), st["qkv"].stride(0), c["n"], c["hq"],
                               st["q_out"].data_ptr(), st["q_out"].stride(0), st["seq"].data_ptr(),
                               st["pos"].data_ptr(), c["base"], st["table"].data_ptr(), c["seqs"],
                               st["table"].shape[1], ROTARY[c["rotary"]], c["rot"], cos, sin, st["n_pos"], stream)
        out = dict(q=st["q_out"], k=st["k"], v=st["v"])
    elif c["op"] == "attend":
        cache = _cache(st)
        if "workspace" not in st:
            size = L.sb_op_prefix_attention_workspace_size(cache, c["b"], c["tq"], c["hq"], c["prefix"],
                                                           st["table"].shape[1])
            st["workspace"] = torch.empty(max(1, size), device="cuda", dtype=torch.uint8)
        rc = L.sb_op_prefix_attention(cache, st["q"].data_ptr(), st["q"].stride(0), st["out"].data_ptr(),
                                      st["out"].stride(0), st["lse"].data_ptr(), c["b"], c["tq"], c["hq"], c["scale"],
                                      st["prefix_table"].data_ptr(), c["prefix"], st["table"].data_ptr(),
                                      st["table"].shape[1], st["lens"].data_ptr(), st["workspace"].data_ptr(),
                                      st["workspace"].numel(), stream)
        out = dict(out=st["out"], lse=st["lse"])
    elif c["op"] == "score":
        ids, alt = (st["top_ids"].data_ptr(), st["top_logp"].data_ptr()) if c["k"] else (None, None)
        rc = L.sb_op_token_logprobs(ELEM[c["dtype"]], st["x"].data_ptr(), c["ld"], c["rows"], c["v"],
                                    st["target"].data_ptr(), c["temperature"], st["logp"].data_ptr(),
                                    st["entropy"].data_ptr(), st["lse"].data_ptr(), c["k"], ids, alt, stream)
        out = {n: st[n] for n in ("logp", "entropy", "lse", "top_ids", "top_logp") if n in st}
    else:
        rc = L.sb_op_token_logprobs_bwd(ELEM[c["dtype"]], st["x"].data_ptr(), c["ld"], c["rows"], c["v"],
                                        st["target"].data_ptr(), c["temperature"], st["lse"].data_ptr(),
                                        st["entropy"].data_ptr(), st["dlogp"].data_ptr(), st["dentropy"].data_ptr(),
                                        st["dx"].data_ptr(), c["ld"], stream)
        out = dict(dx=st["dx"])
    if rc:
        raise RuntimeError(f"{c['op']} failed with {rc}")
    return out


# ---- the plain forms -------------------------------------------------------


def _rotate(x, cos, sin, how, rot):
    """x [n, heads, hd] with the first `rot` values of each head rotated; cos, sin [n, 1, rot / 2]."""
    if not rot:
        return x
    if how == "halves":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def _plain_append(st):
    c = st["case"]
    n, hq, hkv, hd = c["n"], c["hq"], c["hkv"], c["hd"]
    x = st["qkv"].float().view(n, hq + 2 * hkv, hd)
    live = st["seq"] >= 0
    pos = st["pos"].long()
    cos = st["cos"][pos][:, None] if c["rot"] else None
    sin = st["sin"][pos][:, None] if c["rot"] else None
    turned = _rotate(x[:, :hq + hkv], cos, sin, c["rotary"], c["rot"])
    q = torch.where(live[:, None, None], turned[:, :hq], 0.0)
    own_pos = pos - c["base"]
    page = st["table"].long()[st["seq"].clamp_min(0).long(), own_pos // c["page"]]
    slot = (page * c["page"] + own_pos % c["page"])[live]
    st["k"].view(-1, hkv, hd)[slot] = turned[:, hq:][live].to(st["k"].dtype)
    st["v"].view(-1, hkv, hd)[slot] = x[:, hq + hkv:][live].to(st["v"].dtype)
    return dict(q=q.reshape(n, hq * hd).to(st["qkv"].dtype), k=st["k"], v=st["v"])


def _plain_attend(st):
    c = st["case"]
    b, tq, hq, hkv, hd, page, prefix = (c[k] for k in ("b", "tq", "hq", "hkv", "hd", "page", "prefix"))
    group, own_keys = hq // hkv, st["table"].shape[1] * page
    q = st["q"].float().view(b, tq, hkv, group, hd)
    at = torch.arange(prefix, device="cuda")
    slots = st["prefix_table"].long()[at // page] * page + at % page
    kp = st["k"].view(-1, hkv, hd)[slots].float()
    vp = st["v"].view(-1, hkv, hd)[slots].float()
    ks = st["k"][st["table"].long()].float().view(b, own_keys, hkv, hd)
    vs = st["v"][st["table"].long()].float().view(b, own_keys, hkv, hd)
    rows = q.permute(2, 0, 1, 3, 4).reshape(hkv, b * tq * group, hd)
    s_prefix = torch.matmul(rows, kp.permute(1, 2, 0)).view(hkv, b, tq, group, prefix)
    per_seq = q.permute(2, 0, 1, 3, 4).reshape(hkv, b, tq * group, hd)
    s_own = torch.matmul(per_seq, ks.permute(2, 0, 3, 1)).view(hkv, b, tq, group, own_keys)
    s = torch.cat([s_prefix, s_own], -1).mul_(c["scale"])
    # the last of a row's keys, counted from the prefix's first
    lens = st["lens"].long()
    last = prefix + lens[:, None] - tq + torch.arange(tq, device="cuda")[None]
    last = torch.where(lens[:, None] < 0, -1, last)
    seen = torch.arange(prefix + own_keys, device="cuda") <= last[..., None]
    s.masked_fill_(~seen[None, :, :, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p[..., :prefix].reshape(hkv, b * tq * group, prefix), vp.permute(1, 0, 2))
    o = o.view(hkv, b, tq, group, hd)
    o = o + torch.matmul(p[..., prefix:].reshape(hkv, b, tq * group, own_keys),
                         vs.permute(2, 0, 1, 3)).view(hkv, b, tq, group, hd)
    o = torch.where(total > 0, o / total, 0.0)
    lse = (m + total.log())[..., 0]
    return dict(out=o.permute(1, 2, 0, 3, 4).reshape(b * tq, hq * hd).to(st["q"].dtype),
                lse=lse.permute(1, 2, 0, 3).reshape(b * tq, hq))


def _plain_score(st):
    c = st["case"]
    x = st["x"][:, :c["v"]].float()
    z = x / c["temperature"]
    m = z.amax(1, keepdim=True)
    d = z - m
    e = d.exp()
    total = e.sum(1)
    log_total = total.log()
    lse = m[:, 0] + log_total
    entropy = log_total - (e * torch.where(e > 0, d, 0.0)).sum(1) / total
    t = st["target"]
    known = (t >= 0) & (t < c["v"]) & (t == t.floor())
    at = torch.where(known, t, 0.0).long()[:, None]
    logp = torch.where(known, d.gather(1, at)[:, 0] - log_total, 0.0)
    out = dict(logp=logp, entropy=entropy, lse=lse)
    if c["k"]:
        # order by value, then by the lower index: the float's bits as an ordered integer over the reversed index
        bits = (x + 0.0).view(torch.int32).long()
        order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        index = torch.arange(c["v"], device="cuda")
        best = ((order << 20) + (c["v"] - 1 - index)).topk(c["k"], dim=1).values
        ids = c["v"] - 1 - (best & 0xFFFFF)
        out["top_ids"] = ids.int()
        out["top_logp"] = d.gather(1, ids) - log_total[:, None]
    return out


def _plain_score_grad(st):
    c = st["case"]
    v = c["v"]
    z = st["x"][:, :v].float() / c["temperature"]
    lp = z - st["lse"][:, None]
    p = lp.exp()
    t = st["target"]
    known = (t >= 0) & (t < v) & (t == t.floor())
    g = torch.where(known, st["dlogp"], 0.0)[:, None]
    h = st["dentropy"][:, None]
    dz = -p * (g + h * (lp.clamp_min(-1e30) + st["entropy"][:, None]))
    dz.scatter_add_(1, torch.where(known, t, 0.0).long()[:, None], g)
    dx = torch.zeros_like(st["x"])
    dx[:, :v] = (dz / c["temperature"]).to(dx.dtype)
    return dict(dx=dx)


def run(state):
    if own:
        return _own(state)
    return {"append": _plain_append, "attend": _plain_attend, "score": _plain_score,
            "score_grad": _plain_score_grad}[state["case"]["op"]](state)


# ---- what a pass cannot do without -----------------------------------------


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "append":
        values = case["n"] * (case["hq"] + 2 * case["hkv"]) * case["hd"]
        return {"bytes": 2 * values * e + case["n"] * (8 + 4 * case["rot"]), "flops": 3 * values}
    if case["op"] == "attend":
        b, tq, hq, hkv, hd = (case[k] for k in ("b", "tq", "hq", "hkv", "hd"))
        keys = b * (min(tq, case["longest"]) + case["longest"]) / 2  # the lengths are uniform between the two
        kv = 2 * (case["prefix"] + keys) * hkv * hd * e
        seen = tq * (b * case["prefix"] + keys) - b * tq * (tq - 1) / 2
        return {"bytes": int(kv + 2 * b * tq * hq * hd * e + 4 * b * tq * hq), "flops": int(4 * hq * hd * seen)}
    values = case["rows"] * case["v"]
    if case["op"] == "score":
        return {"bytes": values * e + case["rows"] * (16 + 8 * case["k"]), "flops": 5 * values}
    return {"bytes": 2 * values * e + case["rows"] * 20, "flops": 6 * values}


# ---- the definitions in 64 bits --------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, st)
    if case["op"] == "attend":
        return _exact_attend(case, st)
    rows, v, T = case["rows"], case["v"], case["temperature"]
    found = []
    for r in range(0, rows, 512):
        z = st["x"][r:r + 512, :v].double() / T
        lp = torch.log_softmax(z, 1)
        t = st["target"][r:r + 512]
        one = torch.zeros_like(z)
        inside = torch.nonzero((t >= 0) & (t < v) & (t % 1 == 0))[:, 0]
        one[inside, t[inside].long()] = 1.0
        plogp = torch.special.xlogy(lp.exp(), lp.exp())
        if case["op"] == "score":
            logp = torch.zeros(z.shape[0], dtype=torch.float64, device=z.device)
            logp[inside] = lp[inside, t[inside].long()]
            part = [logp, -plogp.sum(1), torch.logsumexp(z, 1)]
            if case["k"]:
                part.append(lp.sort(1, descending=True).values[:, :case["k"]])
            found.append(part)
        else:
            g = st["dlogp"][r:r + 512, None].double() * one.sum(1, keepdim=True)
            h = st["dentropy"][r:r + 512, None].double()
            entropy = -plogp.sum(1, keepdim=True)
            found.append([(g * (one - lp.exp()) - h * (plogp + lp.exp() * entropy)) / T])
    cols = [torch.cat(x) for x in zip(*found)]
    if case["op"] == "score_grad":
        dx = torch.zeros(rows, case["ld"], dtype=torch.float64, device="cuda")
        dx[:, :v] = cols[0]
        return dict(dx=dx)
    out = dict(zip(("logp", "entropy", "lse"), cols))
    if case["k"]:
        out["top_ids"], out["top_logp"] = None, cols[3]
    return out


def _exact_append(case, st):
    hq, hkv, hd, rot = case["hq"], case["hkv"], case["hd"], case["rot"]
    k, v = st["k"].double(), st["v"].double()
    x = st["qkv"].double().view(case["n"], hq + 2 * hkv, hd)
    if rot:
        # the rotation as a product of complex numbers
        turn = torch.complex(st["cos"].double(), st["sin"].double())[st["pos"].long()][:, None]
        head = x[:, :hq + hkv, :rot]
        first, second = (head[..., :rot // 2], head[..., rot // 2:]) if case["rotary"] == "halves" else \
            (head[..., ::2], head[..., 1::2])
        r = torch.complex(first.contiguous(), second.contiguous()) * turn
        x = x.clone()
        if case["rotary"] == "halves":
            x[:, :hq + hkv, :rot // 2], x[:, :hq + hkv, rot // 2:rot] = r.real, r.imag
        else:
            x[:, :hq + hkv, 0:rot:2], x[:, :hq + hkv, 1:rot:2] = r.real, r.imag
    live = torch.nonzero(st["seq"] >= 0)[:, 0]
    at = st["pos"][live].long() - case["base"]
    page = st["table"][st["seq"][live].long(), at // case["page"]].long()
    k[page, at % case["page"]] = x[live, hq:hq + hkv]
    v[page, at % case["page"]] = x[live, hq + hkv:]
    q = torch.zeros(case["n"], hq * hd, dtype=torch.float64, device="cuda")
    q[live] = x[live, :hq].reshape(-1, hq * hd)
    return dict(q=q, k=k, v=v)


def _exact_attend(case, st):
    b, tq, hq, hkv, hd, page, prefix = (case[k] for k in ("b", "tq", "hq", "hkv", "hd", "page", "prefix"))
    if case["b"] * tq * hq * (prefix + case["longest"]) > 4e9:
        return None  # the scores in 64 bits take too long
    g = hq // hkv
    lens = st["lens"].tolist()
    out = torch.zeros(b, tq, hq, hd, dtype=torch.float64, device="cuda")
    lse = torch.full((b, tq, hq), -math.inf, dtype=torch.float64, device="cuda")
    flat_k, flat_v = st["k"].flatten(0, 1), st["v"].flatten(0, 1)
    rows_of = lambda table, n: (table[:-(-n // page)].long()[:, None] * page +  # noqa: E731
                                torch.arange(page, device="cuda")).flatten()[:n]
    shared = rows_of(st["prefix_table"], prefix)
    k0, v0 = flat_k[shared].double(), flat_v[shared].double()
    for s in range(b):
        if lens[s] < 0:
            continue
        mine = rows_of(st["table"][s], lens[s])
        k = torch.cat([k0, flat_k[mine].double()]).transpose(0, 1)
        v = torch.cat([v0, flat_v[mine].double()]).transpose(0, 1)
        q = st["q"][s * tq:(s + 1) * tq].double().view(tq, hkv, g, hd).permute(1, 0, 2, 3).reshape(hkv, tq * g, hd)
        z = (q @ k.transpose(1, 2)).view(hkv, tq, g, -1) * case["scale"]
        n = z.shape[-1]
        late = torch.arange(n, device="cuda")[None] > (n - tq + torch.arange(tq, device="cuda"))[:, None]
        z = z.masked_fill(late[None, :, None], -math.inf)
        l = torch.logsumexp(z, -1)
        p = torch.nan_to_num(torch.exp(z - l[..., None]), nan=0.0)
        o = (p.view(hkv, tq * g, n) @ v).view(hkv, tq, g, hd)
        out[s] = o.permute(1, 0, 2, 3).reshape(tq, hq, hd)
        lse[s] = l.permute(1, 0, 2).reshape(tq, hq)
    return dict(out=out.view(b * tq, hq * hd), lse=lse.view(b * tq, hq))
