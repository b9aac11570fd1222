"""Timed cases of four operators: attention over packed sequences, routing to experts, the stable
permutation of the routed slots by expert, and dropout with a residual whose mask is never stored.

``own = False`` computes them in their plain form out of elementary torch operations; ``own = True``
makes the calls of this package's kernels.  Together they are what a training step of a
mixture-of-experts decoder layer over packed documents needs beside the framework's GEMMs and norms.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"


def listed():
    return [
        # one short prompt through a 12-head layer: nothing but launch latency
        _attn("attention, one short prompt", train=False, tokens=37, docs=1, heads=12, kv_heads=12, dim=64, tail=0),
        # a batch of texts of different lengths through an encoder layer, no causal mask
        _attn("attention, ragged encoder batch", train=False, causal=False, tokens=4001, docs=13, heads=12, kv_heads=12,
              dim=64, tail=95),
        # long prompts of a grouped-query decoder with heads of 128, processed at once
        _attn("attention, long prompts", train=False, tokens=16384, docs=3, heads=32, kv_heads=8, dim=128, tail=0),
        # a packed microbatch of a 12-head decoder: many documents, forward and backward
        _attn("attention step, packed documents", train=True, tokens=4096, docs=11, heads=12, kv_heads=12, dim=64,
              tail=0),
        # a packed microbatch of a wide decoder with grouped queries, a few long documents
        _attn("attention step, long documents", train=True, tokens=8192, docs=5, heads=32, kv_heads=8, dim=128,
              tail=0),
        # generation: the router of a few single tokens
        _route("routing, single tokens", train=False, tokens=3, experts=64, topk=6, scoring="softmax", bias=False,
               groups=1, kept=1, renorm=True, fp32=False, width=0),
        # a microbatch with many small experts in groups, sigmoid scores and a balancing bias
        _route("routing, grouped experts", train=False, tokens=8192, experts=256, topk=8, scoring="sigmoid", bias=True,
               groups=8, kept=4, renorm=True, fp32=True, width=0),
        # a training step of the router: selection, then the gradient of its logits from the expert rows
        _route("routing step", train=True, tokens=4093, experts=64, topk=6, scoring="softmax", bias=False, groups=1,
               kept=1, renorm=True, fp32=False, width=1024),
        # the slots of a few generated tokens, sorted by expert
        _permute("permutation, few slots", slots=96, experts=64),
        # the slots of a large microbatch with many experts
        _permute("permutation, large microbatch", slots=32768 * 8, experts=256),
        # residual dropout of a small, odd microbatch
        _dropout("dropout step, small", rows=1021, width=768, p=0.1, fp32=False),
        # residual dropout of a large microbatch of a wide decoder
        _dropout("dropout step, large", rows=16384, width=4096, p=0.1, fp32=False),
    ]


def draw(rng):
    while True:
        kind = rng.choice(["attention", "attention", "route", "permute", "dropout"])
        if kind == "attention":
            tokens = _log(rng, 1, 16384)
            heads, kv = rng.choice([(12, 12), (16, 16), (16, 4), (32, 32), (32, 8), (8, 1), (5, 5)])
            case = _attn(None, train=rng.random() < 0.5, causal=rng.random() < 0.75, tokens=tokens,
                         docs=rng.randint(1, min(tokens, 40)), heads=heads, kv_heads=kv, dim=rng.choice([64, 128]),
                         tail=rng.choice([0, 0, 1, 70]), spread=rng.randint(1, 10 ** 6))
        elif kind == "route":
            groups = rng.choice([1, 1, 2, 4, 8])
            experts = groups * rng.randint(3, 512 // groups) if groups > 1 else _log(rng, 2, 512)
            kept = rng.randint(1, groups)
            topk = rng.randint(1, min(16, experts // groups * kept))
            train = rng.random() < 0.5
            case = _route(None, train=train, tokens=_log(rng, 1, 8192), experts=experts, topk=topk,
                          scoring=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, groups=groups, kept=kept,
                          renorm=rng.random() < 0.6, fp32=rng.random() < 0.5,
                          width=8 * rng.randint(8, 256) if train else 0)
        elif kind == "permute":
            case = _permute(None, slots=_log(rng, 1, 262144), experts=_log(rng, 2, 1024))
        else:
            case = _dropout(None, rows=_log(rng, 1, 16384), width=8 * _log(rng, 8, 512), fp32=rng.random() < 0.3,
                            p=rng.choice([0.05, 0.1, 0.2, 0.5]))
        most = {"flops": 0, "bytes": 0}
        for c in listed():
            if c["op"] == case["op"]:
                most = {k: max(most[k], work(c)[k]) for k in most}
        if all(work(case)[k] <= most[k] for k in most):
            return case


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _case(name, **values):
    return values if name is None else dict(values, name=name)


def _attn(name, *, train, tokens, docs, heads, kv_heads, dim, tail, causal=True, spread=7):
    return _case(name, op="attention", train=train, causal=causal, tokens=tokens, docs=docs, heads=heads,
                 kv_heads=kv_heads, dim=dim, tail=tail, spread=spread)


def _route(name, *, train, tokens, experts, topk, scoring, bias, groups, kept, renorm, fp32, width):
    return _case(name, op="route", train=train, tokens=tokens, experts=experts, topk=topk, scoring=scoring, bias=bias,
                 groups=groups, kept=kept, renorm=renorm, fp32=fp32, width=width)


def _permute(name, *, slots, experts):
    return _case(name, op="permute", slots=slots, experts=experts)


def _dropout(name, *, rows, width, p, fp32):
    return _case(name, op="dropout", rows=rows, width=width, p=p, fp32=fp32)


def _lengths(case):
    """Document lengths of a packed batch: log-normal shares of the tokens (short ones may round to zero)."""
    rng = random.Random(case["spread"])
    share = [math.exp(rng.gauss(0.0, 1.0)) for _ in range(case["docs"])]
    lens = [int(case["tokens"] * s / sum(share)) for s in share]
    lens[share.index(max(share))] += case["tokens"] - sum(lens)
    return lens


def work(case):
    op = case["op"]
    if op == "attention":
        H, G, D, T = case["heads"], case["kv_heads"], case["dim"], case["tokens"]
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in _lengths(case))
        q, kv, stat = 2 * T * H * D, 4 * T * G * D, 4 * T * H
        flops, moved = 4 * pairs * H * D, 2 * q + kv + stat
        if case["train"]:
            # the backward reads q, k, v, o, its gradient and the log-sum-exp, and writes dq, dk, dv
            flops, moved = flops + 10 * pairs * H * D, moved + 4 * q + 2 * kv + stat
        return {"bytes": moved, "flops": flops}
    if op == "route":
        T, E, K, C = case["tokens"], case["experts"], case["topk"], case["width"]
        logits = T * E * (4 if case["fp32"] else 2)
        moved, flops = logits + 8 * T * K + (4 * E if case["bias"] else 0), 4 * T * E
        if case["train"]:
            moved += 2 * logits + 2 * T * C * (K + 1) + 12 * T * K
            flops += 2 * T * K * C + 6 * T * E
        return {"bytes": moved, "flops": flops}
    if op == "permute":
        return {"bytes": 12 * case["slots"] + 4 * (case["experts"] + 1), "flops": case["slots"]}
    n = case["rows"] * case["width"]
    # 10 rounds of two 32 x 32 bit products for every 8 elements, in each direction
    return {"bytes": 5 * n * (4 if case["fp32"] else 2), "flops": 2 * n * 8}


# ---- inputs -----------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def randn(*shape, scale=1.0, dtype=torch.bfloat16):
        return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)

    s = dict(case=case)
    op = case["op"]
    if op == "attention":
        H, G, D = case["heads"], case["kv_heads"], case["dim"]
        rows = case["tokens"] + case["tail"]
        lens = _lengths(case)
        s["lens"] = lens
        s["cu"] = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=DEV)
        # q | k | v lie side by side, as a fused projection leaves them
        s["qkv"] = randn(rows, (H + 2 * G) * D)
        s["q"], s["k"], s["v"] = _heads(s["qkv"], H, G, D)
        s["o"] = torch.zeros(rows, H, D, dtype=torch.bfloat16, device=DEV)
        s["lse"] = torch.zeros(H, rows, dtype=torch.float32, device=DEV)
        if case["train"]:
            s["do"] = randn(rows, H, D, scale=0.1)
            s["dqkv"] = torch.zeros_like(s["qkv"])
            s["dq"], s["dk"], s["dv"] = _heads(s["dqkv"], H, G, D)
            s["delta"] = torch.zeros(H, rows, dtype=torch.float32, device=DEV)
        if own:
            from pippy_amd import _native as N
            # one plan per batch of sequences serves every layer and both directions
            s["plan"] = N.attn_packed_plan(s["cu"], rows)
    elif op == "route":
        T, E, K, C = case["tokens"], case["experts"], case["topk"], case["width"]
        dtype = torch.float32 if case["fp32"] else torch.bfloat16
        s["logits"] = randn(T, E, dtype=dtype)
        s["bias"] = randn(E, scale=0.05, dtype=torch.float32) if case["bias"] else None
        s["idx"] = torch.zeros(T, K, dtype=torch.int32, device=DEV)
        s["gate"] = torch.zeros(T, K, dtype=torch.float32, device=DEV)
        if case["train"]:
            s["dout"] = randn(T, C, scale=0.1)
            s["y"] = randn(T * K, C)
            s["pos"] = torch.randperm(T * K, generator=g, device=DEV).to(torch.int32)
            s["dlogits"] = torch.zeros(T, E, dtype=dtype, device=DEV)
    elif op == "permute":
        n, E = case["slots"], case["experts"]
        load = torch.rand(E, generator=g, device=DEV) + 0.1
        s["slots"] = torch.multinomial(load, n, replacement=True, generator=g).to(torch.int32)
        s["seg"] = torch.zeros(E + 1, dtype=torch.int32, device=DEV)
        s["row_src"] = torch.zeros(n, dtype=torch.int32, device=DEV)
        s["pos"] = torch.zeros(n, dtype=torch.int32, device=DEV)
        if own:
            from pippy_amd import _native as N
            s["ws"] = torch.empty(N.moe_permute_workspace(n, E), dtype=torch.int32, device=DEV)
    else:
        R, C = case["rows"], case["width"]
        dtype = torch.float32 if case["fp32"] else torch.bfloat16
        s["x"], s["resid"], s["dy"] = (randn(R, C, dtype=dtype) for _ in range(3))
        s["y"], s["dx"] = torch.empty_like(s["x"]), torch.empty_like(s["x"])
        s["rng"] = torch.tensor([seed * 0x9E3779B97F4A7C15 % 2 ** 62, seed % 1000], dtype=torch.int64, device=DEV)
        s["site"] = 3
    return s


def _heads(rows, H, G, D):
    q, k, v = rows.split([H * D, G * D, G * D], dim=-1)
    return q.view(-1, H, D), k.view(-1, G, D), v.view(-1, G, D)


# ---- one pass -----------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    op = {"attention": (_attention_plain, _attention_own), "route": (_route_plain, _route_own),
          "permute": (_permute_plain, _permute_own), "dropout": (_dropout_plain, _dropout_own)}[case["op"]]
    return op[bool(own)](s, case)


def _attention_own(s, case):
    from pippy_amd import _native as N
    N.attn_packed_fwd(s["q"], s["k"], s["v"], s["o"], s["lse"], s["plan"], causal=case["causal"])
    if not case["train"]:
        return s["o"], s["lse"]
    N.attn_packed_bwd(s["q"], s["k"], s["v"], s["o"], s["lse"], s["do"], s["dq"], s["dk"], s["dv"], s["delta"],
                      s["plan"], causal=case["causal"])
    return s["o"], s["lse"], s["dqkv"]


def _route_own(s, case):
    from pippy_amd import _native as N
    how = dict(bias=s["bias"], scoring=case["scoring"], n_group=case["groups"], topk_group=case["kept"],
               group_score="top2" if case["bias"] else "max", renorm=case["renorm"], scale=1.5)
    N.moe_route(s["logits"], s["idx"], s["gate"], **how)
    if not case["train"]:
        return s["idx"], s["gate"]
    N.moe_route_bwd(s["logits"], s["idx"], s["dlogits"], dout=s["dout"], y=s["y"], pos=s["pos"],
                    scoring=case["scoring"], renorm=case["renorm"], scale=1.5)
    return s["idx"], s["gate"], s["dlogits"]


def _permute_own(s, case):
    from pippy_amd import _native as N
    N.moe_permute_ws(s["slots"], case["experts"], s["seg"], s["row_src"], s["pos"], s["ws"])
    return s["seg"], s["row_src"], s["pos"]


def _dropout_own(s, case):
    from pippy_amd import _native as N
    N.dropout_add(s["x"], s["y"], s["rng"], case["p"], resid=s["resid"], site=s["site"])
    N.dropout_bwd(s["dy"], s["dx"], s["rng"], case["p"], site=s["site"])
    return s["y"], s["dx"]


# ---- the plain forms ----------------------------------------------------------------------------------
def _attention_plain(s, case):
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    rep, scale = H // G, D ** -0.5
    q, k, v = (t.float().transpose(0, 1) for t in (s["q"], s["k"], s["v"]))
    o, lse = torch.zeros_like(q), torch.zeros_like(s["lse"])
    dq, dk, dv = (torch.zeros_like(t) for t in (q, k, v))
    r0 = 0
    for n in s["lens"]:
        rows = slice(r0, r0 + n)
        r0 += n
        if n == 0:
            continue
        hidden = torch.ones(n, n, dtype=torch.bool, device=DEV).triu(1) if case["causal"] else None
        for h in range(G):
            heads = slice(h * rep, (h + 1) * rep)
            qh, kh, vh = q[heads, rows].reshape(rep * n, D), k[h, rows], v[h, rows]
            sc = (qh @ kh.t() * scale).view(rep, n, n)
            if hidden is not None:
                sc.masked_fill_(hidden, float("-inf"))
            top = sc.amax(-1, keepdim=True)
            p = torch.exp(sc - top)
            total = p.sum(-1, keepdim=True)
            p = (p / total).view(rep * n, n)
            oh = p @ vh
            o[heads, rows] = oh.view(rep, n, D)
            lse[heads, rows] = (top + torch.log(total)).squeeze(-1)
            if case["train"]:
                doh = s["do"][rows, heads].float().transpose(0, 1).reshape(rep * n, D)
                dv[h, rows] = p.t() @ doh
                dp = doh @ vh.t()
                ds = p * (dp - (doh * oh).sum(-1, keepdim=True)) * scale
                dq[heads, rows] = (ds @ kh).view(rep, n, D)
                dk[h, rows] = ds.t() @ qh
    out = o.transpose(0, 1).to(torch.bfloat16)
    if not case["train"]:
        return out, lse
    return out, lse, torch.cat([t.transpose(0, 1).flatten(1) for t in (dq, dk, dv)], -1).to(torch.bfloat16)


def _route_plain(s, case):
    T, E, K = case["tokens"], case["experts"], case["topk"]
    x = s["logits"].float()
    # the selection compares neighbouring scores: in 64 bits
    wide = x.double()
    choice = torch.softmax(wide, -1) if case["scoring"] == "softmax" else torch.sigmoid(wide)
    if s["bias"] is not None:
        choice = choice + s["bias"].double()
    if case["groups"] > 1:
        by_group = choice.view(T, case["groups"], -1)
        if case["bias"]:
            best = torch.sort(by_group, dim=-1, descending=True).values[..., :2].sum(-1)
        else:
            best = by_group.amax(-1)
        kept = torch.sort(best, dim=-1, descending=True, stable=True).indices[:, :case["kept"]]
        open_ = torch.zeros_like(best, dtype=torch.bool).scatter_(1, kept, True)
        choice = by_group.masked_fill(~open_[..., None], float("-inf")).view(T, E)
    idx = torch.sort(choice, dim=-1, descending=True, stable=True).indices[:, :K]
    if case["scoring"] == "softmax":
        e = torch.exp(x - x.amax(-1, keepdim=True))
        score = e / e.sum(-1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-x))
    picked = score.gather(-1, idx)
    total = picked.sum(-1, keepdim=True) if case["renorm"] else 1.0
    gate = 1.5 * picked / total
    if not case["train"]:
        return idx.to(torch.int32), gate
    rows = s["y"][s["pos"].long()].view(T, K, -1).float()
    dgate = (rows * s["dout"].float()[:, None]).sum(-1)
    if case["renorm"]:
        d = 1.5 * (dgate - (picked / total * dgate).sum(-1, keepdim=True)) / total
    else:
        d = 1.5 * dgate
    dscore = torch.zeros_like(score).scatter_(1, idx, d)
    if case["scoring"] == "softmax":
        dx = score * (dscore - (score * dscore).sum(-1, keepdim=True))
    else:
        dx = dscore * score * (1 - score)
    return idx.to(torch.int32), gate, dx.to(s["logits"].dtype)


def _permute_plain(s, case):
    slots = s["slots"].long()
    order = torch.sort(slots, stable=True).indices
    pos = torch.empty_like(order)
    pos[order] = torch.arange(order.numel(), device=DEV)
    counts = torch.zeros(case["experts"], dtype=torch.int64, device=DEV).index_add_(0, slots, torch.ones_like(slots))
    seg = torch.cat([torch.zeros_like(counts[:1]), counts.cumsum(0)])
    return tuple(t.to(torch.int32) for t in (seg, order, pos))


def _dropout_plain(s, case):
    n = s["x"].numel()
    seed, offset = s["rng"][0], s["rng"][1]
    group = torch.arange((n + 7) // 8, device=DEV)
    low = 0xFFFFFFFF
    c = [group, (offset & low).expand_as(group), (offset >> 32 & low).expand_as(group),
         torch.full_like(group, s["site"])]
    k0, k1 = seed & low, seed >> 32 & low
    for _ in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57      # modulo 2^64
        c = [(p1 >> 32 & low) ^ c[1] ^ k0, p1 & low, (p0 >> 32 & low) ^ c[3] ^ k1, p0 & low]
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    bits = torch.stack([half for w in c for half in (w & 0xFFFF, w >> 16)], -1).flatten()[:n]
    border = round(case["p"] * 65536)
    factor = (bits >= border).view(s["x"].shape).float() * (65536 / (65536 - border))
    y = s["resid"].float() + s["x"].float() * factor
    return y.to(s["x"].dtype), (s["dy"].float() * factor).to(s["x"].dtype)


# ---- the definitions in 64 bits -------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _attention_exact, "route": _route_exact, "permute": _permute_exact,
            "dropout": _dropout_exact}[case["op"]](s, case)


def _attention_exact(s, case):
    H, D, rows = case["heads"], case["dim"], s["q"].shape[0]
    group = H // case["kv_heads"]
    ends = np.cumsum(s["lens"])
    o = torch.zeros(rows, H, D, dtype=torch.float64, device=DEV)
    lse = torch.zeros(H, rows, dtype=torch.float64, device=DEV)
    dq = torch.zeros_like(o)
    dk = torch.zeros(rows, case["kv_heads"], D, dtype=torch.float64, device=DEV)
    dv = torch.zeros_like(dk)
    for end, n in zip(ends, s["lens"]):
        for h in range(H if n else 0):
            at = slice(int(end) - n, int(end))
            q, k, v = s["q"][at, h].double(), s["k"][at, h // group].double(), s["v"][at, h // group].double()
            logit = torch.mm(q, k.T.contiguous()) / math.sqrt(D)
            if case["causal"]:
                i = torch.arange(n, device=DEV)
                logit[i[None, :] > i[:, None]] = -math.inf
            norm = torch.logsumexp(logit, 1)
            weight = torch.exp(logit - norm[:, None])
            lse[h, at] = norm
            o[at, h] = torch.mm(weight, v)
            if not case["train"]:
                continue
            do = s["do"][at, h].double()
            dv[at, h // group] += torch.mm(weight.T.contiguous(), do)
            dweight = torch.mm(do, v.T.contiguous())
            dlogit = weight * (dweight - (weight * dweight).sum(1, keepdim=True)) / math.sqrt(D)
            dq[at, h] = torch.mm(dlogit, k)
            dk[at, h // group] += torch.mm(dlogit.T.contiguous(), q)
    if not case["train"]:
        return o, lse
    return o, lse, torch.cat([dq.reshape(rows, -1), dk.reshape(rows, -1), dv.reshape(rows, -1)], 1)


def _route_exact(s, case):
    T, E, K = case["tokens"], case["experts"], case["topk"]
    x = s["logits"].double().cpu().numpy()
    if case["scoring"] == "softmax":
        score = np.exp(x - x.max(1, keepdims=True))
        score /= score.sum(1, keepdims=True)
    else:
        score = 1.0 / (1.0 + np.exp(-x))
    rank = score if s["bias"] is None else score + s["bias"].double().cpu().numpy()
    if case["groups"] > 1:
        inside = rank.reshape(T, case["groups"], -1)
        ordered = -np.sort(-inside, axis=2)
        value = ordered[:, :, 0] + ordered[:, :, 1] if case["bias"] else ordered[:, :, 0]
        order = np.argsort(-value, axis=1, kind="stable")
        rank = np.full_like(inside, -np.inf)
        lines = np.arange(T)[:, None]
        rank[lines, order[:, :case["kept"]]] = inside[lines, order[:, :case["kept"]]]
        rank = rank.reshape(T, E)
    idx = np.argsort(-rank, axis=1, kind="stable")[:, :K]
    picked = np.take_along_axis(score, idx, 1)
    total = picked.sum(1, keepdims=True) if case["renorm"] else np.ones((T, 1))
    gate = 1.5 * picked / total
    if not case["train"]:
        return idx.astype(np.int32), gate
    y = s["y"].double().cpu().numpy()[s["pos"].cpu().numpy()].reshape(T, K, -1)
    dgate = np.matmul(y, s["dout"].double().cpu().numpy()[:, :, None])[:, :, 0]
    along = 1.5 * (dgate - (gate / 1.5 * dgate).sum(1, keepdims=True)) / total if case["renorm"] else 1.5 * dgate
    dscore = np.zeros((T, E))
    np.put_along_axis(dscore, idx, along, 1)
    if case["scoring"] == "softmax":
        dx = score * dscore - score * (score * dscore).sum(1, keepdims=True)
    else:
        dx = dscore * score * (1.0 - score)
    return idx.astype(np.int32), gate, dx


def _permute_exact(s, case):
    slots = s["slots"].cpu().numpy()
    order = np.argsort(slots, kind="stable").astype(np.int32)
    pos = np.empty_like(order)
    pos[order] = np.arange(len(slots), dtype=np.int32)
    seg = np.concatenate([[0], np.bincount(slots, minlength=case["experts"]).cumsum()]).astype(np.int32)
    return seg, order, pos


def _dropout_exact(s, case):
    seed, offset = (int(v) for v in s["rng"].cpu())
    n = case["rows"] * case["width"]
    u32 = np.uint64(0xFFFFFFFF)
    c0 = np.arange((n + 7) // 8, dtype=np.uint64)
    c1, c2, c3 = (np.full_like(c0, v) for v in (offset % 2 ** 32, offset >> 32, s["site"]))
    key = [seed % 2 ** 32, seed >> 32]
    for _ in range(10):
        a, b = c0 * np.uint64(0xD2511F53), c2 * np.uint64(0xCD9E8D57)
        c0, c1, c2, c3 = ((b >> np.uint64(32)) ^ c1 ^ np.uint64(key[0]), b & u32,
                          (a >> np.uint64(32)) ^ c3 ^ np.uint64(key[1]), a & u32)
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    draws = np.empty((len(c0), 8), dtype=np.uint32)
    for w, c in enumerate((c0, c1, c2, c3)):
        draws[:, 2 * w], draws[:, 2 * w + 1] = c & np.uint64(0xFFFF), c >> np.uint64(16)
    border = round(case["p"] * 65536)
    kept = torch.from_numpy((draws.reshape(-1)[:n] >= border).reshape(case["rows"], -1)).to(DEV)
    scale = 65536.0 / (65536 - border)
    x, resid, dy = (s[k].double() for k in ("x", "resid", "dy"))
    zero = torch.zeros((), dtype=torch.float64, device=DEV)
    return resid + torch.where(kept, x * scale, zero), torch.where(kept, dy * scale, zero)
