"""What is measured of the training operators of the extractor LM (smsgate_amd/models/train_ops.py).

Three operators of a training step, each forward and backward as one pass:

* ``embed``: the token embedding ``scale * (table[ids] + table[add_ids])`` and the table's gradient;
* ``attention``: grouped-query attention over a padded batch, and the gradients of q, k and v (``train``), or its forward
  alone (an evaluation);
* ``loss``: the softmax cross entropy of hidden states over the rows of the (tied) embedding, and the gradients of both.

``own = False``: the plain forms, elementary torch operations in 32 bits, rounded once at the end.  ``own = True``: the
framework's operators as a training program calls them, through autograd.
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---------------------------------------------------------------------------- cases
def listed():
    return [
        # one short message through the small extractor (hidden 256, 8192 ids): launch latency is all there is
        dict(name="embed-one-message", op="embed", rows=45, vocab=8192, hidden=256, dtype="fp32", add=False, scale=1.0),
        # the flagship training step: 128 qa-format examples of about 60 tokens, pointer rows added to the message's
        # positions, fp32 master table trimmed to the ids in use
        dict(name="embed-flagship-step", op="embed", rows=128 * 61, vocab=8576, hidden=576, dtype="fp32", add=True, scale=1.0),
        # a long batch over the whole vocabulary, bf16 table, scaled by sqrt(hidden): the largest
        dict(name="embed-full-vocabulary", op="embed", rows=130999, vocab=49152, hidden=960, dtype="bf16", add=False,
             scale=30.983866769659336),
        # one message through the small extractor's 4 query / 2 key heads
        dict(name="attention-one-message", op="attention", batch=1, seq=37, heads=4, kv_heads=2, dim=64, dtype="bf16",
             causal=True, ragged=False, train=True),
        # the flagship training step's batch, padded at the end
        dict(name="attention-flagship-step", op="attention", batch=128, seq=61, heads=9, kv_heads=3, dim=64, dtype="bf16",
             causal=True, ragged=True, train=True),
        # scoring long threads with the 960-wide variant: forward alone, odd length
        dict(name="attention-evaluation", op="attention", batch=8, seq=2047, heads=15, kv_heads=5, dim=64, dtype="bf16",
             causal=True, ragged=True, train=False),
        # bidirectional fp16 training with 128-wide heads, no sharing of key heads
        dict(name="attention-wide-heads", op="attention", batch=4, seq=1000, heads=8, kv_heads=8, dim=128, dtype="fp16",
             causal=False, ragged=False, train=True),
        # one long document (a whole statement instead of one message): the largest
        dict(name="attention-long-document", op="attention", batch=1, seq=16384, heads=9, kv_heads=3, dim=64, dtype="bf16",
             causal=True, ragged=False, train=True),
        # the answer rows of one message, small extractor
        dict(name="loss-one-answer", op="loss", rows=61, vocab=8192, hidden=256, dtype="bf16", kept=0.5, reduction="mean"),
        # the flagship step of the copy format: 128 padded sequences, the answer rows (about a third) labelled
        dict(name="loss-flagship-step", op="loss", rows=128 * 113, vocab=8192, hidden=576, dtype="bf16", kept=0.33,
             reduction="mean"),
        # fp16, the 960-wide variant, ragged rows and ids, a weight for each row's loss
        dict(name="loss-weighted-rows", op="loss", rows=4001, vocab=32003, hidden=960, dtype="fp16", kept=0.9,
             reduction="none"),
        # every row labelled over the whole vocabulary: the largest
        dict(name="loss-full-vocabulary", op="loss", rows=8192, vocab=49152, hidden=576, dtype="bf16", kept=1.0,
             reduction="mean"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "attention", "attention", "loss"])
    if op == "embed":
        hidden = rng.choice([128, 256, 576, 960, rng.randrange(65, 960)])
        rows = min(_log(rng, 1, 130999), 130999 * 960 // hidden)
        return dict(op=op, rows=rows, vocab=_log(rng, 300, 49152), hidden=hidden, dtype=rng.choice(["bf16", "fp16", "fp32"]),
                    add=rng.random() < 0.5, scale=rng.choice([1.0, math.sqrt(hidden)]))
    if op == "attention":
        kv_heads = rng.choice([1, 2, 3, 5])
        heads = kv_heads * rng.choice([1, 2, 3, 4])
        dim = rng.choice([64, 64, 128])
        seq = _log(rng, 1, 8000)
        most = 9 * 64 * 16384 * 16384 // 2 // (heads * dim * seq * seq)  # half the largest listed case's products
        most = max(1, min(most, 2_000_000 // (heads * seq)))  # and its tensors
        batch = _log(rng, 1, min(128, most))
        return dict(op=op, batch=batch, seq=seq, heads=heads, kv_heads=kv_heads, dim=dim, dtype=rng.choice(["bf16", "fp16"]),
                    causal=rng.random() < 0.75, ragged=rng.random() < 0.5, train=rng.random() < 0.7)
    hidden = rng.choice([128, 256, 576, 960, 8 * rng.randrange(9, 120)])
    vocab = _log(rng, 100, 49152)
    rows = min(_log(rng, 1, 8192), 8192 * 49152 * 576 // (vocab * hidden))
    return dict(op=op, rows=rows, vocab=vocab, hidden=hidden, dtype=rng.choice(["bf16", "fp16"]),
                kept=round(rng.uniform(0.2, 1.0), 3), reduction=rng.choice(["mean", "sum", "none"]))


def _lengths(case):
    """The batch's lengths, as a multiset: from the whole row down to about a third of it."""
    B, T = case["batch"], case["seq"]
    return [T if not case["ragged"] else max(1, T - (7 * b * T) // (10 * B)) for b in range(B)]


def _labelled(case):
    return max(1, min(case["rows"], int(round(case["kept"] * case["rows"]))))


def work(case):
    z = BYTES[case["dtype"]]
    if case["op"] == "embed":
        n, V, H = case["rows"], case["vocab"], case["hidden"]
        two = 2 if case["add"] else 1
        # the rows looked up, x, dx, the table's gradient and the ids of both directions
        return {"bytes": two * min(n, V) * H * z + 2 * n * H * z + V * H * z + 8 * n * two, "flops": two * 2 * n * H}
    if case["op"] == "attention":
        B, T, nh, nkv, D = (case[k] for k in ("batch", "seq", "heads", "kv_heads", "dim"))
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in _lengths(case))
        qo, kv = B * nh * T * D * z, B * nkv * T * D * z
        if not case["train"]:
            return {"bytes": 2 * qo + 2 * kv, "flops": 4 * D * nh * pairs}
        return {"bytes": 4 * qo + 4 * kv, "flops": 14 * D * nh * pairs}
    n, N, V, H = _labelled(case), case["rows"], case["vocab"], case["hidden"]
    return {"bytes": (n + N) * H * z + 2 * V * H * z + 8 * N, "flops": 6 * n * V * H}


# ---------------------------------------------------------------------------- inputs
def _zipf(n, vocab, g):
    """Token ids as text has them: a few very common ones (a shared prompt, separators), a long tail."""
    u = torch.rand(n, generator=g, device=DEVICE, dtype=torch.float64)
    ids = (torch.exp(u * math.log(vocab + 1.0)) - 1.0).long().clamp_(0, vocab - 1)
    return (ids * 7919 + 13) % vocab  # spread over the table


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE)

    t = DTYPES[case["dtype"]]
    s = {"case": dict(case)}
    if case["op"] == "embed":
        n, V, H = case["rows"], case["vocab"], case["hidden"]
        s["ids"] = _zipf(n, V, g)
        if case["add"]:  # pointer rows at the message's positions, none (-1) elsewhere
            none = torch.rand(n, generator=g, device=DEVICE) < 0.3
            ptr = V - 1 - torch.arange(n, device=DEVICE) % min(V, 61)
            s["add"] = torch.where(none, torch.full_like(ptr, -1), ptr)
        s["table"] = (normal(V, H) * 0.02).to(t).requires_grad_()
        s["dx"] = (normal(n, H) * 1e-3).to(t)
    elif case["op"] == "attention":
        B, T, nh, nkv, D = (case[k] for k in ("batch", "seq", "heads", "kv_heads", "dim"))
        for name, h in (("q", nh), ("k", nkv), ("v", nkv)):
            s[name] = normal(B, h, T, D).to(t).requires_grad_(case["train"])
        if case["ragged"]:
            order = torch.randperm(B, generator=g, device=DEVICE)
            s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=DEVICE)[order]
        if case["train"]:
            s["dout"] = normal(B, T, nh * D).to(t)
    else:
        N, V, H = case["rows"], case["vocab"], case["hidden"]
        table = normal(V, H) * 0.05
        labels = _zipf(N, V, g)
        # a partly trained model: final-normed states that lean to their label's row, some more than others
        lean = torch.rand(N, 1, generator=g, device=DEVICE) * 12.0 / (0.05 * math.sqrt(H))
        h = normal(N, H) + lean * table[labels] / (0.05 * math.sqrt(H))
        h = h * torch.rsqrt(h.square().mean(-1, keepdim=True))
        out = torch.randperm(N, generator=g, device=DEVICE)[_labelled(case):]
        labels[out] = -100
        s["h"], s["table"], s["labels"] = h.to(t).requires_grad_(), table.to(t).requires_grad_(), labels
        if case["reduction"] == "none":
            s["dloss"] = torch.rand(N, generator=g, device=DEVICE) / N
    return s


# ---------------------------------------------------------------------------- one pass
def run(state):
    return {"embed": _embed, "attention": _attention, "loss": _loss}[state["case"]["op"]](state)


def _embed(s):
    scale, add = s["case"]["scale"], s.get("add")
    if own:
        from smsgate_amd.models import train_ops

        x = train_ops.embed_lookup(s["ids"], s["table"], add, scale=scale)
        (dtable,) = torch.autograd.grad(x, s["table"], s["dx"])
        return {"x": x, "dtable": dtable}
    with torch.no_grad():
        table = s["table"]
        x = table[s["ids"]].float()
        d = s["dx"].float() * scale
        dtable = torch.zeros(table.shape, dtype=torch.float32, device=table.device).index_add_(0, s["ids"], d)
        if add is not None:
            some, at = (add >= 0).unsqueeze(-1), add.clamp(min=0)
            x = x + table[at].float() * some
            dtable.index_add_(0, at, d * some)
        return {"x": (x * scale).to(table.dtype), "dtable": dtable.to(table.dtype)}


def _attention(s):
    c, lengths = s["case"], s.get("lengths")
    q, k, v = s["q"], s["k"], s["v"]
    scale = 1.0 / math.sqrt(c["dim"])
    if own:
        from smsgate_amd.models import train_ops

        out = train_ops.tiled_attention(q, k, v, scale, causal=c["causal"], lengths=lengths)
        if not c["train"]:
            return {"out": out}
        dq, dk, dv = torch.autograd.grad(out, (q, k, v), s["dout"])
        return {"out": out, "dq": dq, "dk": dk, "dv": dv}
    with torch.no_grad():
        B, nh, T, D = q.shape
        nkv = k.shape[1]
        qf = q.float()
        kf, vf = (t.float().repeat_interleave(nh // nkv, dim=1) for t in (k, v))
        j = torch.arange(T, device=q.device)
        seen = torch.ones(1, 1, T, T, dtype=torch.bool, device=q.device)
        if c["causal"]:
            seen = seen & (j[None, :] <= j[:, None])
        if lengths is not None:
            inside = j[None, :] < lengths[:, None]
            seen = seen & inside[:, None, None, :] & inside[:, None, :, None]
        p = (qf @ kf.transpose(-1, -2)).mul_(scale).masked_fill_(~seen, -math.inf)
        top = p.amax(-1, keepdim=True)
        p = p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
        total = p.sum(-1, keepdim=True)
        p = p.div_(torch.where(total == 0, 1.0, total))
        out = (p @ vf).transpose(1, 2).reshape(B, T, nh * D).to(q.dtype)
        if not c["train"]:
            return {"out": out}
        do = s["dout"].float().reshape(B, T, nh, D).transpose(1, 2)
        dv = (p.transpose(-1, -2) @ do).reshape(B, nkv, nh // nkv, T, D).sum(2)
        dp = do @ vf.transpose(-1, -2)
        ds = dp.sub_((p * dp).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        dq = ds @ kf
        dk = (ds.transpose(-1, -2) @ qf).reshape(B, nkv, nh // nkv, T, D).sum(2)
        return {"out": out, "dq": dq.to(q.dtype), "dk": dk.to(q.dtype), "dv": dv.to(q.dtype)}


def _loss(s):
    reduction = s["case"]["reduction"]
    h, table, labels = s["h"], s["table"], s["labels"]
    if own:
        from smsgate_amd.models import train_ops

        loss = train_ops.lm_loss(h, table, labels, reduction=reduction)
        dh, dtable = torch.autograd.grad(loss, (h, table), s.get("dloss"))
        return {"loss": loss, "dh": dh, "dtable": dtable}
    with torch.no_grad():
        rows = (labels != -100).nonzero().squeeze(1)
        y = labels[rows]
        hs, w = h[rows].float(), table.float()
        p = hs @ w.t()
        target = p.gather(1, y[:, None]).squeeze(1)
        top = p.amax(1, keepdim=True)
        p = p.sub_(top).exp_()
        total = p.sum(1, keepdim=True)
        each = torch.zeros(h.shape[0], device=h.device)
        each[rows] = total.log().squeeze(1) + top.squeeze(1) - target
        if reduction == "none":
            loss, by = each, s["dloss"][rows]
        elif reduction == "sum":
            loss, by = each.sum(), torch.ones(len(rows), device=h.device)
        else:
            loss, by = each.sum() / len(rows), torch.full((len(rows),), 1.0 / len(rows), device=h.device)
        d = p.div_(total)
        d[torch.arange(len(rows), device=h.device), y] -= 1.0
        d = d.mul_(by[:, None])
        dh = torch.zeros(h.shape, dtype=torch.float32, device=h.device)
        dh[rows] = d @ w
        return {"loss": loss, "dh": dh.to(h.dtype), "dtable": (d.t() @ hs).to(table.dtype)}


# ---------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    double = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    with torch.enable_grad():
        return {"embed": _exact_embed, "attention": _exact_attention, "loss": _exact_loss}[case["op"]](case, s, double)


def _exact_embed(case, s, d):
    table, n = d["table"], s["ids"].numel()
    one = torch.ones(n, dtype=torch.float64, device=DEVICE)
    at, which = [s["ids"]], [torch.arange(n, device=DEVICE)]
    if case["add"]:
        keep = s["add"] >= 0
        at.append(s["add"][keep])
        which.append(which[0][keep])
    at, which = torch.cat(at), torch.cat(which)
    # the lookup as a product with a sparse matrix of ones, its gradient with the transpose
    x = torch.zeros(n, table.shape[1], dtype=torch.float64, device=DEVICE)
    x.scatter_add_(0, which[:, None].expand(-1, table.shape[1]), table[at])
    dtable = torch.zeros_like(table)
    dtable.scatter_add_(0, at[:, None].expand(-1, table.shape[1]), (d["dx"] * one[:, None])[which])
    return {"x": x * case["scale"], "dtable": dtable * case["scale"]}


def _exact_attention(case, s, d):
    B, T, nh, nkv, D = (case[k] for k in ("batch", "seq", "heads", "kv_heads", "dim"))
    rep = nh // nkv
    lens = s["lengths"].tolist() if "lengths" in s else [T] * B
    out = torch.zeros(B, T, nh, D, dtype=torch.float64, device=DEVICE)
    grads = {n: torch.zeros_like(d[n]) for n in "qkv"}
    step = rep if T > 4096 else nh  # heads at a time
    for b in range(B):
        n = lens[b]
        if n == 0:
            continue
        for h0 in range(0, nh, step):
            g0, g1 = h0 // rep, (h0 + step) // rep
            q = d["q"][b, h0:h0 + step, :n].clone().requires_grad_()
            k = d["k"][b, g0:g1, :n].clone().requires_grad_()
            v = d["v"][b, g0:g1, :n].clone().requires_grad_()
            grp = torch.arange(step, device=DEVICE) // rep
            score = torch.matmul(q, k[grp].transpose(1, 2)) / math.sqrt(D)
            if case["causal"]:
                score = score + torch.full((n, n), -math.inf, dtype=torch.float64, device=DEVICE).triu(1)
            o = torch.matmul(torch.softmax(score, -1), v[grp])
            out[b, :n, h0:h0 + step] = o.detach().transpose(0, 1)
            if case["train"]:
                do = d["dout"][b, :n].reshape(n, nh, D)[:, h0:h0 + step].transpose(0, 1)
                gq, gk, gv = torch.autograd.grad(o, (q, k, v), do)
                grads["q"][b, h0:h0 + step, :n] = gq
                grads["k"][b, g0:g1, :n] = gk
                grads["v"][b, g0:g1, :n] = gv
            del score, o
    out = out.reshape(B, T, nh * D)
    return {"out": out, **{"d" + n: g for n, g in grads.items()}} if case["train"] else {"out": out}


def _exact_loss(case, s, d):
    h, table = d["h"].requires_grad_(), d["table"].requires_grad_()
    keep = s["labels"] >= 0
    y = s["labels"].clamp(min=0)
    score = torch.matmul(h, table.t())
    each = (torch.logsumexp(score, 1) - score.gather(1, y[:, None])[:, 0]) * keep
    if case["reduction"] == "none":
        loss, by = each, d["dloss"]
    else:
        loss, by = each.sum() / (keep.sum() if case["reduction"] == "mean" else 1), None
    dh, dtable = torch.autograd.grad(loss, (h, table), by)
    return {"loss": loss.detach(), "dh": dh, "dtable": dtable}
