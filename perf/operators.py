"""Measured cases of the sampling, top-k, distillation and shared-prefix attention operators.

Four operators of the C ABI (include/cngpt_cuda.h), each with listed cases that
stand for real calls, a generator of further cases of the same ranges, its
plain form in elementary torch operations and its definition in 64 bits:

  sample   cngpt_cuda_sample: one token per row of logits from given uniform
           numbers, with temperature, top-k, top-p and min-p of every row
  topk     cngpt_cuda_topk: the k largest logits of every row, in order
  distill  cngpt_cuda_distill: the loss of a student against a teacher's top
           logits (and hard targets), with or without its gradient
  prefix   cngpt_cuda_prefix_attention: one query per sequence over a prefix
           that all sequences share and over each sequence's own suffix

With `own` false run() computes the plain form (32 bits; 64 for the cumulative
probabilities that decide a token), with `own` true it calls the library.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one sequence of GPT-2's vocabulary, the usual chat settings: latency
        dict(name="sample one row", op="sample", rows=1, vocab=50257, mode="topk_topp", banned=0.0),
        # a serving batch in which every request has its own settings
        dict(name="sample mixed batch", op="sample", rows=32, vocab=50257, mode="mixed", banned=0.0),
        # a large batch by nucleus alone, part of the vocabulary forbidden (-inf)
        dict(name="sample large top-p", op="sample", rows=256, vocab=50257, mode="topp", banned=0.3),
        # top logits of one short scoring call, an odd vocabulary
        dict(name="topk short", op="topk", rows=37, vocab=32003, k=20),
        # a teacher's top logits for one GPT-2 training batch (8 x 1024 tokens)
        dict(name="topk training batch", op="topk", rows=8192, vocab=50257, k=64),
        # evaluation of a student on one sequence: the loss alone
        dict(name="distill loss", op="distill", rows=1024, vocab=50257, k=32, tau=2.0, alpha=1.0, grad=False, ragged=False),
        # a small ragged batch: entries and rows that count for nothing, an odd vocabulary
        dict(name="distill ragged", op="distill", rows=190, vocab=4999, k=11, tau=1.0, alpha=0.7, grad=True, ragged=True),
        # one GPT-2 training batch, soft and hard loss, loss and gradient
        dict(name="distill training batch", op="distill", rows=8192, vocab=50257, k=64, tau=2.0, alpha=0.5, grad=True,
             ragged=False),
        # the first step after a short prompt, one sample: latency
        dict(name="prefix one sample", op="prefix", batch=1, heads=12, kv_heads=12, hs=64, prefix=100, suffix=9, ragged=False),
        # 16 samples of one prompt within GPT-2's context
        dict(name="prefix 16 samples", op="prefix", batch=16, heads=12, kv_heads=12, hs=64, prefix=768, suffix=255, ragged=False),
        # long shared document, many requests of different lengths
        dict(name="prefix long", op="prefix", batch=48, heads=16, kv_heads=16, hs=64, prefix=16384, suffix=512, ragged=True),
        # grouped heads of another size, an odd prefix
        dict(name="prefix grouped", op="prefix", batch=12, heads=24, kv_heads=6, hs=128, prefix=5003, suffix=77, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("sample", "topk", "distill", "prefix"))
    if op == "sample":
        return dict(op=op, rows=_log(rng, 1, 256), vocab=_log(rng, 65, 50257),
                    mode=rng.choice(("plain", "topk", "topp", "minp", "topk_topp", "mixed")),
                    banned=rng.choice((0.0, 0.0, 0.3, 0.95)))
    if op == "topk":
        vocab = _log(rng, 65, 50257)
        return dict(op=op, rows=_log(rng, 1, 8192), vocab=vocab, k=min(vocab, _log(rng, 1, 256)))
    if op == "distill":
        vocab = _log(rng, 65, 50257)
        return dict(op=op, rows=_log(rng, 1, 8192), vocab=vocab, k=min(vocab, _log(rng, 1, 128)),
                    tau=rng.choice((1.0, 1.5, 2.0, 4.0)), alpha=rng.choice((1.0, 0.9, 0.5)), grad=rng.random() < 0.7,
                    ragged=rng.random() < 0.5)
    kv = rng.choice((2, 4, 6, 8, 12, 16))
    group = rng.choice((1, 1, 1, 2, 4))
    if kv * group > 32:
        group = 1
    return dict(op=op, batch=_log(rng, 1, 48), heads=kv * group, kv_heads=kv, hs=rng.choice((64, 64, 64, 32, 80, 128)),
                prefix=_log(rng, 1, 12000), suffix=_log(rng, 1, 512), ragged=rng.random() < 0.6)


# ----------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _logits(g, rows, vocab):
    """Logits as a language model gives them: a broad body, and for every row a
    few percent of the vocabulary raised well above it."""
    x = torch.randn(rows, vocab, generator=g, device=DEV).mul_(2.0)
    up = torch.rand(rows, vocab, generator=g, device=DEV).sub_(0.975).mul_(40.0).clamp_(min=0.0).square_()
    return x.add_(up, alpha=9.0)


def prepare(case, seed):
    return {"sample": _prepare_sample, "topk": _prepare_topk, "distill": _prepare_distill,
            "prefix": _prepare_prefix}[case["op"]](case, seed)


def _prepare_sample(case, seed):
    g, rows, vocab, mode = _gen(seed), case["rows"], case["vocab"], case["mode"]
    x = _logits(g, rows, vocab)
    if case["banned"]:
        ban = torch.rand(rows, vocab, generator=g, device=DEV) < case["banned"]
        ban[:, 0] = False
        x.masked_fill_(ban, -math.inf)
    r = lambda lo, hi: torch.rand(rows, generator=g, device=DEV) * (hi - lo) + lo  # noqa: E731
    temperature, top_p, min_p = r(0.6, 1.2), r(0.7, 0.98), r(0.01, 0.2)
    top_k = torch.randint(1, max(2, min(vocab, 200)), (rows,), generator=g, device=DEV, dtype=torch.int32)
    if mode == "mixed":  # every request has its own: each filter off in some rows, some rows greedy
        temperature[torch.rand(rows, generator=g, device=DEV) < 0.1] = 0.0
        top_k[torch.rand(rows, generator=g, device=DEV) < 0.4] = 0
        top_p[torch.rand(rows, generator=g, device=DEV) < 0.4] = 1.0
        min_p[torch.rand(rows, generator=g, device=DEV) < 0.6] = 0.0
    return dict(op="sample", logits=x, temperature=temperature,
                top_k=top_k if mode in ("topk", "topk_topp", "mixed") else None,
                top_p=top_p if mode in ("topp", "topk_topp", "mixed") else None,
                min_p=min_p if mode in ("minp", "mixed") else None,
                u=torch.rand(rows, generator=g, device=DEV),
                tokens=torch.empty(rows, dtype=torch.int32, device=DEV),
                logprob=torch.empty(rows, dtype=torch.float32, device=DEV))


def _prepare_topk(case, seed):
    g, rows, k = _gen(seed), case["rows"], case["k"]
    return dict(op="topk", logits=_logits(g, rows, case["vocab"]), k=k,
                values=torch.empty(rows, k, dtype=torch.float32, device=DEV),
                indices=torch.empty(rows, k, dtype=torch.int32, device=DEV))


def _prepare_distill(case, seed):
    g, rows, vocab, k = _gen(seed), case["rows"], case["vocab"], case["k"]
    x = _logits(g, rows, vocab)
    # the teacher's list: tokens spread over the vocabulary without repetition, logits falling
    first = torch.randint(0, vocab, (rows, 1), generator=g, device=DEV)
    step = torch.arange(k, device=DEV)[None, :] * max(1, vocab // k)
    ti = ((first + step) % vocab).to(torch.int32)
    tv = (torch.rand(rows, k, generator=g, device=DEV) * 12.0).sort(dim=1, descending=True).values
    tgt = torch.randint(0, vocab, (rows,), generator=g, device=DEV, dtype=torch.int32)
    if case["ragged"]:  # lists of different lengths; padding rows without list or target
        length = torch.randint(1, k + 1, (rows, 1), generator=g, device=DEV)
        ti[torch.arange(k, device=DEV)[None, :] >= length] = -1
        pad = torch.rand(rows, generator=g, device=DEV) < 0.2
        ti[pad] = -1
        tgt[pad] = -1
    return dict(op="distill", logits=x, top_val=tv, top_idx=ti, targets=tgt, tau=case["tau"], alpha=case["alpha"],
                scale=1.0 / rows, grad=case["grad"], loss=torch.empty((), dtype=torch.float32, device=DEV),
                row_loss=torch.empty(rows, dtype=torch.float32, device=DEV),
                dlogits=torch.empty(rows, vocab, dtype=torch.float32, device=DEV) if case["grad"] else None)


def _prepare_prefix(case, seed):
    g, B, H, Hk, hs, P, S = (_gen(seed), case["batch"], case["heads"], case["kv_heads"], case["hs"], case["prefix"],
                             case["suffix"])
    n = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    length = torch.full((B,), S, dtype=torch.int32, device=DEV)
    if case["ragged"]:
        length = torch.randint(0, S + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
    return dict(op="prefix", q=n(B, H, hs) * 1.5, pk=n(P, Hk, hs), pv=n(P, Hk, hs), sk=n(B, S, Hk, hs), sv=n(B, S, Hk, hs),
                length=length, scale=1.0 / math.sqrt(hs), out=torch.empty(B, H, hs, device=DEV), ws=None)


# -------------------------------------------------------------------- run
def run(state):
    if own:
        return {"sample": _own_sample, "topk": _own_topk, "distill": _own_distill, "prefix": _own_prefix}[state["op"]](state)
    return {"sample": _plain_sample, "topk": _plain_topk, "distill": _plain_distill, "prefix": _plain_prefix}[state["op"]](state)


_LIB = None


def _lib():
    global _LIB
    from cngpt_b200 import abi
    if _LIB is None:
        _LIB = abi.load()
    _LIB.cngpt_cuda_set_stream(torch.cuda.current_stream().cuda_stream)
    return _LIB


def _ok(status):
    if status:
        raise RuntimeError("status %d: %s" % (status, _LIB.cngpt_cuda_last_message().decode()))


def _p(t):
    return None if t is None else t.data_ptr()


def _own_sample(s):
    x = s["logits"]
    _ok(_lib().cngpt_cuda_sample(x.data_ptr(), x.stride(0), x.shape[0], x.shape[1], _p(s["temperature"]), _p(s["top_k"]),
                                 _p(s["top_p"]), _p(s["min_p"]), s["u"].data_ptr(), s["tokens"].data_ptr(),
                                 s["logprob"].data_ptr()))
    return dict(tokens=s["tokens"], logprob=s["logprob"])


def _own_topk(s):
    x = s["logits"]
    _ok(_lib().cngpt_cuda_topk(x.data_ptr(), x.stride(0), x.shape[0], x.shape[1], s["k"], s["values"].data_ptr(),
                               s["indices"].data_ptr()))
    return dict(values=s["values"], indices=s["indices"])


def _own_distill(s):
    x, d = s["logits"], s["dlogits"]
    _ok(_lib().cngpt_cuda_distill(x.data_ptr(), x.stride(0), x.shape[0], x.shape[1], s["top_val"].data_ptr(),
                                  s["top_idx"].data_ptr(), s["top_idx"].shape[1], s["targets"].data_ptr(), s["tau"],
                                  s["alpha"], s["scale"], s["loss"].data_ptr(), s["row_loss"].data_ptr(), _p(d),
                                  0 if d is None else d.stride(0)))
    out = dict(loss=s["loss"], row_loss=s["row_loss"])
    if d is not None:
        out["dlogits"] = d
    return out


def _own_prefix(s):
    q, pk, sk = s["q"], s["pk"], s["sk"]
    B, H, hs = q.shape
    P, Hk, S = pk.shape[0], pk.shape[1], sk.shape[1]
    lib = _lib()
    if s["ws"] is None:
        n = lib.cngpt_cuda_prefix_attention_workspace(B, H, Hk, hs, P, S)
        s["ws"] = torch.empty(max(n, 16), dtype=torch.uint8, device=DEV)
    _ok(lib.cngpt_cuda_prefix_attention(q.data_ptr(), H * hs, pk.data_ptr(), s["pv"].data_ptr(), Hk * hs, P, sk.data_ptr(),
                                        s["sv"].data_ptr(), Hk * hs, S * Hk * hs, s["length"].data_ptr(), S,
                                        s["out"].data_ptr(), H * hs, B, H, Hk, hs, s["scale"], s["ws"].data_ptr(),
                                        s["ws"].numel()))
    return s["out"]


def _plain_sample(s):
    """Filters in the order top-k, top-p (over what top-k keeps), min-p; the
    cumulative probabilities in 64 bits, since they decide a whole number."""
    x, u = s["logits"], s["u"].double()
    rows, vocab = x.shape
    temp = s["temperature"].double()
    greedy = ~(temp > 0)
    v, order = torch.sort(x, dim=1, descending=True, stable=True)
    top = v[:, :1].double()
    t = torch.where(greedy, torch.ones_like(temp), temp)[:, None]
    w = torch.exp((v.double() - top) / t)  # weights in falling order, the largest 1
    rank = torch.arange(vocab, device=x.device)[None, :]
    keep = w > 0
    if s["top_k"] is not None:
        k = s["top_k"][:, None].long()
        keep &= (k <= 0) | (rank < k)
    if s["top_p"] is not None:
        p = s["top_p"].double()[:, None]
        wk = torch.where(keep, w, torch.zeros_like(w))
        before = torch.cumsum(wk, 1) - wk
        keep &= (p >= 1) | (before < p * wk.sum(1, keepdim=True)) | (rank == 0)
    if s["min_p"] is not None:
        keep &= (w >= s["min_p"].double()[:, None].clamp(max=1.0))
    keep &= ~greedy[:, None] | (rank == 0)
    wi = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, torch.zeros_like(w)))  # back in the vocabulary's order
    cdf = torch.cumsum(wi, 1)
    total = cdf[:, -1:]
    hit = (cdf > u[:, None] * total) & (wi > 0)
    tokens = hit.to(torch.int8).argmax(1, keepdim=True)
    logprob = torch.log(wi.gather(1, tokens) / total)
    return dict(tokens=tokens[:, 0].to(torch.int32), logprob=logprob[:, 0].float())


def _plain_topk(s):
    v, i = torch.sort(s["logits"], dim=1, descending=True, stable=True)
    return dict(values=v[:, : s["k"]].contiguous(), indices=i[:, : s["k"]].to(torch.int32))


def _plain_distill(s):
    x, tau, alpha, scale = s["logits"], s["tau"], s["alpha"], s["scale"]
    rows, vocab = x.shape
    ti, tgt = s["top_idx"].long(), s["targets"].long()
    ok = ti >= 0
    any_ok = ok.any(1, keepdim=True)
    m = x.max(1, keepdim=True).values
    # the teacher's distribution over its list
    z = torch.where(ok, s["top_val"] / tau, torch.full_like(s["top_val"], -math.inf))
    z = z - torch.where(any_ok, z.max(1, keepdim=True).values, torch.zeros_like(m))
    ez = torch.exp(z)
    sz = torch.where(any_ok, ez.sum(1, keepdim=True), torch.ones_like(m))
    p = ez / sz
    logp = torch.where(ok, z - torch.log(sz), torch.zeros_like(z))
    e = torch.exp((x - m) / tau)
    se = e.sum(1, keepdim=True)
    at = ti.clamp(min=0)
    logq = (x.gather(1, at) - m) / tau - torch.log(se)
    row = alpha * tau * tau * (p * (logp - torch.where(ok, logq, torch.zeros_like(logq)))).sum(1)
    grad = None
    if s["grad"]:
        grad = e.mul_(torch.where(any_ok, alpha * tau * scale / se, torch.zeros_like(se)))
        grad.scatter_add_(1, at, p * (-alpha * tau * scale))
    if alpha < 1:
        has = (tgt >= 0)[:, None]
        e1 = torch.exp(x - m)
        s1 = e1.sum(1, keepdim=True)
        t = tgt.clamp(min=0)[:, None]
        row = row + (1 - alpha) * torch.where(has, torch.log(s1) + m - x.gather(1, t), torch.zeros_like(m))[:, 0]
        if grad is not None:
            grad.add_(e1.mul_(torch.where(has, (1 - alpha) * scale / s1, torch.zeros_like(s1))))
            grad.scatter_add_(1, t, torch.where(has, torch.full_like(m, -(1 - alpha) * scale), torch.zeros_like(m)))
    out = dict(loss=row.sum() * scale, row_loss=row)
    if grad is not None:
        out["dlogits"] = grad
    return out


def _plain_prefix(s):
    q, pk, pv, sk, sv = s["q"], s["pk"], s["pv"], s["sk"], s["sv"]
    B, H, hs = q.shape
    P, Hk = pk.shape[:2]
    S = sk.shape[1]
    qg = q.view(B, Hk, H // Hk, hs) * s["scale"]
    a = torch.matmul(qg.permute(1, 0, 2, 3).reshape(Hk, -1, hs), pk.permute(1, 2, 0)).view(Hk, B, H // Hk, P).permute(1, 0, 2, 3)
    b = torch.matmul(qg, sk.permute(0, 2, 3, 1))
    b = b.masked_fill(torch.arange(S, device=q.device)[None, None, None, :] >= s["length"][:, None, None, None], -math.inf)
    x = torch.cat((a, b), 3)
    m = x.max(3, keepdim=True).values
    e = torch.exp(x - torch.where(m == -math.inf, torch.zeros_like(m), m))
    z = e.sum(3, keepdim=True)
    e = e / torch.where(z == 0, torch.ones_like(z), z)
    o = torch.matmul(e[..., :P].permute(1, 0, 2, 3).reshape(Hk, -1, P), pv.permute(1, 0, 2)).view(Hk, B, H // Hk, hs)
    o = o.permute(1, 0, 2, 3) + torch.matmul(e[..., P:], sv.permute(0, 2, 1, 3))
    return o.reshape(B, H, hs).contiguous()


# ------------------------------------------------------------ 64-bit values
def exact(case, seed):
    s = prepare(case, seed)
    return {"sample": _exact_sample, "topk": _exact_topk, "distill": _exact_distill, "prefix": _exact_prefix}[case["op"]](s)


def _exact_sample(s):
    """Row by row: candidates in falling order (the lower index first), the
    three filters in turn, then the inverse of the cumulative sum."""
    a = {k: None if s[k] is None else s[k].cpu().numpy().astype(np.float64)
         for k in ("logits", "temperature", "top_k", "top_p", "min_p", "u")}
    tokens, logprob = [], []
    for r, x in enumerate(a["logits"]):
        c = np.flatnonzero(x > -np.inf)
        c = c[np.argsort(-x[c], kind="stable")]
        if not a["temperature"][r] > 0:
            tokens.append(c[0])
            logprob.append(0.0)
            continue
        w = np.exp((x[c] - x[c[0]]) / a["temperature"][r])
        if a["top_k"] is not None and a["top_k"][r] > 0:
            c, w = c[: int(a["top_k"][r])], w[: int(a["top_k"][r])]
        if a["top_p"] is not None and a["top_p"][r] < 1:
            n = 1 + int(np.searchsorted(np.cumsum(w), a["top_p"][r] * w.sum()))
            c, w = c[:n], w[:n]
        if a["min_p"] is not None:
            n = int(np.sum(w >= min(1.0, a["min_p"][r])))
            c, w = c[:n], w[:n]
        o = np.argsort(c)
        c, w = c[o], w[o]
        cum = np.cumsum(w)
        at = min(int(np.searchsorted(cum, a["u"][r] * cum[-1], side="right")), len(c) - 1)
        tokens.append(c[at])
        logprob.append(math.log(w[at]) - math.log(cum[-1]))
    return dict(tokens=np.array(tokens, np.int32), logprob=np.array(logprob, np.float64))


def _exact_topk(s):
    return dict(values=torch.topk(s["logits"], s["k"], dim=1).values.double(), indices=None)


def _exact_distill(s):
    tau, alpha, scale = s["tau"], s["alpha"], s["scale"]
    parts = []
    for lo in range(0, s["logits"].shape[0], 1024):
        x = s["logits"][lo:lo + 1024].double()
        ti, tgt = s["top_idx"][lo:lo + 1024].long(), s["targets"][lo:lo + 1024].long()
        n = x.shape[0]
        # the teacher's distribution laid out over the vocabulary
        z = s["top_val"][lo:lo + 1024].double() / tau
        z = torch.where(ti < 0, torch.full_like(z, -math.inf), z)
        soft = (ti >= 0).any(1)
        p = torch.softmax(torch.where(soft[:, None], z, torch.zeros_like(z)), 1) * (ti >= 0)
        ent = torch.where(p > 0, p * torch.log(torch.where(p > 0, p, torch.ones_like(p))), torch.zeros_like(p)).sum(1)
        lq = x / tau - torch.logsumexp(x / tau, 1, keepdim=True)
        row = alpha * tau ** 2 * (ent - (p * lq.gather(1, ti.clamp(min=0))).sum(1))
        l1 = x - torch.logsumexp(x, 1, keepdim=True)
        hard = tgt >= 0
        row = row - (1 - alpha) * torch.where(hard, l1[torch.arange(n, device=x.device), tgt.clamp(min=0)], torch.zeros_like(row))
        d = None
        if s["grad"]:
            d = alpha * tau * soft[:, None] * torch.exp(lq)
            d.scatter_add_(1, ti.clamp(min=0), -alpha * tau * p)
            if alpha < 1:
                h = torch.exp(l1)
                h[torch.arange(n, device=x.device), tgt.clamp(min=0)] -= 1.0
                d += (1 - alpha) * hard[:, None] * h
            d *= scale
        parts.append((row, d))
    row = torch.cat([p[0] for p in parts])
    out = dict(loss=row.sum() * scale, row_loss=row)
    if s["grad"]:
        out["dlogits"] = torch.cat([p[1] for p in parts])
    return out


def _exact_prefix(s):
    """Sequence by sequence: one softmax over the keys that it sees."""
    B, H, hs = s["q"].shape
    group = H // s["pk"].shape[1]
    pk, pv = (s[k].double().repeat_interleave(group, 1).transpose(0, 1) for k in ("pk", "pv"))
    out = torch.zeros(B, H, hs, dtype=torch.float64, device=s["q"].device)
    for b, n in enumerate(s["length"].tolist()):
        k, v = (torch.cat((p, s[name][b, :n].double().repeat_interleave(group, 1).transpose(0, 1)), 1)
                for p, name in ((pk, "sk"), (pv, "sv")))
        if k.shape[1]:
            a = torch.softmax(torch.einsum("hd,hkd->hk", s["q"][b].double(), k) * s["scale"], 1)
            out[b] = torch.einsum("hk,hkd->hd", a, v)
    return out


# ------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "sample":  # every logit read once, an exponential and a sum for each
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + 28 * case["rows"], "flops": 4 * n}
    if op == "topk":  # every logit read once and compared
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + 8 * case["rows"] * case["k"], "flops": n}
    if op == "distill":  # every logit read once, its gradient written once
        n = case["rows"] * case["vocab"]
        both = 2 if case["alpha"] < 1 else 1
        return {"bytes": (8 if case["grad"] else 4) * n + 8 * case["rows"] * case["k"] + 8 * case["rows"],
                "flops": (3 * both + (2 * both if case["grad"] else 0)) * n}
    B, H, Hk, hs, P, S = (case[k] for k in ("batch", "heads", "kv_heads", "hs", "prefix", "suffix"))
    mean = S / 2 if case["ragged"] else S  # suffix lengths are uniform where they differ
    return {"bytes": 4 * (2 * Hk * hs * (P + B * mean) + 2 * B * H * hs) + 4 * B,
            "flops": 4 * B * H * hs * (P + mean)}
