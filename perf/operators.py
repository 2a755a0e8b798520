"""Language-model operators beside the merging path, as measurable cases.

Kinds of cases
  attn    `attention_masked`: softmax attention of packed documents or padded
          sequences, scores capped by a tanh, biased by the distance of query
          and key, masked by document, causality and a prefix that every
          query of the document sees; query heads share key heads.  With
          "train" the gradients of q, k and v belong to the pass.
  prefix  `attention_shared_prefix`: the new tokens of many sequences over one
          prefix that they all share and the keys of their own.
  norm    `norm_gate_residual`: the norm after a block, its gate and residual
          scale, the residual and the next block's norm; with "train" the
          gradients of the activations and of all parameters.

Lengths are texts ("1374,2748"): documents of a packed batch, or the key
lengths of a padded one.
"""
import math
import sys
from pathlib import Path

import torch

own = False

_PKG = str(Path(__file__).resolve().parent.parent / "gpa-vggt_amd")
_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_LOG2E = 1.0 / math.log(2.0)


def listed():
    return [
        # One new token for each of eight sequences over caches of ragged
        # lengths (padded to 4,096): a decode step's attention, where the
        # latency of the call counts.
        dict(name="attn_token", kind="attn", dtype="bf16", batch=8, heads=16, kv_heads=4, d=128, m=1,
             n=4096, docs=1, lens="4096,17,1,2900,801,4095,333,2048", causal=True, prefix=0,
             cap=50.0, slope=False, lse=False, train=False),
        # One token of one sequence whose cache is long: the keys have to be
        # split over the chip.
        dict(name="attn_token_long", kind="attn", dtype="f16", batch=1, heads=8, kv_heads=2, d=64, m=1,
             n=130_001, docs=1, lens="130001", causal=True, prefix=0, cap=0.0, slope=True,
             lse=True, train=False),
        # Scenes of one to four frames (1,374 tokens each) packed on the token
        # axis, every token sees its scene: the aggregator's heads.
        dict(name="attn_scenes", kind="attn", dtype="bf16", batch=1, heads=16, kv_heads=16, d=64, m=10_992,
             n=10_992, docs=4, lens="1374,5496,2748,1374", causal=False, prefix=0, cap=30.0,
             slope=False, lse=True, train=False),
        # A training step of short documents: few rows, where launches count.
        dict(name="attn_train_short", kind="attn", dtype="f16", batch=2, heads=4, kv_heads=4, d=64, m=197,
             n=197, docs=3, lens="60,1,136", causal=True, prefix=5, cap=0.0, slope=True, lse=False,
             train=True),
        # A training step of a decoder: packed documents of odd lengths,
        # capped causal scores, four query heads on each key head.
        dict(name="attn_train", kind="attn", dtype="bf16", batch=2, heads=16, kv_heads=4, d=128, m=4096,
             n=4096, docs=4, lens="1001,63,2000,1032", causal=True, prefix=0, cap=50.0, slope=False,
             lse=False, train=True),
        # A prefix model: the first tokens of the one document see each other,
        # the others are causal, with a bias by distance.
        dict(name="attn_train_prefix", kind="attn", dtype="bf16", batch=1, heads=8, kv_heads=8, d=64, m=8191,
             n=8191, docs=1, lens="8191", causal=True, prefix=1374, cap=0.0, slope=True, lse=False,
             train=True),
        # Four short requests under a system prompt.
        dict(name="prefix_small", kind="prefix", dtype="bf16", batch=4, heads=8, kv_heads=2, d=64, m=1,
             p=512, n=64, own_min=1, own_max=64, cap=0.0, slope=False, lse=False),
        # 64 requests under a long prompt, a decode step.
        dict(name="prefix_decode", kind="prefix", dtype="bf16", batch=64, heads=32, kv_heads=8, d=128, m=1,
             p=8192, n=512, own_min=3, own_max=512, cap=50.0, slope=False, lse=False),
        # Sixteen requests that check four drafted tokens each, fp16, no shared heads.
        dict(name="prefix_draft", kind="prefix", dtype="f16", batch=16, heads=16, kv_heads=16, d=64, m=4,
             p=32_771, n=2048, own_min=4, own_max=2048, cap=0.0, slope=True, lse=True),
        # A decode step's norms: eight rows.
        dict(name="norm_token", kind="norm", dtype="bf16", norm="rms", groups=1, rows=8, c=2048,
             gate="channel", scale=1.0, train=False),
        # The aggregator's width over a scene of eight frames, a gate for each
        # frame, LayerNorm with biases.
        dict(name="norm_frames", kind="norm", dtype="bf16", norm="layer", groups=8, rows=1374, c=1024,
             gate="group", scale=0.5, train=True),
        # A decoder's training step.
        dict(name="norm_train", kind="norm", dtype="bf16", norm="rms", groups=1, rows=16_384, c=4096,
             gate="channel", scale=1.0, train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _split(rng, total, parts):
    """`parts` lengths from one up that add to `total`."""
    cuts = sorted(rng.sample(range(1, total), parts - 1)) if parts > 1 else []
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def draw(rng):
    kind = rng.choice(["attn", "attn", "token", "prefix", "norm"])
    kv = rng.choice([1, 2, 4, 8])
    shape = dict(dtype=rng.choice(["bf16", "bf16", "f16"]), kv_heads=kv, heads=kv * rng.choice([1, 2, 4]),
                 d=rng.choice([64, 128]))
    score = dict(cap=rng.choice([0.0, 20.0, 50.0]), slope=rng.random() < 0.4, lse=rng.random() < 0.3)
    if kind == "attn":
        m = _log(rng, 2, 4600)
        docs = min(rng.choice([1, 1, 2, 5, 9]), m)
        return dict(kind="attn", **shape, batch=rng.choice([1, 1, 2]), m=m, n=m, docs=docs,
                    lens=",".join(map(str, _split(rng, m, docs))), causal=rng.random() < 0.7,
                    prefix=rng.choice([0, 0, 3, 100]), **score, train=rng.random() < 0.6)
    if kind == "token":
        n, batch, m = _log(rng, 1, 60_000), _log(rng, 1, 16), rng.choice([1, 1, 1, 2, 5])
        n = max(n, m)
        return dict(kind="attn", **shape, batch=batch, m=m, n=n, docs=1,
                    lens=",".join(str(max(m, _log(rng, 1, n))) for _ in range(batch)),
                    causal=True, prefix=0, **score, train=False)
    if kind == "prefix":
        m = rng.choice([1, 1, 1, 2, 4])
        n = _log(rng, m, 2000)
        return dict(kind="prefix", **shape, batch=_log(rng, 2, 64), m=m, p=_log(rng, 1, 30_000), n=n,
                    own_min=min(n, max(m, n // 9)), own_max=n, **score)
    c = 8 * _log(rng, 4, 600)
    groups = _log(rng, 1, 40)
    return dict(kind="norm", dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), norm=rng.choice(["rms", "layer"]),
                groups=groups, rows=_log(rng, 1, max(2, 12_000_000 // (groups * c))), c=c,
                gate=rng.choice(["channel", "group", "none"]), scale=rng.choice([1.0, 0.5, 1.7]),
                train=rng.random() < 0.6)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, dt, *shape, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dt)


def _slopes(case):
    """The usual geometric slopes, 2^-8 at the last head."""
    h = case["heads"]
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device="cuda") if case["slope"] else None


def _lens(case):
    return [int(x) for x in case["lens"].split(",")]


def _own_lens(case):
    """Own lengths spread over own_min .. own_max, the longest first."""
    span = case["own_max"] - case["own_min"] + 1
    return [case["own_max"] - (i * 7919) % span for i in range(case["batch"])]


def _offsets(case):
    """(query offsets, key offsets) as a program holds them: the running sums
    of the document lengths, or [0, length] of every padded sequence."""
    lens = _lens(case)
    if case["m"] == case["n"]:
        off = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")
        return off, None
    return None, torch.tensor([[0, x] for x in lens], dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = _gen(seed)
    dt = _DT[case["dtype"]]
    if case["kind"] == "norm":
        grad = case["train"]
        x = _randn(g, dt, case["groups"], case["rows"], case["c"], std=2.0, mean=0.2)
        y = _randn(g, dt, case["groups"], case["rows"], case["c"], std=0.7)
        c = case["c"]
        gate = {"none": lambda: None, "channel": lambda: _randn(g, dt, c, std=0.3, mean=0.5),
                "group": lambda: _randn(g, dt, case["groups"], 1, c, std=0.3, mean=0.5)}[case["gate"]]()
        layer = case["norm"] == "layer"
        par = [_randn(g, dt, c, std=0.2, mean=1.0), _randn(g, dt, c, std=0.1) if layer else None,
               _randn(g, dt, c, std=0.2, mean=1.0), _randn(g, dt, c, std=0.1) if layer else None]
        leaves = [t.requires_grad_(grad) for t in (x, y, gate, *par) if t is not None]
        return dict(case=case, x=x, y=y, gate=gate, par=par, leaves=leaves,
                    gh=_randn(g, dt, *x.shape) if grad else None, gn=_randn(g, dt, *x.shape) if grad else None)
    b, h, hk, m, n, d = (case[i] for i in ("batch", "heads", "kv_heads", "m", "n", "d"))
    # Scores with a spread of 3: past the start of training, before a cap of 50 bites.
    q = _randn(g, dt, b, m, h, d, std=math.sqrt(3.0))
    k = _randn(g, dt, b, n, hk, d, std=math.sqrt(3.0))
    v = _randn(g, dt, b, n, hk, d)
    state = dict(case=case, q=q, k=k, v=v, slopes=_slopes(case))
    if case["kind"] == "prefix":
        return dict(state, pk=_randn(g, dt, hk, case["p"], d, std=math.sqrt(3.0)),
                    pv=_randn(g, dt, hk, case["p"], d),
                    lens=torch.tensor(_own_lens(case), dtype=torch.int32, device="cuda"))
    for t in (q, k, v):
        t.requires_grad_(case["train"])
    qo, ko = _offsets(case)
    return dict(state, qo=qo, ko=ko, go=_randn(g, dt, b, m, h, d) if case["train"] else None)


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _capped(s, cap):
    return torch.tanh(s / cap) * cap if cap else s


def _softmax(s, seen):
    """Weights and log2 of the denominators of rows that may see nothing."""
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top).detach()
    e = torch.exp(s - top)
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total), (top + torch.log(total))[..., 0] * _LOG2E


def _places(off, count):
    """Document number, place in the document and documents' lengths of
    `count` tokens; off [B, docs + 1]."""
    at = torch.arange(count, device="cuda").expand(off.shape[0], count).contiguous()
    doc = torch.searchsorted(off, at, right=True) - 1
    return doc, at - torch.gather(off, 1, doc.clamp(0, off.shape[1] - 2))


def _plain_attention(q, k, v, scale, cap, slopes, causal, prefix, qo, ko):
    """q [B, H, M, D], k and v [B, Hk, N, D]; qo and ko [B, docs + 1]."""
    B, H, M, D = q.shape
    Hk, N = k.shape[1:3]
    docs = qo.shape[1] - 1
    qd, qp = _places(qo, M)
    kd, kp = _places(ko, N)
    longer = (ko.diff() - qo.diff()).gather(1, qd.clamp(0, docs - 1))          # keys before the first query
    qp = qp + longer
    seen = (qd[:, :, None] == kd[:, None, :]) & (qd >= 0)[:, :, None] & (qd < docs)[:, :, None]
    if causal:
        seen = seen & ((kp[:, None, :] <= qp[:, :, None]) | (kp[:, None, :] < prefix))
    s = torch.matmul(q.float().reshape(B, Hk, H // Hk * M, D) * scale, k.float().mT.contiguous())
    s = _capped(s, cap).view(B, H, M, N)
    if slopes is not None:
        s = s - slopes[:, None, None] * (qp[:, :, None] - kp[:, None, :]).abs().float()[:, None]
    w, lse = _softmax(s, seen[:, None])
    o = torch.matmul(w.view(B, Hk, -1, N), v.float().contiguous())
    return o.view(B, H, M, D).to(q.dtype), lse


def _plain_prefix(q, pk, pv, k, v, lens, scale, cap, slopes):
    B, H, M, D = q.shape
    Hk, N = k.shape[1:3]
    G, P = H // Hk, pk.shape[1]
    qf = q.float().view(B, Hk, G * M, D) * scale
    s_p = torch.matmul(qf.transpose(0, 1).reshape(Hk, B * G * M, D), pk.float().mT.contiguous())
    s_p = s_p.view(Hk, B, G, M, P).transpose(0, 1)
    s_o = torch.matmul(qf, k.float().mT.contiguous()).view(B, Hk, G, M, N)
    s = _capped(torch.cat((s_p, s_o), -1), cap).view(B, H, M, P + N)
    place = torch.arange(P + N, device=q.device)
    mine = P + lens.long()[:, None] - M + torch.arange(M, device=q.device)     # [B, M]
    if slopes is not None:
        s = s - slopes[:, None, None] * (mine[:, :, None] - place).abs().float()[:, None]
    seen = (place < P) | (place <= mine[:, :, None])
    w, lse = _softmax(s, seen[:, None])
    w = w.view(B, Hk, G * M, P + N)
    o = torch.matmul(w[..., P:].contiguous(), v.float().contiguous())
    o_p = torch.matmul(w[..., :P].transpose(0, 1).reshape(Hk, B * G * M, P), pv.float())
    o = o + o_p.view(Hk, B, G * M, D).transpose(0, 1)
    return o.reshape(B, H, M, D).to(q.dtype), lse


def _plain_normed(t, weight, bias, layer, eps):
    if layer:
        t = t - t.mean(-1, keepdim=True)
    t = t * torch.rsqrt((t * t).mean(-1, keepdim=True) + eps) * weight.float()
    return t if bias is None else t + bias.float()


def _plain_norm(x, y, gate, par, scale, layer, eps):
    u = _plain_normed(y.float(), par[0], par[1], layer, eps)
    h = x.float() + scale * (u if gate is None else gate.float() * u)
    return h.to(x.dtype), _plain_normed(h, par[2], par[3], layer, eps).to(x.dtype)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _run_norm(state):
    case, x, y, gate, par = (state[i] for i in ("case", "x", "y", "gate", "par"))
    layer = case["norm"] == "layer"
    with torch.set_grad_enabled(case["train"]):
        if own:
            from merging.fused_norms import norm_gate_residual
            out = norm_gate_residual(x, y, par[2], post_weight=par[0], gate=gate, scale=case["scale"],
                                     post_bias=par[1], pre_bias=par[3], kind=case["norm"], eps=1e-6)
        else:
            out = _plain_norm(x, y, gate, par, case["scale"], layer, 1e-6)
        if not case["train"]:
            return list(out)
        return [*(t.detach() for t in out), *torch.autograd.grad(out, state["leaves"], (state["gh"], state["gn"]))]


def _run_prefix(state):
    case = state["case"]
    q, k, v = (state[i].transpose(1, 2) for i in "qkv")
    scale = case["d"] ** -0.5
    if own:
        from merging.fused_attention import attention_shared_prefix
        got = attention_shared_prefix(q, state["pk"], state["pv"], k, v, scale, lengths=state["lens"],
                                      cap=case["cap"] or None, slopes=state["slopes"], return_lse=case["lse"])
        return list(got) if case["lse"] else [got]
    o, lse = _plain_prefix(q, state["pk"], state["pv"], k, v, state["lens"], scale, case["cap"], state["slopes"])
    return [o, lse] if case["lse"] else [o]


def _run_attn(state):
    case, qo, ko = state["case"], state["qo"], state["ko"]
    scale, prefix = case["d"] ** -0.5, case["prefix"] if case["causal"] else 0
    with torch.set_grad_enabled(case["train"]):
        q, k, v = (state[i].transpose(1, 2) for i in "qkv")
        if own:
            from merging.fused_attention import attention_masked
            got = attention_masked(q, k, v, scale, cap=case["cap"] or None, slopes=state["slopes"],
                                   causal=case["causal"], prefix=prefix or None, offsets=qo, k_offsets=ko,
                                   return_lse=case["lse"])
            got = list(got) if case["lse"] else [got]
        else:
            whole = torch.tensor([0, case["m"]], dtype=torch.int32, device="cuda")
            to = (whole if qo is None else qo).long().expand(case["batch"], -1).contiguous()
            ko = to if ko is None else ko.long()
            o, lse = _plain_attention(q, k, v, scale, case["cap"], state["slopes"], case["causal"], prefix, to, ko)
            got = [o, lse] if case["lse"] else [o]
        if not case["train"]:
            return got
        grads = torch.autograd.grad(got[0], [state[i] for i in "qkv"], state["go"].transpose(1, 2))
        return [*(t.detach() for t in got), *grads]


def run(state):
    if own and _PKG not in sys.path:
        sys.path.insert(1, _PKG)
    return {"attn": _run_attn, "prefix": _run_prefix, "norm": _run_norm}[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def _pairs(case):
    """Query-key pairs of one head of the whole batch."""
    def doc(lq, lk):
        if not case["causal"]:
            return lq * lk
        pre = min(case["prefix"], lk)
        first = lk - lq                                       # place of the first query
        # sum over the queries of max(pre, place + 1), at most lk
        low = min(max(pre - first, 0), lq)                    # queries whose prefix reaches past them
        return low * pre + sum(range(first + low + 1, first + lq + 1))
    if case["m"] == case["n"]:
        return case["batch"] * sum(doc(x, x) for x in _lens(case))
    return sum(doc(case["m"], x) for x in _lens(case))


def work(case):
    if case["kind"] == "norm":
        size = 4 if case["dtype"] == "f32" else 2
        each = case["groups"] * case["rows"] * case["c"]
        # forward: x and y in, h and the normed out; backward: x, y and both
        # gradients in, two gradients out.
        return {"bytes": size * each * (10 if case["train"] else 4), "flops": each * (60.0 if case["train"] else 18.0)}
    b, h, hk, m, n, d = (case[i] for i in ("batch", "heads", "kv_heads", "m", "n", "d"))
    rows = 2 * b * h * m * d                                  # bytes of q, and of o
    lse = 4 * b * h * m if case["lse"] else 0
    if case["kind"] == "prefix":
        lens = _own_lens(case)
        keys = 2 * 2 * hk * d * (case["p"] + sum(lens))
        pairs = h * sum(m * case["p"] + m * x - m * (m - 1) // 2 for x in lens)
        return {"bytes": 2 * rows + keys + lse, "flops": 4.0 * d * pairs}
    used = n * b if case["m"] == case["n"] else sum(_lens(case))
    keys = 2 * 2 * hk * d * used
    pairs = h * _pairs(case)
    if not case["train"]:
        return {"bytes": 2 * rows + keys + lse, "flops": 4.0 * d * pairs}
    # and for the gradients do in, dq, dk and dv out; five products for two.
    return {"bytes": 4 * rows + 2 * keys + lse, "flops": 14.0 * d * pairs}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _head64(q, k, v, place, scale, cap, slope, limit, go=None):
    """One head of one document: q [m, D] at `place` [m] sees the keys before
    `limit` [m].  (o, log2 LSE, and with go the gradients of q, k, v)."""
    q, k, v = q.double(), k.double(), v.double()
    j = torch.arange(k.shape[0], device=q.device)
    raw = (q @ k.t()) * scale
    t = torch.tanh(raw / cap) if cap else None
    s = raw if t is None else cap * t
    if slope is not None:
        s = s - slope.double() * (place[:, None] - j).abs().double()
    s = s.masked_fill(j >= limit[:, None], -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[:, None])
    o = p @ v
    if go is None:
        return o, lse * _LOG2E
    go = go.double()
    ds = p * (go @ v.t() - (go * o).sum(-1, keepdim=True)) * scale
    if t is not None:
        ds = ds * (1 - t * t)
    return o, lse * _LOG2E, ds @ k, ds.t() @ q, p.t() @ go


def _attn64(case, seed):
    st = prepare(case, seed)
    b, h, hk, m, n, d = (case[i] for i in ("batch", "heads", "kv_heads", "m", "n", "d"))
    q, k, v = (st[i].detach() for i in "qkv")
    new = lambda *s: torch.zeros(*s, dtype=torch.float64, device="cuda")  # noqa: E731
    o, lse = new(b, h, m, d), new(b, h, m)
    dq, dk, dv = new(b, m, h, d), new(b, n, hk, d), new(b, n, hk, d)
    for i in range(b):
        lens = _lens(case) if m == n else [_lens(case)[i]]
        at = 0
        for lk in lens:
            lq = lk if m == n else m
            rows, keys = slice(at, at + lq), slice(at, at + lk)
            place = torch.arange(lk - lq, lk, device="cuda")
            limit = torch.clamp(place + 1, min=case["prefix"]).clamp(max=lk) if case["causal"] \
                else torch.full_like(place, lk)
            for j in range(h):
                g = j * hk // h
                got = _head64(q[i, rows, j], k[i, keys, g], v[i, keys, g], place, d ** -0.5, case["cap"],
                              None if st["slopes"] is None else st["slopes"][j], limit,
                              st["go"][i, rows, j] if case["train"] else None)
                o[i, j, rows], lse[i, j, rows] = got[:2]
                if case["train"]:
                    dq[i, rows, j] = got[2]
                    dk[i, keys, g] += got[3]
                    dv[i, keys, g] += got[4]
            at += lk
    return [o, *([lse] if case["lse"] else []), *([dq, dk, dv] if case["train"] else [])]


def _prefix64(case, seed):
    st = prepare(case, seed)
    b, h, hk, m, d, p = (case[i] for i in ("batch", "heads", "kv_heads", "m", "d", "p"))
    o = torch.zeros(b, h, m, d, dtype=torch.float64, device="cuda")
    lse = torch.zeros(b, h, m, dtype=torch.float64, device="cuda")
    for i, x in enumerate(_own_lens(case)):
        place = torch.arange(p + x - m, p + x, device="cuda")
        for g in range(hk):
            k = torch.cat((st["pk"][g], st["k"][i, :x, g]))
            v = torch.cat((st["pv"][g], st["v"][i, :x, g]))
            for j in range(g * h // hk, (g + 1) * h // hk):
                o[i, j], lse[i, j] = _head64(st["q"][i, :, j], k, v, place, d ** -0.5, case["cap"],
                                             None if st["slopes"] is None else st["slopes"][j], place + 1)
    return [o, lse] if case["lse"] else [o]


def _norm64_back(dn, t, weight, layer, eps):
    """Gradients of t, weight and bias of a norm of t."""
    mid = t - t.mean(-1, keepdim=True) if layer else t
    inv = 1.0 / torch.sqrt((mid * mid).mean(-1, keepdim=True) + eps)
    hat = mid * inv
    g = dn * weight
    back = g - hat * (g * hat).mean(-1, keepdim=True)
    if layer:
        back = back - g.mean(-1, keepdim=True)
    return back * inv, (dn * hat).sum((0, 1)), dn.sum((0, 1))


def _norm64(case, seed):
    st = prepare(case, seed)
    layer, eps, scale = case["norm"] == "layer", 1e-6, case["scale"]
    x, y = st["x"].detach().double(), st["y"].detach().double()
    w1, b1, w2, b2 = (None if t is None else t.detach().double() for t in st["par"])
    gate = torch.ones((), dtype=torch.float64, device="cuda") if st["gate"] is None else st["gate"].detach().double()

    def normed(t, w, b):
        mid = t - t.mean(-1, keepdim=True) if layer else t
        t = mid / torch.sqrt((mid * mid).mean(-1, keepdim=True) + eps) * w
        return t if b is None else t + b
    u = normed(y, w1, b1)
    h = x + scale * gate * u
    out = [h, normed(h, w2, b2)]
    if case["train"]:
        gh, gn = st["gh"].double(), st["gn"].double()
        dh, dw2, db2 = _norm64_back(gn, h, w2, layer, eps)
        dh = dh + gh
        dy, dw1, db1 = _norm64_back(scale * gate * dh, y, w1, layer, eps)
        out += [dh, dy]
        if case["gate"] == "channel":
            out.append((scale * dh * u).sum((0, 1)))
        elif case["gate"] == "group":
            out.append((scale * dh * u).sum(1, keepdim=True))
        out += [dw1, db1, dw2, db2] if layer else [dw1, dw2]
    return out


def exact(case, seed):
    with torch.no_grad():
        if case["kind"] == "attn":
            return _attn64(case, seed)
        return _prefix64(case, seed) if case["kind"] == "prefix" else _norm64(case, seed)
