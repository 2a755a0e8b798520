"""The operators around attention in a decoder over video tokens, as measurable cases.

Kinds of cases
  turn    `rotate_heads`: the position rotation of one tensor's heads, with one
          to three axes (time, height, width).
  heads   `qk_norm_rotate`: the norm of every query and key head and the
          rotation, in one pass; with "train" the gradients of both and of the
          norms' parameters.
  tree    `draft_tree` and `attention_tree`: a step that checks drafted tokens,
          a tree of them for each sequence, against the sequence's cache.
  linear  `linear_gate_residual`: a projection with bias, activation, gate and
          residual; with "train" the gradients of all its tensors.

Sections are texts ("8,12,12"): the rotated pairs of features of each axis.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

_PKG = str(Path(__file__).resolve().parent.parent / "gpa-vggt_amd")
_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_LOG2E = 1.0 / math.log(2.0)
_EPS = 1e-6


def listed():
    return [
        # Patches of four frames (37 x 37 each) rotated by row and column, each
        # axis in its own half of the head with its own ladder of frequencies:
        # the aggregator's rotation, without its norm.
        dict(name="turn_grid", kind="turn", dtype="bf16", batch=1, tokens=5476, heads=16, d=64, sections="16,16",
             base=100.0, ladder="own", pairing="blocks", places="grid", train=False),
        # fp32, a part of the features rotated, places far behind the start, odd sizes.
        dict(name="turn_far", kind="turn", dtype="f32", batch=3, tokens=1367, heads=6, d=96, sections="20,14",
             base=10000.0, ladder="own", pairing="blocks", places="far", train=True),
        # A decode step: one new token of eight sequences, latency counts.
        dict(name="heads_token", kind="heads", dtype="bf16", batch=8, tokens=1, heads=16, kv_heads=4, d=128,
             norm="rms", sections="64", base=10000.0, ladder="shared", pairing="half", places="far", train=False),
        # Training on a scene of eight frames: time, row and column.
        dict(name="heads_video", kind="heads", dtype="bf16", batch=1, tokens=10_992, heads=16, kv_heads=16, d=64,
             norm="layer", sections="8,12,12", base=10000.0, ladder="shared", pairing="half", places="grid", train=True),
        # A decoder's training step, neighbouring features in pairs.
        dict(name="heads_decoder", kind="heads", dtype="bf16", batch=2, tokens=8192, heads=32, kv_heads=8, d=128,
             norm="rms", sections="64", base=500000.0, ladder="shared", pairing="interleaved", places="line", train=True),
        # Seven drafted tokens of one sequence over a short cache.
        dict(name="tree_small", kind="tree", dtype="bf16", batch=1, heads=8, kv_heads=2, d=64, drafted=7, ragged=False,
             n=700, len_min=611, cap=0.0, slope=False, lse=False),
        # Trees of up to 64 tokens for eight requests, ragged caches.
        dict(name="tree_batch", kind="tree", dtype="bf16", batch=8, heads=32, kv_heads=8, d=128, drafted=64, ragged=True,
             n=8192, len_min=1201, cap=50.0, slope=False, lse=False),
        # One request with a long cache: the keys have to be split over the chip.
        dict(name="tree_long", kind="tree", dtype="f16", batch=1, heads=8, kv_heads=2, d=64, drafted=26, ragged=False,
             n=130_001, len_min=130_001, cap=0.0, slope=True, lse=True),
        # The output projection of a decode step: the weight's bytes.
        dict(name="linear_token", kind="linear", dtype="bf16", rows=8, k=4096, n=4096, bias=False, act="none",
             gate=True, residual=True, train=False),
        # The aggregator's first MLP product over eight frames.
        dict(name="linear_mlp", kind="linear", dtype="bf16", rows=10_992, k=1024, n=4096, bias=True, act="gelu",
             gate=False, residual=False, train=False),
        # Odd sizes in training, all options.
        dict(name="linear_odd", kind="linear", dtype="f16", rows=1374, k=777, n=1001, bias=True, act="silu",
             gate=True, residual=True, train=True),
        # A decoder's training step.
        dict(name="linear_train", kind="linear", dtype="bf16", rows=8192, k=4096, n=4096, bias=True, act="gelu_tanh",
             gate=False, residual=True, train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["turn", "heads", "tree", "linear", "linear"])
    if kind == "linear":
        k, n = _log(rng, 16, 4100), _log(rng, 16, 4100)
        if rng.random() < 0.7:
            k, n = 8 * -(-k // 8), 8 * -(-n // 8)
        return dict(kind="linear", dtype=rng.choice(["bf16", "f16"]), rows=_log(rng, 1, 8000), k=k, n=n,
                    bias=rng.random() < 0.6, act=rng.choice(["none", "gelu", "gelu_tanh", "silu", "relu"]),
                    gate=rng.random() < 0.4, residual=rng.random() < 0.5, train=rng.random() < 0.5)
    if kind == "tree":
        kv, batch = rng.choice([1, 2, 4, 8]), _log(rng, 1, 16)
        n = _log(rng, 1, min(60_000, 190_000 // batch))
        return dict(kind="tree", dtype=rng.choice(["bf16", "bf16", "f16"]), batch=batch, heads=kv * rng.choice([1, 2, 4, 5]),
                    kv_heads=kv, d=rng.choice([64, 128]), drafted=_log(rng, 1, max(2, min(96, 500_000 // (n * batch)))),
                    ragged=rng.random() < 0.5, n=n, len_min=rng.randint(0, n), cap=rng.choice([0.0, 0.0, 30.0]),
                    slope=rng.random() < 0.3, lse=rng.random() < 0.3)
    parts = rng.choice([1, 2, 3])
    d = rng.choice([64, 64, 128, 128, 80, 96, 256, 2 * rng.randint(8, 64)])
    pairs = rng.choice([d // 2, d // 2, max(parts, d // 4)])
    cuts = [0] + sorted(rng.sample(range(1, pairs), parts - 1)) + [pairs]
    if rng.random() < 0.6 and parts == 2:
        cuts[1] = pairs // 2
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 4])
    shape = dict(dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), batch=rng.choice([1, 1, 2, 5]),
                 tokens=_log(rng, 1, 8_000_000 // (5 * heads * d)), heads=heads, d=d)
    turn = dict(sections=",".join(str(b - a) for a, b in zip(cuts, cuts[1:])), base=rng.choice([100.0, 10000.0, 1e6]),
                ladder=rng.choice(["shared", "own"]), pairing=rng.choice(["half", "interleaved", "blocks"]),
                places=rng.choice(["line", "grid", "far"]), train=rng.random() < 0.6)
    if kind == "turn":
        return dict(kind="turn", **shape, **turn)
    return dict(kind="heads", **shape, kv_heads=kv, norm=rng.choice(["rms", "rms", "layer"]), **turn)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _randn(g, dt, *shape, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dt)


def _sections(case):
    return [int(x) for x in case["sections"].split(",")]


def _places(case, g):
    """Positions [B, N, axes]: a line (the same on all axes), frames of a 37 x
    37 grid behind five special tokens (whose axes are 0 but time), or a line
    from a far start for each sequence."""
    b, n, axes = case["batch"], case["tokens"], len(_sections(case))
    at = torch.arange(n, device="cuda")
    if case["places"] == "grid":
        place = at % 1374 - 5
        cols = [at // 1374, torch.where(place < 0, 0, place // 37 + 1), torch.where(place < 0, 0, place % 37 + 1)]
        return torch.stack(cols[3 - axes:], -1).int().expand(b, n, axes).contiguous()
    at = at[None, :, None].expand(b, n, axes)
    if case["places"] == "far":
        at = at + torch.randint(100_000, 4_000_000, (b, 1, axes), generator=g, device="cuda")
    return at.int().contiguous()


def _pairs_of(case):
    """(first feature, second feature, axis, frequency) of every rotated pair, as lists."""
    sections, base = _sections(case), case["base"]
    total, first, second, axis, freq = sum(sections), [], [], [], []
    for a, size in enumerate(sections):
        begin = len(first)
        for i in range(size):
            j = begin + i
            x, y = {"half": (j, total + j), "interleaved": (2 * j, 2 * j + 1),
                    "blocks": (2 * begin + i, 2 * begin + size + i)}[case["pairing"]]
            first.append(x)
            second.append(y)
            axis.append(a)
            freq.append(base ** (-i / size) if case["ladder"] == "own" else base ** (-j / total))
    return first, second, axis, freq


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, grad = _DT[case["dtype"]], case.get("train", False)
    if case["kind"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        maybe = lambda want, **s: _randn(g, dt, n, **s).requires_grad_(grad) if want else None  # noqa: E731
        st = dict(case=case, x=_randn(g, dt, m, k).requires_grad_(grad),
                  w=_randn(g, dt, n, k, std=k ** -0.5).requires_grad_(grad), bias=maybe(case["bias"], std=0.3),
                  gate=maybe(case["gate"], std=0.2, mean=0.4),
                  residual=_randn(g, dt, m, n, std=2.0).requires_grad_(grad) if case["residual"] else None)
        st["leaves"] = [st[i] for i in ("x", "w", "bias", "gate", "residual") if st[i] is not None]
        return dict(st, gy=_randn(g, dt, m, n) if grad else None)
    b, h, d = case["batch"], case["heads"], case["d"]
    if case["kind"] == "tree":
        # Drafted tokens hang on earlier ones: most on one of the last few, some on the root.
        t, n, hk, rng = case["drafted"], case["n"], case["kv_heads"], random.Random(int(seed))
        parents = [[max(-1, i - 1 - int(rng.expovariate(0.4))) for i in range(t)] for _ in range(b)]
        lens = [n - (i * 7919) % (n - case["len_min"] + 1) for i in range(b)]
        sizes = [max(1, t - (i * 5) % t) for i in range(b)] if case["ragged"] else None
        ints = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        return dict(case=case, q=_randn(g, dt, b, t, h, d, std=math.sqrt(3.0)),
                    k=_randn(g, dt, b, t, hk, d, std=math.sqrt(3.0)), v=_randn(g, dt, b, t, hk, d),
                    ck=_randn(g, dt, b, hk, n, d, std=math.sqrt(3.0)), cv=_randn(g, dt, b, hk, n, d),
                    parents=ints(parents), lens=ints(lens), sizes=ints(sizes),
                    slopes=torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device="cuda")
                    if case["slope"] else None)
    first, second, axis, freq = _pairs_of(case)
    n, kinds = case["tokens"], case["kind"] == "heads"
    st = dict(case=case, places=_places(case, g), sections=tuple(_sections(case)), first=torch.tensor(first, device="cuda"),
              second=torch.tensor(second, device="cuda"), axis=torch.tensor(axis, dtype=torch.int32, device="cuda"),
              freq=torch.tensor(freq, dtype=torch.float64, device="cuda"))
    if not kinds:
        x = _randn(g, dt, b, n, h, d, std=1.5).requires_grad_(grad)
        return dict(st, x=[x], par=[], grads=[_randn(g, dt, b, n, h, d)] if grad else None)
    # Queries and keys as they lie in a block's fused projection.
    hk = case["kv_heads"]
    qkv = _randn(g, dt, b, n, h + 2 * hk, d, std=1.5, mean=0.1)
    x = [qkv[:, :, :h].detach().requires_grad_(grad), qkv[:, :, h:h + hk].detach().requires_grad_(grad)]
    par = [_randn(g, dt, d, std=0.2, mean=1.0).requires_grad_(grad) for _ in range(2)]
    if case["norm"] == "layer":
        par += [_randn(g, dt, d, std=0.1).requires_grad_(grad) for _ in range(2)]
    return dict(st, x=x, par=par, grads=[_randn(g, dt, *t.shape) for t in x] if grad else None)


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _plain_turn(x, st):
    """x [B, N, H, D] in fp32, rotated."""
    angle = st["places"].double()[..., st["axis"]] * st["freq"]               # [B, N, pairs]
    cos, sin = torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]
    a, b = x[..., st["first"]], x[..., st["second"]]
    x = x.index_copy(3, st["first"], a * cos - b * sin)
    return x.index_copy(3, st["second"], b * cos + a * sin)


def _plain_normed(x, weight, bias, layer):
    x = x.float()
    if layer:
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * weight.float()
    return x if bias is None else x + bias.float()


def _plain_tree(parents, lens, sizes):
    """(positions [B, T], which drafted tokens each of them sees [B, T, T])."""
    T = parents.shape[1]
    at = torch.arange(T, device="cuda")
    step = (parents[:, :, None] == at).double() + torch.eye(T, dtype=torch.float64, device="cuda")
    seen = torch.matrix_power(step, T) > 0
    depth = seen.sum(-1) - 1
    fine = torch.ones_like(depth, dtype=torch.bool) if sizes is None else at < sizes[:, None]
    return torch.where(fine, lens[:, None] + depth, 0).int(), seen & fine[:, :, None], fine


def _plain_tree_attention(st, scale):
    case = st["case"]
    b, h, hk, d, t, n = (case[i] for i in ("batch", "heads", "kv_heads", "d", "drafted", "n"))
    at, tail, fine = _plain_tree(st["parents"], st["lens"], st["sizes"])
    q = st["q"].float().transpose(1, 2).reshape(b, hk, h // hk * t, d) * scale
    k = torch.cat((st["ck"], st["k"].transpose(1, 2)), 2).float()
    v = torch.cat((st["cv"], st["v"].transpose(1, 2)), 2).float()
    s = torch.matmul(q, k.mT.contiguous()).view(b, h, t, n + t)
    if case["cap"]:
        s = torch.tanh(s / case["cap"]) * case["cap"]
    if st["slopes"] is not None:
        place = torch.cat((torch.arange(n, device="cuda").expand(b, n), at), 1)
        s = s - st["slopes"][:, None, None] * (at[:, :, None] - place[:, None]).abs().float()[:, None]
    cache = (torch.arange(n, device="cuda") < st["lens"][:, None])[:, None] & fine[:, :, None]
    s = s.masked_fill(~torch.cat((cache, tail), 2)[:, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = torch.exp(s - top)
    total = e.sum(-1, keepdim=True)
    w = e / torch.where(total == 0, torch.ones_like(total), total)
    o = torch.matmul(w.view(b, hk, h // hk * t, n + t), v).view(b, h, t, d)
    return at, o.to(st["q"].dtype), (top + torch.log(total))[..., 0] * _LOG2E


def _plain_act(z, act):
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return torch.where(z > 0, z, torch.zeros_like(z)) if act == "relu" else z


def _plain_linear(x, w, bias, act, gate, residual):
    z = torch.matmul(x.float(), w.float().t())
    if bias is not None:
        z = z + bias.float()
    y = _plain_act(z, act)
    if gate is not None:
        y = y * gate.float()
    return (y if residual is None else y + residual.float()).to(x.dtype)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _run_linear(st):
    case = st["case"]
    with torch.set_grad_enabled(case["train"]):
        if own:
            from merging.fused_linear import linear_gate_residual
            y = linear_gate_residual(st["x"], st["w"], st["bias"], gate=st["gate"], residual=st["residual"],
                                     activation=None if case["act"] == "none" else case["act"])
        else:
            y = _plain_linear(st["x"], st["w"], st["bias"], case["act"], st["gate"], st["residual"])
        return [y.detach(), *torch.autograd.grad(y, st["leaves"], st["gy"])] if case["train"] else [y]


def _run_tree(st):
    case = st["case"]
    if own:
        from merging.fused_attention import attention_tree, draft_tree
        at, seen = draft_tree(st["parents"], st["lens"], sizes=st["sizes"])
        q, k, v = (st[i].transpose(1, 2) for i in "qkv")
        got = attention_tree(q, st["ck"], st["cv"], k, v, case["d"] ** -0.5, lengths=st["lens"], seen=seen,
                             cap=case["cap"] or None, slopes=st["slopes"], return_lse=case["lse"])
        return [at, *got] if case["lse"] else [at, got]
    at, o, lse = _plain_tree_attention(st, case["d"] ** -0.5)
    return [at, o, lse] if case["lse"] else [at, o]


def _run_rotary(st):
    case, par = st["case"], st["par"]
    with torch.set_grad_enabled(case["train"]):
        if own:
            from merging.fused_rotary import RotaryAxes, qk_norm_rotate, rotate_heads
            x = [t.transpose(1, 2) for t in st["x"]]
            rotary = RotaryAxes(st["freq"], st["axis"], case["pairing"], st["sections"])
            if case["kind"] == "turn":
                out = [rotate_heads(x[0], st["places"], rotary)]
            else:
                out = qk_norm_rotate(*x, st["places"], rotary, q_weight=par[0], k_weight=par[1],
                                     q_bias=par[2] if par[2:] else None, k_bias=par[3] if par[2:] else None,
                                     kind=case["norm"], eps=_EPS)
            out = [t.transpose(1, 2) for t in out]
        elif case["kind"] == "turn":
            out = [_plain_turn(st["x"][0].float(), st).to(st["x"][0].dtype)]
        else:
            out = [_plain_turn(_plain_normed(x, w, b, case["norm"] == "layer"), st).to(x.dtype)
                   for x, w, b in zip(st["x"], par, par[2:] or (None, None))]
        if not case["train"]:
            return out
        return [*(t.detach() for t in out), *torch.autograd.grad(out, st["x"] + par, st["grads"])]


def run(st):
    if own and _PKG not in sys.path:
        sys.path.insert(1, _PKG)
    return {"linear": _run_linear, "tree": _run_tree}.get(st["case"]["kind"], _run_rotary)(st)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        once = m * k + n * k
        if not case["train"]:
            return {"bytes": size * (once + m * n * (2 if case["residual"] else 1)), "flops": 2.0 * m * n * k}
        # and the output's gradient in, those of x and w out.  (The residual's is the output's.)
        return {"bytes": size * (2 * once + m * n * (3 if case["residual"] else 2)), "flops": 6.0 * m * n * k}
    b, h, d = case["batch"], case["heads"], case["d"]
    if case["kind"] == "tree":
        t, n = case["drafted"], case["n"]
        keys = sum(n - (i * 7919) % (n - case["len_min"] + 1) for i in range(b))
        rows = [max(1, t - (i * 5) % t) if case["ragged"] else t for i in range(b)]
        pairs = sum(r * (n - (i * 7919) % (n - case["len_min"] + 1)) for i, r in enumerate(rows))
        return {"bytes": 2 * (2 * case["kv_heads"] * d * (keys + b * t) + 2 * b * t * h * d) + (4 * b * t * h if case["lse"] else 0),
                "flops": 4.0 * d * h * pairs}
    values = b * case["tokens"] * d * (h + case.get("kv_heads", 0))
    norm = case["kind"] == "heads"
    # forward: in and out; backward: the gradient in and out, under a norm the input too.
    passes = (5 if norm else 4) if case["train"] else 2
    return {"bytes": size * values * passes + 4 * b * case["tokens"] * len(_sections(case)),
            "flops": values * (30.0 if norm else 8.0) * (0.5 if not case["train"] else 1.0)}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _linear64(case, st):
    d = lambda t: None if t is None else t.detach().double()  # noqa: E731
    x, w, bias, gate, residual, gy = (d(st[i]) for i in ("x", "w", "bias", "gate", "residual", "gy"))
    z = x @ w.t() + (0.0 if bias is None else bias)
    act = case["act"]
    if act == "gelu":
        cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
        y, slope = z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    elif act == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        sig = torch.sigmoid(2.0 * c * (z + 0.044715 * z ** 3))
        y, slope = z * sig, sig + z * sig * (1.0 - sig) * 2.0 * c * (1.0 + 3.0 * 0.044715 * z * z)
    elif act == "silu":
        sig = torch.sigmoid(z)
        y, slope = z * sig, sig + z * sig * (1.0 - sig)
    elif act == "relu":
        y, slope = z.clamp(min=0.0), (z > 0).double()
    else:
        y, slope = z, torch.ones_like(z)
    out = [(y if gate is None else y * gate) + (0.0 if residual is None else residual)]
    if case["train"]:
        dz = gy * slope * (1.0 if gate is None else gate)
        out += [dz @ w, dz.t() @ x]
        out += [dz.sum(0)] if bias is not None else []
        out += [(gy * y).sum(0)] if gate is not None else []
        out += [gy] if residual is not None else []
    return out


def _tree64(case, st):
    b, h, hk, d, t, n = (case[i] for i in ("batch", "heads", "kv_heads", "d", "drafted", "n"))
    o = torch.zeros(b, h, t, d, dtype=torch.float64, device="cuda")
    lse = torch.full((b, h, t), -math.inf, dtype=torch.float64, device="cuda")
    for i in range(b):
        parents, length = st["parents"][i].tolist(), int(st["lens"][i])
        size = t if st["sizes"] is None else int(st["sizes"][i])
        chains = [[] for _ in range(t)]                       # a token's ancestors and itself
        for j in range(size):
            chains[j] = (chains[parents[j]] if parents[j] >= 0 else []) + [j]
        sees = torch.zeros(size, length + t, dtype=torch.bool)
        sees[:, :length] = True
        for j in range(size):
            sees[j, [length + x for x in chains[j]]] = True
        sees = sees.cuda()
        mine = torch.tensor([length + len(c) - 1 for c in chains], device="cuda")
        place = torch.cat((torch.arange(length, device="cuda"), mine)).double()
        for j in range(h):
            kv = j * hk // h
            k = torch.cat((st["ck"][i, kv, :length], st["k"][i, :, kv])).double()
            v = torch.cat((st["cv"][i, kv, :length], st["v"][i, :, kv])).double()
            s = st["q"][i, :size, j].double() @ k.t() * d ** -0.5
            if case["cap"]:
                s = case["cap"] * torch.tanh(s / case["cap"])
            if st["slopes"] is not None:
                s = s - st["slopes"][j].double() * (mine[:size, None].double() - place).abs()
            s = s.masked_fill(~sees, -math.inf)
            lse[i, j, :size] = torch.logsumexp(s, -1) * _LOG2E
            o[i, j, :size] = torch.softmax(s, -1) @ v
    return [None, o, lse] if case["lse"] else [None, o]


def _turned64(x, st, sign):
    """x [B, N, H, D] rotated by sign times the angles, as complex numbers."""
    angle = st["places"].double()[..., st["axis"]] * st["freq"] * sign
    z = torch.complex(x[..., st["first"]], x[..., st["second"]]) * torch.polar(torch.ones_like(angle), angle)[:, :, None]
    x = x.clone()
    x[..., st["first"]], x[..., st["second"]] = z.real, z.imag
    return x


def _rotary64(case, st):
    out, dx, dw, db = [], [], [], []
    layer = case.get("norm") == "layer"
    for i, x in enumerate(st["x"]):
        x = x.detach().double()
        if case["kind"] == "turn":
            out.append(_turned64(x, st, 1.0))
            dx += [_turned64(st["grads"][i].double(), st, -1.0)] if case["train"] else []
            continue
        w = st["par"][i].detach().double()
        mid = x - x.mean(-1, keepdim=True) if layer else x
        inv = 1.0 / torch.sqrt((mid * mid).mean(-1, keepdim=True) + _EPS)
        hat = mid * inv
        n = hat * w + (st["par"][2 + i].detach().double() if layer else 0.0)
        out.append(_turned64(n, st, 1.0))
        if case["train"]:
            dn = _turned64(st["grads"][i].double(), st, -1.0)
            dw.append((dn * hat).sum((0, 1, 2)))
            db += [dn.sum((0, 1, 2))] if layer else []
            g = dn * w
            back = g - hat * (g * hat).mean(-1, keepdim=True)
            dx.append((back - g.mean(-1, keepdim=True) if layer else back) * inv)
    return out + dx + dw + db


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {"linear": _linear64, "tree": _tree64}.get(case["kind"], _rotary64)(case, st)
