"""Operators of a training step beside the contractions and the attention core, as cases that can be timed.

Three kinds, each through the public operator-level entry points:

  scan      the gated linear recurrence of a sequence-mixing layer over packed sequences (ts2_op_recurrence_forward,
            ts2_op_recurrence_backward): h[t] = a h[t-1] + (1 - a) x[t], a = sigmoid(gate[t]), per channel
  balance   the load-balance term of a mixture-of-experts router with the experts' counts and its gradient
            (ts2_op_moe_balance_forward, ts2_op_moe_balance_backward)
  orth      the orthogonalised update of weight matrices by Newton-Schulz products (ts2_op_orthogonalize)

Gates are normal around a decay of 0.9, router logits are normal with some experts preferred, and the matrices to
orthogonalise are a few strong directions over noise, as accumulated gradients are."""
import math

import torch

own = False  # True: the framework's operators, False: the plain form

TYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
COEF = (3.4445, -4.7750, 2.0315)  # a s + b s^3 + c s^5 on every singular value
STEPS = 5


def _scan(**kw):
    return dict(dict(op="scan", dir="forward", type="f16", tokens=77, dim=256, seqs=1, carry=False, pad=0), **kw)


def _balance(**kw):
    return dict(dict(op="balance", dir="train", type="f32", tokens=512, experts=8, selected=2, masked=False), **kw)


def _orth(**kw):
    return dict(dict(op="orth", type="f32", batch=1, rows=128, cols=256), **kw)


def listed():
    return [
        # one short text through a narrow model: latency
        _scan(name="scan_short_f16"),
        # the forward pass of a training step: 64 documents of about 1024 tokens packed one behind the other, 768 channels
        _scan(name="scan_packed_bf16", type="bf16", tokens=65536, dim=768, seqs=64),
        # a document longer than a batch goes on from the state that the last batch left, fp32
        _scan(name="scan_long_f32", type="f32", tokens=32768, dim=512, carry=True),
        # the backward pass of a ragged micro-batch, an odd number of channels, a padded end, gradients of the carried states
        _scan(name="scan_ragged_backward_f16", dir="backward", tokens=5001, dim=333, seqs=7, carry=True, pad=19),
        # the backward pass of a wide model with long sequences
        _scan(name="scan_wide_backward_bf16", dir="backward", type="bf16", tokens=32768, dim=2048, seqs=8),
        # the smallest mixture: 4 x 128 tokens, 8 experts
        _balance(name="balance_small_f32"),
        # a mixture layer of a training step, 32 experts, 2 selected, 32 x 1024 tokens
        _balance(name="balance_moe_f32", tokens=32768, experts=32),
        # many small experts, 8 selected, padded sequences, 16-bit logits
        _balance(name="balance_wide_bf16", type="bf16", tokens=65537, experts=128, selected=8, masked=True),
        # one matrix of the smallest model: a chain of tiny products
        _orth(name="orth_small_f32"),
        # matrices of sizes that no tile divides, 16-bit momentum, more rows than columns
        _orth(name="orth_ragged_bf16", type="bf16", batch=3, rows=1000, cols=333),
        # the expert matrices of a mixture layer: 32 of 1024 x 1024
        _orth(name="orth_experts_f32", batch=32, rows=1024, cols=1024),
        # the expansion matrix of a wide model, [8192][2048]
        _orth(name="orth_wide_f32", rows=8192, cols=2048),
    ]


def work(case):
    c = case
    if c["op"] == "scan":
        n = (c["tokens"] - c["pad"]) * c["dim"]
        state = 8.0 * c["seqs"] * c["dim"] if c["carry"] else 0.0
        if c["dir"] == "forward":  # gate and x in, h out; exponential, sum, quotient, two products with a sum
            return {"bytes": 3.0 * SIZE[c["type"]] * n + state, "flops": 8.0 * n}
        return {"bytes": 6.0 * SIZE[c["type"]] * n + 1.5 * state, "flops": 16.0 * n}
    if c["op"] == "balance":
        n = c["tokens"] * c["experts"]
        tables = 4.0 * c["tokens"] * c["selected"] + (c["tokens"] if c["masked"] else 0)
        if c["dir"] == "count":
            return {"bytes": SIZE[c["type"]] * n + tables, "flops": 5.0 * n}
        return {"bytes": 2.0 * SIZE[c["type"]] * n + tables, "flops": 9.0 * n}
    n, m = min(c["rows"], c["cols"]), max(c["rows"], c["cols"])
    # X X^T and its square are symmetric: half of each
    return {"bytes": (SIZE[c["type"]] + 2.0) * c["batch"] * n * m,
            "flops": c["batch"] * STEPS * (1.0 * n * n * m + 1.0 * n * n * n + 2.0 * n * n * m)}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _scan_state(c, gen):
    T, D, n, t = c["tokens"], c["dim"], c["seqs"], TYPE[c["type"]]
    used = T - c["pad"]
    randn = lambda *shape: torch.randn(shape, device="cuda", generator=gen)
    cuts = torch.randperm(used - 1, device="cuda", generator=gen)[:n - 1].sort().values + 1 if n > 1 else torch.empty(0, device="cuda")
    ptr = torch.cat([torch.zeros(1, device="cuda"), cuts, torch.full((1,), used, device="cuda")]).to(torch.int32)
    st = {"c": c, "ptr": ptr, "gate": (2.2 + 1.5 * randn(T, D)).to(t), "x": randn(T, D).to(t),
          "h0": randn(n, D) if c["carry"] else None}
    if c["dir"] == "forward":
        st.update(h=torch.zeros((T, D), device="cuda", dtype=t), h_last=torch.zeros((n, D), device="cuda") if c["carry"] else None)
    else:  # what the forward pass left
        st.update(h=_scan_forward_plain(st)["h"], dh=randn(T, D).to(t), dh_last=randn(n, D) if c["carry"] else None)
        st.update(dgate=torch.zeros((T, D), device="cuda", dtype=t), dx=torch.zeros((T, D), device="cuda", dtype=t),
                  dh0=torch.zeros((n, D), device="cuda") if c["carry"] else None)
    return st


def _balance_state(c, gen):
    T, E, t = c["tokens"], c["experts"], TYPE[c["type"]]
    logits = torch.randn((T, E), device="cuda", generator=gen) + 0.7 * torch.randn((E,), device="cuda", generator=gen)
    logits = logits.to(t)
    ids = logits.float().topk(c["selected"], dim=1).indices.to(torch.int32).contiguous()
    mask = (torch.rand(T, device="cuda", generator=gen) < 0.9).to(torch.uint8) if c["masked"] else None
    return {"c": c, "logits": logits, "ids": ids, "mask": mask, "counts": torch.zeros(E + 1, device="cuda", dtype=torch.int32),
            "prob": torch.zeros(E, device="cuda"), "loss": torch.zeros(1, device="cuda"),
            "dloss": torch.full((1,), 0.01, device="cuda"), "dlogits": torch.zeros((T, E), device="cuda", dtype=t)}


def _orth_state(c, gen):
    b, r, k = c["batch"], c["rows"], c["cols"]
    strong = min(8, r, k)
    g = torch.randn((b, r, strong), device="cuda", generator=gen) @ torch.randn((b, strong, k), device="cuda", generator=gen)
    g = (0.5 * g + torch.randn((b, r, k), device="cuda", generator=gen)) * 1e-3
    return {"c": c, "g": g.to(TYPE[c["type"]]), "out": torch.zeros((b, r, k), device="cuda", dtype=torch.bfloat16)}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return {"scan": _scan_state, "balance": _balance_state, "orth": _orth_state}[case["op"]](case, gen)


# ---- the plain form -------------------------------------------------------------------------------------------------

def _starts(ptr, T):
    """Per token: whether a sequence starts there; and the starts and ends of the sequences."""
    first = ptr[:-1].long()
    s = torch.zeros(T, device="cuda", dtype=torch.bool)
    s[first] = True
    return s, first, ptr[1:].long() - 1


def _doubling(a, b):
    """h[t] = a[t] h[t-1] + b[t] along dim 0, h[-1] = 0, by doubling the length of what is joined."""
    k = 1
    while k < a.shape[0]:  # log2(tokens) steps over whole tensors
        b = torch.cat([b[:k], b[k:] + a[k:] * b[:-k]])
        a = torch.cat([a[:k], a[k:] * a[:-k]])
        k *= 2
    return b


def _scan_forward_plain(st):
    c, T = st["c"], st["c"]["tokens"]
    used = T - c["pad"]
    s, first, last = _starts(st["ptr"], used)
    g = st["gate"][:used].float()
    a, b = 1 / (1 + torch.exp(-g)), 1 / (1 + torch.exp(g)) * st["x"][:used].float()
    if c["carry"]:
        b[first] += a[first] * st["h0"]
    h = _doubling(torch.where(s[:, None], 0.0, a), b)
    out = torch.zeros((T, c["dim"]), device="cuda", dtype=TYPE[c["type"]])
    out[:used] = h.to(out.dtype)
    return {"h": out, "h_last": h[last]} if c["carry"] else {"h": out}


def _scan_backward_plain(st):
    c, T = st["c"], st["c"]["tokens"]
    used = T - c["pad"]
    s, first, last = _starts(st["ptr"], used)
    g, x = st["gate"][:used].float(), st["x"][:used].float()
    a, keep = 1 / (1 + torch.exp(-g)), 1 / (1 + torch.exp(g))
    before = torch.cat([torch.zeros_like(g[:1]), st["h"][:used - 1].float()])
    before = torch.where(s[:, None], 0.0, before)
    dh = st["dh"][:used].float()
    if c["carry"]:
        before[first] = st["h0"]
        dh[last] += st["dh_last"]
    after = torch.cat([torch.where(s[1:, None], 0.0, a[1:]), torch.zeros_like(g[:1])])
    e = _doubling(after.flip(0), dh.flip(0)).flip(0)
    out = {n: torch.zeros((T, c["dim"]), device="cuda", dtype=TYPE[c["type"]]) for n in ("dgate", "dx")}
    out["dgate"][:used] = (a * keep * (before - x) * e).to(out["dx"].dtype)
    out["dx"][:used] = (keep * e).to(out["dx"].dtype)
    if c["carry"]:
        out["dh0"] = a[first] * e[first]
    return out


def _balance_plain(st):
    c = st["c"]
    T, E, k = c["tokens"], c["experts"], c["selected"]
    l = st["logits"].float()
    on = st["mask"].bool() if c["masked"] else torch.ones(T, device="cuda", dtype=torch.bool)
    p = torch.exp(l - l.amax(dim=1, keepdim=True))
    p = p / p.sum(dim=1, keepdim=True) * on[:, None]
    n = on.sum()
    counts = ((st["ids"][:, :, None] == torch.arange(E, device="cuda")) & on[:, None, None]).sum(dim=(0, 1))
    share = counts.double() * E / (k * n)
    prob = p.double().sum(dim=0) / n
    out = {"counts": torch.cat([counts, n[None]]).to(torch.int32), "prob": prob.float(), "loss": (share * prob).sum()[None].float()}
    if c["dir"] == "train":
        f = (share - share.mean()).float()
        out["dlogits"] = (st["dloss"] / n * p * (f - (p * f).sum(dim=1, keepdim=True))).to(TYPE[c["type"]])
    return out


def _orth_plain(st):
    a, b, k = COEF
    x = st["g"].float()
    x = x / torch.sqrt((x * x).double().sum(dim=(1, 2), keepdim=True)).float()
    tall = x.shape[1] > x.shape[2]
    x = x.transpose(1, 2) if tall else x
    for _ in range(STEPS):
        s = x @ x.transpose(1, 2)
        x = a * x + (b * s + k * (s @ s)) @ x
    return {"out": (x.transpose(1, 2) if tall else x).to(torch.bfloat16)}


# ---- one pass -------------------------------------------------------------------------------------------------------

def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(name, *args):
    import ctypes as C

    from tscale2_b200 import capi
    lib = capi.load_library()
    rc = getattr(lib, name)(0, C.c_void_p(torch.cuda.current_stream().cuda_stream), *args)
    if rc != capi.TS2_OK:
        raise capi.Ts2Error(rc, lib.ts2_last_error(None).decode())


def _kind(c):
    from tscale2_b200 import capi
    return {"f32": capi.OUT_F32, "f16": capi.OUT_F16, "bf16": capi.OUT_BF16}[c["type"]]


def _scan_own(st):
    c, D = st["c"], st["c"]["dim"]
    if c["dir"] == "forward":
        _call("ts2_op_recurrence_forward", _kind(c), _ptr(st["gate"]), D, _ptr(st["x"]), D, c["tokens"], D, c["seqs"], _ptr(st["ptr"]),
              _ptr(st["h0"]), _ptr(st["h"]), D, _ptr(st["h_last"]))
        return {n: st[n] for n in ("h", "h_last") if st[n] is not None}
    _call("ts2_op_recurrence_backward", _kind(c), _ptr(st["gate"]), D, _ptr(st["x"]), D, _ptr(st["h"]), D, c["tokens"], D, c["seqs"],
          _ptr(st["ptr"]), _ptr(st["h0"]), _ptr(st["dh"]), D, _ptr(st["dh_last"]), _ptr(st["dgate"]), D, _ptr(st["dx"]), D, _ptr(st["dh0"]))
    return {n: st[n] for n in ("dgate", "dx", "dh0") if st[n] is not None}


def _balance_own(st):
    c, E = st["c"], st["c"]["experts"]
    _call("ts2_op_moe_balance_forward", _kind(c), _ptr(st["logits"]), E, c["tokens"], E, c["selected"], _ptr(st["ids"]), _ptr(st["mask"]),
          _ptr(st["counts"]), _ptr(st["prob"]), _ptr(st["loss"]))
    out = {n: st[n] for n in ("counts", "prob", "loss")}
    if c["dir"] == "train":
        _call("ts2_op_moe_balance_backward", _kind(c), _ptr(st["logits"]), E, c["tokens"], E, c["selected"], _ptr(st["mask"]),
              _ptr(st["counts"]), _ptr(st["dloss"]), 1.0, _ptr(st["dlogits"]), E, 0)
        out["dlogits"] = st["dlogits"]
    return out


def _orth_own(st):
    import ctypes as C

    c = st["c"]
    r, k = c["rows"], c["cols"]
    _call("ts2_op_orthogonalize", _kind(c), _ptr(st["g"]), k, r * k, c["batch"], r, k, (C.c_float * 3)(*COEF), STEPS, 1.0, _ptr(st["out"]), k,
          r * k)
    return {"out": st["out"]}


def run(state):
    op = state["c"]["op"]
    if own:
        return {"scan": _scan_own, "balance": _balance_own, "orth": _orth_own}[op](state)
    if op == "scan":
        return (_scan_forward_plain if state["c"]["dir"] == "forward" else _scan_backward_plain)(state)
    return _balance_plain(state) if op == "balance" else _orth_plain(state)


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def _scan_exact(st):
    c, T, D = st["c"], st["c"]["tokens"], st["c"]["dim"]
    ptr = st["ptr"].tolist()
    a = torch.sigmoid(st["gate"].double())
    keep = torch.sigmoid(-st["gate"].double())
    x = st["x"].double()
    zero = torch.zeros(D, device="cuda", dtype=torch.float64)
    n = c["seqs"]
    if c["dir"] == "forward":
        h, h_last = torch.zeros((T, D), device="cuda", dtype=torch.float64), torch.zeros((n, D), device="cuda", dtype=torch.float64)
        u = keep * x
        for s in range(n):
            now = st["h0"][s].double() if c["carry"] else zero
            for t in range(ptr[s], ptr[s + 1]):
                now = torch.addcmul(u[t], a[t], now)
                h[t] = now
            h_last[s] = now
        return {"h": h, "h_last": h_last} if c["carry"] else {"h": h}
    out = {k: torch.zeros((T, D), device="cuda", dtype=torch.float64) for k in ("dgate", "dx")}
    dh0, e = torch.zeros((n, D), device="cuda", dtype=torch.float64), torch.zeros((T, D), device="cuda", dtype=torch.float64)
    before = torch.zeros((T, D), device="cuda", dtype=torch.float64)
    dh = st["dh"].double()
    for s in range(n):
        b, f = ptr[s], ptr[s + 1]
        before[b + 1:f] = st["h"][b:f - 1].double()
        before[b] = st["h0"][s].double() if c["carry"] else zero
        now = st["dh_last"][s].double() if c["carry"] else zero
        for t in range(f - 1, b - 1, -1):
            now = now + dh[t]
            e[t] = now
            now = now * a[t]
        dh0[s] = now
    out["dgate"] = e * a * keep * (before - x)
    out["dx"] = e * keep
    out["dgate"][ptr[n]:], out["dx"][ptr[n]:] = 0, 0
    if c["carry"]:
        out["dh0"] = dh0
    return out


def _balance_exact(st):
    c = st["c"]
    rows = torch.nonzero(st["mask"])[:, 0] if c["masked"] else torch.arange(c["tokens"], device="cuda")
    l = st["logits"].double().requires_grad_(True)
    counts = torch.bincount(st["ids"][rows].flatten().long(), minlength=c["experts"])
    prob = torch.softmax(l[rows], dim=1).mean(dim=0)
    loss = c["experts"] * (counts.double() / (c["selected"] * len(rows)) * prob).sum()
    out = {"counts": torch.cat([counts, torch.tensor([len(rows)], device="cuda")]).to(torch.int32), "prob": prob.detach(),
           "loss": loss.detach()[None]}
    if c["dir"] == "train":
        out["dlogits"] = torch.autograd.grad(loss, l)[0] * st["dloss"].double()
    return out


def _orth_exact(st):
    out = []
    for g in st["g"]:
        x = g.double()
        x = x / torch.linalg.matrix_norm(x)
        wide = x.shape[0] <= x.shape[1]
        for _ in range(STEPS):
            # X (X^T X) or (X X^T) X, whichever square is the smaller one
            y = (x @ x.T) @ x if wide else x @ (x.T @ x)
            z = (x @ x.T) @ y if wide else y @ (x.T @ x)
            x = COEF[0] * x + COEF[1] * y + COEF[2] * z
        out.append(x)
    return {"out": torch.stack(out)}


def exact(case, seed):
    st = prepare(case, seed)
    return {"scan": _scan_exact, "balance": _balance_exact, "orth": _orth_exact}[case["op"]](st)


# ---- more cases of the same ranges ----------------------------------------------------------------------------------

def _log(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))


def draw(rng):
    op = rng.choice(["scan", "scan", "balance", "orth"])
    kind = rng.choice(["f32", "f16", "bf16"])
    if op == "scan":
        most = max(work(c)["bytes"] for c in listed() if c["op"] == "scan")
        while True:
            tokens, dim = _log(rng, 1, 65536), _log(rng, 16, 4096)
            pad = rng.choice([0, 0, tokens // 9])
            c = _scan(dir=rng.choice(["forward", "backward"]), type=kind, tokens=tokens, dim=rng.choice([dim, max(16, dim // 16 * 16)]),
                      seqs=_log(rng, 1, min(64, tokens - pad)), carry=rng.random() < 0.4, pad=pad)
            if work(c)["bytes"] <= most:
                return c
    if op == "balance":
        most = max(work(c)["bytes"] for c in listed() if c["op"] == "balance")
        while True:
            experts = _log(rng, 2, 256)
            c = _balance(dir=rng.choice(["train", "train", "count"]), type=kind, tokens=_log(rng, 40, 131072), experts=experts,
                         selected=rng.randint(1, min(8, experts)), masked=rng.random() < 0.5)
            if work(c)["bytes"] <= most:
                return c
    most = max(work(c)["flops"] for c in listed() if c["op"] == "orth")
    while True:
        c = _orth(type=kind, batch=_log(rng, 1, 32), rows=_log(rng, 16, 8192), cols=_log(rng, 16, 8192))
        if work(c)["flops"] <= most and c["batch"] * c["rows"] * c["cols"] <= 1 << 26:
            return c
