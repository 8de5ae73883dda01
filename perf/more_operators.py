"""More operators of a training step beside the contractions and the attention core, as cases that can be timed.

Three kinds, each through the public operator-level entry points:

  linear    the product of a dense layer with bias, activation and residual in its epilogue, and its backward pass
            (ts2_op_linear_forward, ts2_op_linear_backward): y = act(x W^T + bias) + residual
  route     the choice of experts from a router's logits and the gradient of their weights (ts2_op_moe_route_forward,
            ts2_op_moe_route_backward): softmax or sigmoid scores, a bias for balance, groups, top-k, renormalised weights
  adamw     one AdamW step of all tensors of a model (ts2_op_adamw), moments in 32 bits or in 8: e4m3 values with a power of two for
            32 neighbours, rounded up or down by a hash so that slow averages keep moving

Activations and gradients are normal, weights have the variance of an initialisation, router logits are normal with some experts
preferred, moments are those of normal gradients whose size differs from row to row."""
import ctypes
import math

import torch

own = False  # True: the framework's operators, False: the plain form

TYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _linear(**kw):
    return dict(dict(op="linear", dir="forward", type="bf16", act="none", tokens=1, inner=256, outer=256, bias=True, residual=False, kept=False), **kw)


def _route(**kw):
    return dict(dict(op="route", dir="train", type="f32", score="softmax", tokens=512, experts=8, selected=2, groups=1, kept_groups=1, group_top=1,
                     bias=False, renormalize=True, masked=False, add=False), **kw)


def _adamw(**kw):
    return dict(dict(op="adamw", bits=32, grad="f32", copy="none", blocks=2, dim=256, wide=512, labels=500, tight=False, step=100), **kw)


def listed():
    return [
        # one token through the expansion of a wide layer, as when a text is continued
        _linear(name="linear_token_bf16", act="silu", inner=2048, outer=8192),
        # a short text of 77 tokens through a model of 768 channels
        _linear(name="linear_short_f16", type="f16", act="gelu", tokens=77, inner=768, outer=6144),
        # the expansion of a wide layer in training, what the activation was given is kept for the backward pass
        _linear(name="linear_expand_bf16", act="gelu", tokens=32768, inner=2048, outer=8192, kept=True),
        # a contraction that joins the residual stream
        _linear(name="linear_contract_f16", type="f16", tokens=65536, inner=2048, outer=768, residual=True),
        # the backward pass of a ragged micro-batch whose sizes no tile and no 16-byte access divides
        _linear(name="linear_ragged_backward_f16", dir="backward", type="f16", act="relu", tokens=5001, inner=333, outer=1001),
        # the backward pass of the expansion
        _linear(name="linear_wide_backward_bf16", dir="backward", act="gelu", tokens=32768, inner=2048, outer=8192),
        # the smallest mixture: 4 x 128 tokens, 8 experts, 2 selected
        _route(name="route_small_f32"),
        # many experts in groups, sigmoid scores, a bias that keeps them balanced; a training step of 32 x 1024 tokens
        _route(name="route_groups_bf16", type="bf16", score="sigmoid", tokens=32768, experts=256, selected=8, groups=8, kept_groups=4, group_top=2,
               bias=True),
        # weights as the softmax gives them, padded sequences, the gradient joins that of another loss
        _route(name="route_masked_f16", type="f16", tokens=65537, experts=128, selected=4, renormalize=False, masked=True, add=True),
        # the smallest model's tensors: latency
        _adamw(name="adamw_small_f32"),
        # a model of 12 blocks, 768 channels: moments in 32 bits, fp32 gradients
        _adamw(name="adamw_model_f32", blocks=12, dim=768, wide=6144, labels=32001),
        # the same with moments in 8 bits, bf16 gradients and a bf16 copy of the weights
        _adamw(name="adamw_model_8bit", bits=8, grad="bf16", copy="bf16", blocks=12, dim=768, wide=6144, labels=32001),
    ]


def work(case):
    c = case
    if c["op"] == "linear":
        T, n, m = c["tokens"], c["inner"], c["outer"]
        if c["dir"] == "forward":  # x, W and the residual in; y and what is kept out
            return {"bytes": 2.0 * (T * n + n * m + T * m * (1 + c["residual"] + c["kept"])) + 4.0 * m * c["bias"], "flops": 2.0 * T * n * m}
        return {"bytes": 2.0 * (2 * T * n + 2 * n * m + T * m * (1 + (c["act"] != "none"))) + 4.0 * m * c["bias"], "flops": 4.0 * T * n * m}
    if c["op"] == "route":
        n, k = c["tokens"] * c["experts"], c["tokens"] * c["selected"]
        fixed = 8.0 * k + (c["tokens"] if c["masked"] else 0) + (4 * c["experts"] if c["bias"] else 0)
        if c["dir"] == "forward":  # exponential, sum, quotient, comparisons
            return {"bytes": SIZE[c["type"]] * n + fixed, "flops": (5.0 + c["selected"]) * n}
        return {"bytes": (2.0 + c["add"]) * SIZE[c["type"]] * n + fixed + 4.0 * k, "flops": (9.0 + c["selected"]) * n}
    n = sum(_sizes(c))
    moments = 16.0 if c["bits"] == 32 else 4 + 4 / 32  # read and written
    return {"bytes": n * (8.0 + SIZE[c["grad"]] + moments + (2 if c["copy"] != "none" else 0)), "flops": 14.0 * n}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _linear_state(c, gen):
    T, n, m, t = c["tokens"], c["inner"], c["outer"], TYPE[c["type"]]
    randn = lambda *shape: torch.randn(shape, device="cuda", generator=gen)
    st = {"c": c, "x": randn(T, n).to(t), "w": (randn(m, n) / math.sqrt(n)).to(t)}
    if c["dir"] == "forward":
        st.update(bias=0.3 * randn(m) if c["bias"] else None, residual=randn(T, m).to(t) if c["residual"] else None,
                  y=torch.zeros((T, m), device="cuda", dtype=t), z=torch.zeros((T, m), device="cuda", dtype=t) if c["kept"] else None)
    else:  # what the forward pass kept
        st.update(z=randn(T, m).to(t) if c["act"] != "none" else None, dy=randn(T, m).to(t), dx=torch.zeros((T, n), device="cuda", dtype=t),
                  dw=torch.zeros((m, n), device="cuda", dtype=t), dbias=torch.zeros(m, device="cuda") if c["bias"] else None)
    return st


def _route_state(c, gen):
    T, E, k, t = c["tokens"], c["experts"], c["selected"], TYPE[c["type"]]
    randn = lambda *shape: torch.randn(shape, device="cuda", generator=gen)
    st = {"c": c, "logits": (randn(T, E) + 0.7 * randn(E)).to(t), "bias": 0.05 * randn(E) if c["bias"] else None,
          "mask": (torch.rand(T, device="cuda", generator=gen) < 0.9).to(torch.uint8) if c["masked"] else None,
          "ids": torch.zeros((T, k), device="cuda", dtype=torch.int32), "weights": torch.zeros((T, k), device="cuda")}
    if c["dir"] == "train":
        st.update(dweights=randn(T, k), other=(0.1 * randn(T, E)).to(t) if c["add"] else None)
        st["dlogits"] = st["other"].clone() if c["add"] else torch.zeros((T, E), device="cuda", dtype=t)
    return st


def _sizes(c):
    """Elements of every tensor of the model: an embedding, and per block four square matrices, an expansion, a contraction, their biases and
    two scales."""
    d, w = c["dim"], c["wide"]
    return [c["labels"] * d] + [d * d, d * d, d * d, d * d, d * w, w, w * d, d, d, d] * c["blocks"]


RECORD = 72  # bytes of a tensor in the table that ts2_op_adamw reads: seven addresses, elements, rate, decay


def _adamw_state(c, gen):
    sizes = _sizes(c)
    unit = 1 if c["tight"] else 64  # tensors one behind the other, or where an allocator puts them
    at, total = [], 0
    for n in sizes:
        at.append(total)
        total += -(-n // unit) * unit
    randn = lambda: torch.randn(total, device="cuda", generator=gen)
    row = torch.exp(1.5 * torch.randn(total // 256 + 1, device="cuda", generator=gen)).repeat_interleave(256)[:total]
    st = {"c": c, "sizes": sizes, "at": at, "param": 0.05 * randn(), "grad": (1e-2 * row * randn()).to(TYPE[c["grad"]]),
          "copy": torch.zeros(total, device="cuda", dtype=TYPE[c["copy"]]) if c["copy"] != "none" else None}
    m, v = 3e-3 * row * randn(), 1e-4 * row * row * (0.5 + torch.rand(total, device="cuda", generator=gen))
    blocks_at, blocks = [], 0  # the first block of 32 of every tensor
    for n in sizes:
        blocks_at.append(blocks)
        blocks += -(-n // 32)
    st["blocks_at"] = blocks_at
    if c["bits"] == 32:
        st.update(m=m, v=v, m_scale=None, v_scale=None)
    else:
        for name, x in (("m", m), ("v", v)):
            st[name] = torch.zeros(total, device="cuda", dtype=torch.uint8)
            st[name + "_scale"] = torch.zeros(blocks, device="cuda", dtype=torch.uint8)
            for n, a, b in zip(sizes, at, blocks_at):
                codes, scale = _encode(x[a:a + n].double(), torch.full((n,), 0.5, device="cuda", dtype=torch.float64), name == "v")
                st[name][a:a + n], st[name + "_scale"][b:b + -(-n // 32)] = codes, scale
    table = (ctypes.c_uint64 * (RECORD // 8 * len(sizes)))()
    for i, (n, a, b) in enumerate(zip(sizes, at, blocks_at)):
        where = [(st["param"], a), (st["grad"], a), (st["m"], a), (st["v"], a), (st["m_scale"], b), (st["v_scale"], b), (st["copy"], a)]
        for j, (x, o) in enumerate(where):
            table[RECORD // 8 * i + j] = 0 if x is None else x.data_ptr() + o * x.element_size()
        table[RECORD // 8 * i + 7] = n
        two = (ctypes.c_float * 2)(1.0, 0.0 if _vector(i) else 0.1)  # vectors are not decayed
        ctypes.memmove(ctypes.addressof(table) + RECORD * i + 64, two, 8)
    st["table"] = table
    return st


def _vector(i):
    return i > 0 and (i - 1) % 10 in (5, 7, 8, 9)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return {"linear": _linear_state, "route": _route_state, "adamw": _adamw_state}[case["op"]](case, gen)


# ---- the plain form -------------------------------------------------------------------------------------------------

def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z / (1 + torch.exp(-z)) if act == "silu" else z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).float()
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


def _linear_plain(st):
    c, t = st["c"], TYPE[st["c"]["type"]]
    x, w = st["x"].float(), st["w"].float()
    if c["dir"] == "forward":
        z = x @ w.t()
        if c["bias"]:
            z += st["bias"]
        y = _act(z, c["act"])
        if c["residual"]:
            y = y + st["residual"].float()
        return {"y": y.to(t), "z": z.to(t)} if c["kept"] else {"y": y.to(t)}
    dz = st["dy"].float()
    if c["act"] != "none":
        dz = dz * _act_slope(st["z"].float(), c["act"])
    out = {"dx": (dz @ w).to(t), "dw": (dz.t() @ x).to(t)}
    if c["bias"]:
        out["dbias"] = dz.sum(dim=0)
    return out


def _pick(key, k):
    """The k largest of each row, the lowest index first among equal ones."""
    return torch.sort(key, dim=1, descending=True, stable=True).indices[:, :k]


def _route_plain(st):
    c = st["c"]
    T, E, k, G = c["tokens"], c["experts"], c["selected"], c["groups"]
    l = st["logits"].double()  # the order of near scores has to be right
    if c["score"] == "softmax":
        s = torch.exp(l - l.amax(dim=1, keepdim=True))
        s = s / s.sum(dim=1, keepdim=True)
    else:
        s = 1 / (1 + torch.exp(-l))
    key = s + st["bias"].double() if c["bias"] else s
    if G > 1:
        per = E // G
        rank = torch.sort(key.view(T, G, per), dim=2, descending=True).values[:, :, :c["group_top"]].sum(dim=2)
        keep = torch.zeros((T, G), device="cuda", dtype=torch.bool)
        keep.scatter_(1, _pick(rank, c["kept_groups"]), True)
        inside = keep[:, :, None].expand(T, G, per).reshape(T, E)
    if not c["bias"]:  # scores ascend with the logits: those tell apart what the rounding of a score would not
        key = l
    if G > 1:
        key = torch.where(inside, key, -math.inf)
    ids = _pick(key, k)
    on = st["mask"].bool() if c["masked"] else torch.ones(T, device="cuda", dtype=torch.bool)
    # the weights in 32 bits: of a softmax among the chosen ones its quotients are those of the chosen exponentials
    f = st["logits"].float()
    chosen = f.gather(1, ids)
    if c["score"] == "softmax":
        e = torch.exp(chosen - (chosen if c["renormalize"] else f).amax(dim=1, keepdim=True))
        total = e.sum(dim=1, keepdim=True) if c["renormalize"] else torch.exp(f - f.amax(dim=1, keepdim=True)).sum(dim=1, keepdim=True)
        weights = SCALE * e / total
        sig = None
    else:
        sig = 1 / (1 + torch.exp(-chosen))
        weights = SCALE * (sig / sig.sum(dim=1, keepdim=True) if c["renormalize"] else sig)
    out = {"ids": torch.where(on[:, None], ids, -1).to(torch.int32), "weights": torch.where(on[:, None], weights, 0.0)}
    if c["dir"] == "train":
        dw = st["dweights"]
        wd = (weights * dw).sum(dim=1, keepdim=True) / SCALE
        if c["renormalize"]:
            d = weights * (dw - wd) * (1 if sig is None else 1 - sig)
        else:
            d = weights * dw if sig is None else weights * dw * (1 - sig)
        dl = torch.zeros((T, E), device="cuda").scatter_(1, ids, d)
        if c["score"] == "softmax" and not c["renormalize"]:
            p = torch.exp(f - f.amax(dim=1, keepdim=True))
            dl -= SCALE * wd * p / p.sum(dim=1, keepdim=True)
        dl = torch.where(on[:, None], dl, 0.0)
        if c["add"]:
            dl = dl + st["dlogits"].float()
            st["dlogits"].copy_(dl)  # a second pass adds once more
            out["dlogits"] = st["dlogits"]
        else:
            out["dlogits"] = dl.to(TYPE[c["type"]])
    return out


SCALE = 2.5  # of the weights
RATE, EPS, GRAD_SCALE, SEED = 1e-3, 1e-8, 0.5, 12345
BETA1, BETA2 = (ctypes.c_float(b).value for b in (0.9, 0.999))
M32, M64 = (1 << 32) - 1, (1 << 64) - 1


def _mix64(x):
    """Steele, Lea, Flood: the output function of SplitMix64."""
    x = (x + 0x9E3779B97F4A7C15) & M64
    x = ((x ^ (x >> 30)) * 0xBF58476D1CE4E5B9) & M64
    x = ((x ^ (x >> 27)) * 0x94D049BB133111EB) & M64
    return x ^ (x >> 31)


def _key(step, tensor):
    return _mix64(_mix64((SEED + step) & M64) ^ tensor) & M32


def _uniforms(n, key):
    """Two numbers in [0, 1), multiples of 2^-16, for each of n elements."""
    x = ((torch.arange(n, device="cuda") * 0x9E3779B1) + key) & M32
    x = ((x ^ (x >> 16)) * 0x85EBCA6B) & M32  # the finaliser of MurmurHash3
    x = ((x ^ (x >> 13)) * 0xC2B2AE35) & M32
    x = x ^ (x >> 16)
    return (x >> 16).double() / 65536, (x & 0xFFFF).double() / 65536


def _exponent(x):
    """floor(log2 x) of positive numbers."""
    return torch.frexp(x).exponent - 1


def _encode(x, u, floor_at_one):
    """e4m3 bytes and a power of two (its exponent + 127) for every 32 neighbours; u decides what rounds up."""
    n = x.numel()
    pad = -n % 32
    a = torch.nn.functional.pad(x.abs(), (0, pad)).view(-1, 32)
    top = a.amax(dim=1)
    e = torch.where(top > 0, _exponent(top) - 7, -127).clamp(-127, 127)
    a = torch.ldexp(a, (9 - e)[:, None]).view(-1)[:n]  # in the smallest steps of e4m3
    up = torch.where(a >= 8, _exponent(a.clamp(min=8)) - 3, 0)
    q = torch.floor(torch.ldexp(a, -up) + u).long()
    if floor_at_one:
        q = torch.where((a > 0) & (q < 1), 1, q)
    code = up * 8 + q
    return (code + torch.where(x < 0, 128, 0)).to(torch.uint8), (e + 127).to(torch.uint8)


def _decode(codes, scale, n):
    c = codes.long()
    e, q = (c & 127) >> 3, c & 7
    a = torch.where(e > 0, torch.ldexp((8 + q).double(), e - 1), q.double())
    a = torch.ldexp(a, scale.long().repeat_interleave(32)[:n] - 127 - 9)
    return torch.where(c > 127, -a, a)


def _adamw_plain(st):
    c = st["c"]
    c1, c2 = 1 - BETA1 ** c["step"], 1 - BETA2 ** c["step"]
    for i, (n, a, b) in enumerate(zip(st["sizes"], st["at"], st["blocks_at"])):
        p, g = st["param"][a:a + n], st["grad"][a:a + n].float() * GRAD_SCALE
        if c["bits"] == 32:
            m, v = st["m"][a:a + n], st["v"][a:a + n]
            m.mul_(BETA1).add_(g * (1 - BETA1))
            v.mul_(BETA2).add_(g * g * (1 - BETA2))
        else:  # in 64 bits up to the rounding to 8
            sm, sv = st["m_scale"][b:b + -(-n // 32)], st["v_scale"][b:b + -(-n // 32)]
            d = g.double()
            m = _decode(st["m"][a:a + n], sm, n) * BETA1 + d * (1 - BETA1)
            v = _decode(st["v"][a:a + n], sv, n) * BETA2 + d * d * (1 - BETA2)
            u = _uniforms(n, _key(c["step"], i))
            st["m"][a:a + n], sm[:] = _encode(m, u[0], False)
            st["v"][a:a + n], sv[:] = _encode(v, u[1], True)
            m, v = m.float(), v.float()
        p.mul_(1 - RATE * (0.0 if _vector(i) else 0.1)).sub_(RATE / c1 * m / (torch.sqrt(v) / math.sqrt(c2) + EPS))
        if st["copy"] is not None:
            st["copy"][a:a + n] = p.to(st["copy"].dtype)
    return _adamw_out(st)


def _adamw_out(st):
    out = {"param": st["param"]}
    if st["c"]["bits"] == 32:
        out.update(m=st["m"], v=st["v"])
    else:
        out.update({n: st[n].view(torch.float8_e4m3fn) for n in ("m", "v")})
        out.update({n: st[n].view(torch.float8_e8m0fnu) for n in ("m_scale", "v_scale")})
    if st["copy"] is not None:
        out["copy"] = st["copy"]
    return out


# ---- one pass -------------------------------------------------------------------------------------------------------

def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(name, *args):
    from tscale2_b200 import capi
    lib = capi.load_library()
    rc = getattr(lib, name)(0, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream), *args)
    if rc != capi.TS2_OK:
        raise capi.Ts2Error(rc, lib.ts2_last_error(None).decode())


def _kind(name):
    from tscale2_b200 import capi
    return {"f32": capi.OUT_F32, "f16": capi.OUT_F16, "bf16": capi.OUT_BF16, "none": capi.OUT_F32}[name]


def _linear_own(st):
    from tscale2_b200 import capi
    c = st["c"]
    T, n, m = c["tokens"], c["inner"], c["outer"]
    act = {"none": capi.ACT_NONE, "relu": capi.ACT_RELU, "gelu": capi.ACT_GELU, "silu": capi.ACT_SILU}[c["act"]]
    if c["dir"] == "forward":
        _call("ts2_op_linear_forward", _kind(c["type"]), act, T, n, m, _ptr(st["x"]), n, _ptr(st["w"]), n, _ptr(st["bias"]), _ptr(st["residual"]), m,
              _ptr(st["y"]), m, _ptr(st["z"]), m)
        return {k: st[k] for k in ("y", "z") if st[k] is not None}
    _call("ts2_op_linear_backward", _kind(c["type"]), act, T, n, m, _ptr(st["dy"]), m, _ptr(st["z"]), m, _ptr(st["x"]), n, _ptr(st["w"]), n, _ptr(st["dx"]),
          n, _kind(c["type"]), _ptr(st["dw"]), n, _ptr(st["dbias"]))
    return {k: st[k] for k in ("dx", "dw", "dbias") if st[k] is not None}


def _route_own(st):
    from tscale2_b200 import capi
    c = st["c"]
    T, E, k = c["tokens"], c["experts"], c["selected"]
    score = capi.SCORE_SOFTMAX if c["score"] == "softmax" else capi.SCORE_SIGMOID
    _call("ts2_op_moe_route_forward", _kind(c["type"]), score, _ptr(st["logits"]), E, T, E, k, _ptr(st["bias"]), c["groups"], c["kept_groups"],
          c["group_top"], c["renormalize"], SCALE, _ptr(st["mask"]), _ptr(st["ids"]), _ptr(st["weights"]))
    out = {n: st[n] for n in ("ids", "weights")}
    if c["dir"] == "train":
        _call("ts2_op_moe_route_backward", _kind(c["type"]), score, _ptr(st["logits"]), E, T, E, k, c["renormalize"], SCALE, _ptr(st["mask"]),
              _ptr(st["ids"]), _ptr(st["dweights"]), _ptr(st["dlogits"]), E, c["add"])
        out["dlogits"] = st["dlogits"]
    return out


def _adamw_own(st):
    c = st["c"]
    _call("ts2_op_adamw", _kind(c["grad"]), c["bits"], _kind(c["copy"]), ctypes.cast(st["table"], ctypes.c_void_p), len(st["sizes"]), RATE, BETA1, BETA2, EPS,
          c["step"], GRAD_SCALE, None, SEED)
    return _adamw_out(st)


def run(state):
    op = state["c"]["op"]
    if own:
        return {"linear": _linear_own, "route": _route_own, "adamw": _adamw_own}[op](state)
    return {"linear": _linear_plain, "route": _route_plain, "adamw": _adamw_plain}[op](state)


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def _linear_exact(st):
    c = st["c"]
    F = torch.nn.functional
    act = {"none": lambda z: z, "relu": torch.relu, "gelu": F.gelu, "silu": F.silu}[c["act"]]
    x, w = st["x"].double(), st["w"].double()
    if c["dir"] == "forward":
        z = F.linear(x, w, st["bias"].double() if c["bias"] else None)
        y = act(z)
        if c["residual"]:
            y = y + st["residual"].double()
        return {"y": y, "z": z} if c["kept"] else {"y": y}
    dz = st["dy"].double()
    if c["act"] != "none":
        z = st["z"].double().requires_grad_(True)
        dz = torch.autograd.grad(act(z), z, dz)[0]
    out = {"dx": torch.matmul(dz, w), "dw": torch.matmul(dz.mT, x)}
    if c["bias"]:
        out["dbias"] = torch.ones(c["tokens"], device="cuda", dtype=torch.float64) @ dz
    return out


def _route_exact(st):
    c = st["c"]
    T, E, k, G = c["tokens"], c["experts"], c["selected"], c["groups"]
    l = st["logits"].double().requires_grad_(True)
    s = torch.softmax(l, dim=1) if c["score"] == "softmax" else torch.sigmoid(l)
    with torch.no_grad():
        key = s + (st["bias"].double() if c["bias"] else 0.0)
        # of equal keys the lowest index: the place among the row's keys, counted, as a number with no two equal
        left = torch.ones((T, E), device="cuda", dtype=torch.bool)
        if G > 1:
            two = key.view(T, G, E // G).topk(c["group_top"], dim=2).values.sum(dim=2)
            ok = torch.zeros((T, G), device="cuda", dtype=torch.bool)
            for _ in range(c["kept_groups"]):
                two_left = torch.where(ok, -math.inf, two)
                best = (two_left == two_left.amax(dim=1, keepdim=True)).int().argmax(dim=1)
                ok[torch.arange(T, device="cuda"), best] = True
            left = ok.repeat_interleave(E // G, dim=1)
        order = key if c["bias"] else l
        ids = []
        for _ in range(k):
            now = torch.where(left, order, -math.inf)
            best = (now == now.amax(dim=1, keepdim=True)).int().argmax(dim=1)
            left[torch.arange(T, device="cuda"), best] = False
            ids.append(best)
        ids = torch.stack(ids, dim=1)
    w = s.gather(1, ids)
    if c["renormalize"]:
        w = w / w.sum(dim=1, keepdim=True)
    on = st["mask"].double()[:, None] if c["masked"] else torch.ones((T, 1), device="cuda", dtype=torch.float64)
    w = SCALE * w * on
    out = {"ids": torch.where(on > 0, ids, -1).to(torch.int32), "weights": w.detach()}
    if c["dir"] == "train":
        out["dlogits"] = torch.autograd.grad((w * st["dweights"].double()).sum(), l)[0]
        if c["add"]:
            out["dlogits"] = out["dlogits"] + st["other"].double()
    return out


def _adamw_exact(st):
    c = st["c"]
    out = {"param": st["param"].double()}
    short = c["bits"] == 8
    for name in ("m", "v"):
        out[name] = st[name].view(torch.float8_e4m3fn).double() if short else st[name].double()
        if short:
            out[name + "_scale"] = st[name + "_scale"].view(torch.float8_e8m0fnu).double()
    for i, (n, a, b) in enumerate(zip(st["sizes"], st["at"], st["blocks_at"])):
        g = st["grad"][a:a + n].double() * GRAD_SCALE
        u = _uniforms(n, _key(c["step"], i)) if short else None
        new = []
        for j, (name, beta, x) in enumerate((("m", BETA1, g), ("v", BETA2, g * g))):
            old = out[name][a:a + n].clone()
            nb = -(-n // 32)
            if short:
                old *= out[name + "_scale"][b:b + nb].repeat_interleave(32)[:n]
            now = beta * old + (1 - beta) * x
            new.append(now)
            if short:  # e4m3 has steps of 2^(e - 3) from 2^e on, and of 2^-9 below 2^-6
                top = torch.zeros(nb * 32, device="cuda", dtype=torch.float64)
                top[:n] = now.abs()
                scale = torch.exp2(torch.floor(torch.log2(top.view(nb, 32).amax(dim=1))).clamp(min=-120) - 7)
                y = now / scale.repeat_interleave(32)[:n]
                step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
                y = torch.copysign(torch.floor(y.abs() / step + u[j]) * step, y)
                out[name][a:a + n] = torch.where((y == 0) & (now > 0), 2.0 ** -9, y) if name == "v" else y
                out[name + "_scale"][b:b + nb] = scale
            else:
                out[name][a:a + n] = now
        decay = 0.0 if _vector(i) else 0.1
        p = out["param"][a:a + n]
        p -= RATE * (decay * p + new[0] / (1 - BETA1 ** c["step"]) / ((new[1] / (1 - BETA2 ** c["step"])).sqrt() + EPS))
    if st["copy"] is not None:
        out["copy"] = torch.zeros_like(out["param"])
        for n, a in zip(st["sizes"], st["at"]):
            out["copy"][a:a + n] = out["param"][a:a + n]
    return out


def exact(case, seed):
    st = prepare(case, seed)
    return {"linear": _linear_exact, "route": _route_exact, "adamw": _adamw_exact}[case["op"]](st)


# ---- more cases of the same ranges ----------------------------------------------------------------------------------

def _log(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))


def draw(rng):
    op = rng.choice(["linear", "linear", "route", "adamw"])
    if op == "linear":
        tokens = rng.choice([1, _log(rng, 1, 32), _log(rng, 32, 1024), _log(rng, 1024, 65536), _log(rng, 1024, 65536)])
        inner, outer = _log(rng, 64, 8192), _log(rng, 8, 8192)
        if rng.random() < 0.6:  # most layers are multiples of something
            inner, outer = max(64, inner // 64 * 64), max(8, outer // 8 * 8)
        direction = rng.choice(["forward", "backward"])
        most = max(work(c)["flops"] for c in listed() if c["op"] == "linear")
        c = _linear(dir=direction, type=rng.choice(["f16", "bf16"]), act=rng.choice(["none", "relu", "gelu", "silu"]), tokens=tokens, inner=inner,
                    outer=outer, bias=rng.random() < 0.7, residual=direction == "forward" and rng.random() < 0.4,
                    kept=direction == "forward" and rng.random() < 0.4)
        while work(c)["flops"] > most:
            c["tokens"] = c["tokens"] // 2
        return c
    if op == "route":
        most = max(work(c)["bytes"] for c in listed() if c["op"] == "route")
        while True:
            groups = rng.choice([1, 1, 2, 4, 8])
            experts = max(groups * 2, _log(rng, 4, 512) // groups * groups)
            kept = rng.randint(1, groups)
            selected = rng.randint(1, min(8, experts // groups * kept))
            c = _route(dir=rng.choice(["train", "train", "forward"]), type=rng.choice(["f32", "f16", "bf16"]), score=rng.choice(["softmax", "sigmoid"]),
                       tokens=_log(rng, 1, 131072), experts=experts, selected=selected, groups=groups, kept_groups=kept,
                       group_top=rng.choice([1, 2]) if groups > 1 else 1, bias=rng.random() < 0.5, renormalize=rng.random() < 0.6,
                       masked=rng.random() < 0.4)
            c["add"] = c["dir"] == "train" and rng.random() < 0.3
            if work(c)["bytes"] <= most:
                return c
    most = max(work(c)["bytes"] for c in listed() if c["op"] == "adamw")
    while True:
        dim = _log(rng, 64, 2048)
        if rng.random() < 0.5:
            dim = max(64, dim // 64 * 64)
        c = _adamw(bits=rng.choice([8, 32]), grad=rng.choice(["f32", "f16", "bf16"]), copy=rng.choice(["none", "f16", "bf16"]), blocks=rng.randint(1, 16),
                   dim=dim, wide=dim * rng.randint(1, 8), labels=_log(rng, 256, 40000), tight=rng.random() < 0.3, step=_log(rng, 1, 100000))
        if work(c)["bytes"] <= most:
            return c
