"""The dense layer, the choice of experts, the balance and AdamW as a training step of a small mixture uses them together: a dense layer with a residual, a router on
what it gives, every expert's dense layer on the tokens that chose it, their weighted sum, the balance of the router's choices, all the way back, and one
AdamW step of all tensors, three times over; against the same in float64 with the choices given.

Tolerance: bf16 activations and gradients, five roundings (2^-9 each, half a step) between the inputs and a weight gradient, averaged by the sums over tokens:
5 x 2^-9 x 2 = 2e-2 of a gradient's norm.  AdamW's update is about the sign of a gradient where that is small, so parameters are compared by the update that the call's
own gradient gives (test_adamw_gpu.py's tolerance), and losses along the way only for being finite."""
import ctypes as C

import pytest

from tscale2_b200 import capi
from tscale2_b200.device import check

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F = torch.nn.functional
BF, F32 = capi.OUT_BF16, capi.OUT_F32


def ptr(t):
    return None if t is None else t.data_ptr()


def stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def rel(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


class Layer:
    """a dense layer's fp32 parameters, their bf16 copy, gradients and moments"""

    def __init__(self, m, n, gen, bits):
        self.p = {"w": torch.randn((m, n), device="cuda", generator=gen) / n ** 0.5, "b": 0.1 * torch.randn(m, device="cuda", generator=gen)}
        self.w16 = self.p["w"].bfloat16()
        self.g = {k: torch.zeros_like(v) for k, v in self.p.items()}
        self.bits = bits
        state = torch.float32 if bits == 32 else torch.uint8
        self.m, self.v = ({k: torch.zeros(v.shape, device="cuda", dtype=state) for k, v in self.p.items()} for _ in range(2))
        self.ms, self.vs = ({k: torch.zeros(-(-v.numel() // 32), device="cuda", dtype=torch.uint8) for k, v in self.p.items()} for _ in range(2))

    def forward(self, x, act, residual=None, z=None):
        T, n = x.shape
        m = self.w16.shape[0]
        y = torch.empty((T, m), device="cuda", dtype=torch.bfloat16)
        check(capi.load_library().ts2_op_linear_forward(0, stream(), BF, act, T, n, m, ptr(x), n, ptr(self.w16), n, ptr(self.p["b"]), ptr(residual), m, ptr(y), m, ptr(z), m))
        return y

    def backward(self, x, act, dy, z, add=False):
        """dx; dw and db into self.g"""
        T, n = x.shape
        m = self.w16.shape[0]
        dx = torch.empty_like(x)
        check(capi.load_library().ts2_op_linear_backward(0, stream(), BF, act, T, n, m, ptr(dy), m, ptr(z), m, ptr(x), n, ptr(self.w16), n, ptr(dx), n,
                                                         capi.OUT_F32_ADD if add else F32, ptr(self.g["w"]), n, ptr(self.g["b"])))
        return dx

    def records(self):
        out = []
        for k in ("w", "b"):
            r = capi.AdamwTensor()
            r.param, r.grad, r.m, r.v = ptr(self.p[k]), ptr(self.g[k]), ptr(self.m[k]), ptr(self.v[k])
            if self.bits == 8:
                r.m_scale, r.v_scale = ptr(self.ms[k]), ptr(self.vs[k])
            r.copy = ptr(self.w16) if k == "w" else None
            r.n, r.rate, r.decay = self.p[k].numel(), 1.0, 0.1 if k == "w" else 0.0
            out.append(r)
        return out


@pytest.mark.parametrize("bits", [32, 8])
def test_steps_of_a_mixture(bits):
    lib = capi.load_library()
    gen = torch.Generator(device="cuda").manual_seed(2)
    T, D, X, E, k = 700, 136, 264, 12, 3
    inner = Layer(D, D, gen, bits)
    router = Layer(E, D, gen, bits)
    experts = [Layer(X, D, gen, bits) for _ in range(E)]
    x, target = (torch.randn(s, device="cuda", generator=gen).bfloat16() for s in ((T, D), (T, X)))
    layers = [inner, router, *experts]
    for step in (1, 2, 3):
        before = [{k: v.double().clone() for k, v in l.p.items()} for l in layers]
        copies = [l.w16.double() for l in layers]
        z = torch.empty((T, D), device="cuda", dtype=torch.bfloat16)
        h = inner.forward(x, capi.ACT_SILU, residual=x, z=z)
        logits = router.forward(h, capi.ACT_NONE)
        ids, weights = torch.empty((T, k), device="cuda", dtype=torch.int32), torch.empty((T, k), device="cuda")
        check(lib.ts2_op_moe_route_forward(0, stream(), BF, capi.SCORE_SOFTMAX, ptr(logits), E, T, E, k, None, 4, 3, 2, 1, 1.0, None, ptr(ids), ptr(weights)))
        counts, prob, loss = torch.empty(E + 1, device="cuda", dtype=torch.int32), torch.empty(E, device="cuda"), torch.empty(1, device="cuda")
        check(lib.ts2_op_moe_balance_forward(0, stream(), BF, ptr(logits), E, T, E, k, ptr(ids), None, ptr(counts), ptr(prob), ptr(loss)))
        out, kept = torch.zeros((T, X), device="cuda"), []
        for e in range(E):
            rows, place = (ids == e).nonzero(as_tuple=True)
            mine = h[rows].contiguous()
            ze = torch.empty((len(rows), X), device="cuda", dtype=torch.bfloat16)
            y = experts[e].forward(mine, capi.ACT_GELU, z=ze)
            out.index_add_(0, rows, weights[rows, place, None] * y.float())
            kept.append((rows, place, mine, ze, y))
        dout = (out - target.float()) / T
        dweights, dh = torch.zeros((T, k), device="cuda"), torch.zeros((T, D), device="cuda")
        for e, (rows, place, mine, ze, y) in enumerate(kept):
            dweights[rows, place] = (dout[rows] * y.float()).sum(1)
            dy = (weights[rows, place, None] * dout[rows] * 64).bfloat16()  # bf16 has the range of fp32; the factor only shows that it is passed on
            dh.index_add_(0, rows, experts[e].backward(mine, capi.ACT_GELU, dy, ze).float())
        dlogits = torch.empty((T, E), device="cuda", dtype=torch.bfloat16)
        check(lib.ts2_op_moe_route_backward(0, stream(), BF, capi.SCORE_SOFTMAX, ptr(logits), E, T, E, k, 1, 64.0, None, ptr(ids), ptr(dweights), ptr(dlogits), E, 0))
        check(lib.ts2_op_moe_balance_backward(0, stream(), BF, ptr(logits), E, T, E, k, None, ptr(counts), None, 0.64, ptr(dlogits), E, 1))
        dh = dh + router.backward(h, capi.ACT_NONE, dlogits, None).float()
        inner.backward(x, capi.ACT_SILU, dh.bfloat16(), z)

        # the same in float64 with the choices given, from the copies that the products read
        ws = [c.requires_grad_(True) for c in copies]
        bs = [b["b"].clone().requires_grad_(True) for b in before]
        x64 = x.double()
        h64 = F.silu(x64 @ ws[0].T + bs[0]) + x64
        l64 = h64 @ ws[1].T + bs[1]
        w64 = torch.softmax(l64.gather(1, ids.long()), 1)
        o64 = torch.zeros((T, X), device="cuda", dtype=torch.float64)
        for e, (rows, place, *_) in enumerate(kept):
            o64 = o64.index_add(0, rows, w64[rows, place, None] * F.gelu(h64[rows] @ ws[2 + e].T + bs[2 + e]))
        p64 = torch.softmax(l64, 1).mean(0)
        assert torch.equal(counts[:E].cpu(), torch.bincount(ids.flatten().cpu(), minlength=E).int())
        total = 0.5 / T * ((o64 - target.double()) ** 2).sum() + 0.01 * E / (k * T) * (counts[:E].double() * p64).sum()
        total.backward()
        assert torch.isfinite(total) and torch.isfinite(loss).all()
        assert rel(out, o64.detach()) < 2e-2 and rel(weights, w64.detach()) < 2e-2
        for l, w, b in zip(layers, ws, bs):
            assert rel(l.g["w"], 64 * w.grad) < 2e-2 and rel(l.g["b"], 64 * b.grad) < 2e-2

        records = [r for l in layers for r in l.records()]
        table = (capi.AdamwTensor * len(records))(*records)
        scale = torch.tensor([1 / 64], device="cuda")
        check(lib.ts2_op_adamw(0, stream(), F32, bits, BF, C.cast(table, C.c_void_p), len(records), 1e-2, 0.9, 0.999, 1e-8, step, 1.0, ptr(scale), 7))
        for l, b in zip(layers, before):
            assert torch.equal(l.w16, l.p["w"].bfloat16())
            if step == 1:  # from zero moments the update is the sign of the gradient, and a decay
                for k_, decay in (("w", 0.1), ("b", 0.0)):
                    g = l.g[k_].double() / 64
                    want = b[k_] * (1 - 1e-2 * decay) - 1e-2 * g / (g.abs() + 1e-8)
                    assert ((l.p[k_].double() - want).abs() <= 2.0 ** -22 * (1 + want.abs())).all()
            else:
                assert all((l.p[k_].double() != b[k_]).any() for k_ in ("w", "b"))
