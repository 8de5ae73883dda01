"""ts2_op_moe_route_forward and _backward against the definition in float64.

ids are equal; where the test makes near keys it makes them differ by more than fp64 rounds.  weights: an fp32 quotient of exponentials.  exp has 2^-22 and
an argument that fp32 holds to 2^-24 of it, so a weight is off by (2^-20 + 2^-23 |l - max|) of itself at most, the softmax's sum of E terms by (E / 32 + 8) 2^-24
more.  dlogits: products and differences of those, of terms no larger than scale |d| w: twice that of their sizes, and half a step of the type."""
import ctypes as C

import pytest

from tscale2_b200 import capi
from tscale2_b200.device import check

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
KIND = {"f32": capi.OUT_F32, "f16": capi.OUT_F16, "bf16": capi.OUT_BF16}
SCORE = {"softmax": capi.SCORE_SOFTMAX, "sigmoid": capi.SCORE_SIGMOID}
INF, NAN = float("inf"), float("nan")


def stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def ptr(t):
    return None if t is None else t.data_ptr()


def scores(l, score):
    if score == "sigmoid":
        return 1 / (1 + torch.exp(-l))
    top = l.amax(1, keepdim=True)
    e = torch.exp(l - torch.where(top == -INF, 0.0, top))
    return e / e.sum(1, keepdim=True)


def choose(logits, score, k, bias, groups, kept, top, mask):
    """the definition, row by row on the host"""
    l = logits.double()
    s = scores(l, score)
    key = s + (bias.double() if bias is not None else 0.0)
    gone = (l == -INF) | torch.isnan(key) | (key == -INF)
    key, l, gone = key.cpu().tolist(), l.cpu().tolist(), gone.cpu().tolist()
    T, E = logits.shape
    out = []
    for t in range(T):
        ids = [e for e in range(E) if not gone[t][e]]
        if groups > 1:
            per = E // groups
            rank = []
            for g in range(groups):
                best = sorted((key[t][e] for e in ids if e // per == g), reverse=True)[:top]
                rank.append(sum(best) if len(best) == top else -INF)
            order = [g for g in sorted(range(groups), key=lambda g: (-rank[g], g)) if rank[g] > -INF][:kept]
            ids = [e for e in ids if e // per in order]
        by = key if bias is not None else l
        ids = sorted(ids, key=lambda e: (-by[t][e], e))[:k]
        if mask is not None and not mask[t]:
            ids = []
        out.append(ids + [-1] * (k - len(ids)))
    return torch.tensor(out, device="cuda", dtype=torch.int32).view(T, k)


def weights_of(l, ids, score, renorm, scale):
    """autograd's way, with choices not made as zeros"""
    made = ids >= 0
    at = ids.clamp(min=0).long()
    if score == "softmax":
        m = torch.where(made, l.gather(1, at), -INF)
        if renorm:
            top = m.amax(1, keepdim=True)
            e = torch.where(made, torch.exp(m - torch.where(top == -INF, 0.0, top).detach()), 0.0)
            return scale * e / e.sum(1, keepdim=True).clamp(min=1e-300)
        row = torch.where(made.any(1, keepdim=True), l, torch.zeros_like(l))
        return scale * torch.where(made, torch.softmax(row, 1).gather(1, at), 0.0)
    m = torch.where(made, l.gather(1, at), 0.0)
    if renorm:
        low = torch.where(made, torch.nn.functional.logsigmoid(m), -INF)
        top = low.amax(1, keepdim=True)
        e = torch.where(made, torch.exp(low - torch.where(top == -INF, 0.0, top).detach()), 0.0)
        return scale * e / e.sum(1, keepdim=True).clamp(min=1e-300)
    return scale * torch.where(made, torch.sigmoid(m), 0.0)


def case(kind, score, T, E, k, bias=False, groups=1, kept=1, top=1, renorm=True, masked=False, add=False, pad=0, first=0, scale=1.5, seed=0, logits=None, b=None):
    lib = capi.load_library()
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(s, device="cuda", generator=gen)
    t, ld = TYPE[kind], E + pad
    flat = torch.full((first + T * ld + 8,), NAN, device="cuda", dtype=t)
    l = flat.as_strided((T, E), (ld, 1), first)
    l.copy_(randn(T, E) + 0.7 * randn(E) if logits is None else logits)
    if bias and b is None:
        b = 0.1 * randn(E)
    mask = (torch.rand(T, device="cuda", generator=gen) < 0.8).to(torch.uint8) if masked else None
    if masked:
        l[mask == 0] = torch.tensor([NAN, INF, -INF] * (E // 3 + 1), device="cuda", dtype=t)[:E]
    ids, w = torch.full((T * k + 1,), 99, device="cuda", dtype=torch.int32), torch.full((T * k + 1,), 7.0, device="cuda")
    check(lib.ts2_op_moe_route_forward(0, stream(), KIND[kind], SCORE[score], ptr(l), ld, T, E, k, ptr(b), groups, kept, top, renorm, scale, ptr(mask), ptr(ids),
                                       ptr(w)))
    want = choose(l, score, k, b, groups, kept, top, mask)
    assert ids[-1] == 99 and w[-1] == 7
    ids, w = ids[:-1].view(T, k), w[:-1].view(T, k)
    assert torch.equal(ids, want), (ids != want).nonzero()[:5]
    used = (want >= 0).any(1, keepdim=True)
    l64 = torch.where(used, l.double(), 0.0).requires_grad_(True)
    w64 = weights_of(l64, want, score, renorm, scale)
    finite = torch.where(torch.isfinite(l64), l64, 0.0).detach()
    spread = finite.amax(1, keepdim=True) - finite.amin(1, keepdim=True) + finite.abs().amax(1, keepdim=True)
    part = 2.0 ** -20 + 2.0 ** -23 * spread + (E / 32 + 8) * 2.0 ** -24
    assert torch.isfinite(w).all() and ((w.double() - w64).abs() <= part * w64 + 1e-37).all()
    d = randn(T, k)
    d = torch.where(want >= 0, d, NAN)  # not read where nothing was chosen
    dl = torch.full((first + T * ld + 8,), 3.0, device="cuda", dtype=t)
    to = dl.as_strided((T, E), (ld, 1), first)
    if add:
        to.copy_(randn(T, E))
    old = to.double().clone()
    check(lib.ts2_op_moe_route_backward(0, stream(), KIND[kind], SCORE[score], ptr(l), ld, T, E, k, renorm, scale, ptr(mask), ptr(ids), ptr(d), ptr(to), ld, add))
    d64 = torch.where(want >= 0, d, 0.0).double()
    g = torch.autograd.grad((w64 * d64).sum(), l64)[0] if T else l64.detach()
    g = torch.where(used, torch.nan_to_num(g), 0.0)
    sizes = (w64.detach() * d64.abs())
    at = want.clamp(min=0).long()
    reach = torch.zeros((T, E), device="cuda", dtype=torch.float64).scatter_add_(1, at, sizes + w64.detach() * sizes.sum(1, keepdim=True) / scale)
    if score == "softmax" and not renorm:
        reach += scores(torch.nan_to_num(l64.detach()), score) * sizes.sum(1, keepdim=True)
    total = g + (old if add else 0)
    step = total.abs() * torch.finfo(t).eps / 2 + (2.0 ** -25 if kind == "f16" else 0)
    off = (to.double() - total).abs()
    assert torch.isfinite(to.double()).all() and (off <= 1.01 * (2 * part * reach + step) + 1e-37).all(), (off - 2 * part * reach - step).max()
    if pad:
        rest = dl.clone()
        rest.as_strided((T, E), (ld, 1), first).fill_(3.0)
        assert (rest == 3).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 2), (3, 8, 8), (77, 5, 3), (200, 64, 6), (65, 100, 8), (130, 128, 4), (33, 256, 8), (17, 384, 32), (9, 777, 10),
                                   (5, 1024, 32), (1000, 16, 1)])
def test_plain(kind, score, renorm, T, E, k):
    case(kind, score, T, E, k, renorm=renorm, seed=T + E + k)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,k,groups,kept,top", [(8, 2, 4, 2, 1), (8, 4, 4, 2, 2), (256, 8, 8, 4, 2), (160, 6, 8, 3, 1), (64, 6, 32, 5, 2), (96, 3, 2, 1, 2), (1024, 32, 32, 4, 2),
                                                 (12, 3, 3, 3, 1), (100, 5, 10, 2, 2)])
@pytest.mark.parametrize("bias", [True, False])
def test_groups(score, E, k, groups, kept, top, bias):
    for kind in ("bf16", "f32"):
        case(kind, score, 120, E, k, bias, groups, kept, top, masked=True, seed=E)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("E,pad,first", [(64, 0, 1), (64, 3, 0), (33, 0, 0), (8, 8, 0), (256, 64, 2), (130, 2, 4)])
@pytest.mark.parametrize("add", [False, True])
def test_pitches_masks_and_sums(kind, E, pad, first, add):
    for renorm in (True, False):
        case(kind, "softmax", 300, E, 4, True, renorm=renorm, masked=True, add=add, pad=pad, first=first, seed=E + pad)
        case(kind, "sigmoid", 300, E, 4, True, renorm=renorm, masked=True, add=add, pad=pad, first=first, seed=E + pad)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [None, "zero", "levels"])
@pytest.mark.parametrize("E,k,groups", [(8, 3, 1), (64, 8, 1), (64, 8, 8), (256, 8, 8), (512, 32, 1)])
def test_ties_go_to_the_lowest_index(score, bias, E, k, groups):
    gen = torch.Generator(device="cuda").manual_seed(3)
    logits = torch.randint(-2, 3, (200, E), device="cuda", generator=gen).float()
    logits[:4] = 0
    b = None if bias is None else torch.zeros(E, device="cuda") if bias == "zero" else torch.randint(0, 2, (E,), device="cuda", generator=gen).float()
    case("bf16", score, 200, E, k, bias is not None, groups, max(1, groups // 2), 1, logits=logits, b=b)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_near_keys_are_told_apart(score):
    """keys that fp32 cannot tell apart, and fp64 can: biases that make up for all but a little of a score"""
    gen = torch.Generator(device="cuda").manual_seed(4)
    T, E, k = 400, 64, 8
    logits = torch.randn((1, E), device="cuda", generator=gen).expand(T, E).contiguous()
    s = scores(logits[:1].double(), score)[0]
    b = (1.0 - s).float()  # every key is 1 up to the rounding of the bias, 2^-25, and what the score's own fp32 would lose
    case("f32", score, T, E, k, True, logits=logits, b=b)
    case("f32", score, T, E, k, True, 8, 4, 2, logits=logits, b=b)
    logits = (logits + 1e-6 * torch.randn((T, E), device="cuda", generator=gen))
    case("f32", score, T, E, k, True, 8, 4, 2, logits=logits, b=b)


@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_rows_with_little_or_nothing_to_choose_from(score, renorm):
    T, E = 24, 16
    l = torch.randn((T, E), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    l[0] = -INF
    l[1, 1:] = -INF
    l[2, 3] = NAN
    l[3, 3] = INF
    l[4] = NAN
    l[5, ::2] = -INF
    l[6] = torch.finfo(torch.float32).min
    l[7, 1:] = torch.finfo(torch.float32).min
    l[8] = torch.finfo(torch.float32).max
    l[9] = -100 - 3 * torch.arange(E, device="cuda")
    l[10] = 200.0
    l[11, :3] = -INF
    l[12] = -INF
    l[12, 14:] = torch.tensor([-200.0, -201.0], device="cuda")
    for b in (None, torch.linspace(-0.1, 0.1, E, device="cuda"), torch.tensor([-INF, 0.5, INF, NAN] * 4, device="cuda")):
        for groups, kept, top in ((1, 1, 1), (4, 2, 2), (4, 2, 1)):
            case("f32", score, T, E, 6, b is not None, groups, kept, top, renorm=renorm, logits=l, b=b)


def test_ids_that_were_not_made_and_ids_made_twice():
    """ids of the caller's: outside of the experts, and the same one twice; a gradient of a weight each"""
    T, E, k = 3, 8, 4
    l = torch.randn((T, E), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    ids = torch.tensor([[1, -1, 8, 2], [3, 3, 5, 0], [-5, 99, -1, 1 << 30]], device="cuda", dtype=torch.int32)
    d = torch.randn((T, k), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    ok = (ids >= 0) & (ids < E)
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            out = torch.zeros((T, E), device="cuda")
            check(capi.load_library().ts2_op_moe_route_backward(0, stream(), KIND["f32"], SCORE[score], ptr(l), E, T, E, k, renorm, 2.0, None, ptr(ids), ptr(d), ptr(out), E, 0))
            l64 = l.double().requires_grad_(True)
            w = weights_of(l64, torch.where(ok, ids, -1), score, renorm, 2.0)
            want = torch.autograd.grad((w * torch.where(ok, d, 0.0)).sum(), l64)[0]
            assert (out - want).abs().max() < 2e-6 and (out[2] == 0).all()


def test_gradient_against_differences():
    gen = torch.Generator(device="cuda").manual_seed(9)
    T, E, k = 20, 32, 4
    l = torch.randn((T, E), device="cuda", generator=gen)
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            ids, w, d = torch.zeros((T, k), device="cuda", dtype=torch.int32), torch.zeros((T, k), device="cuda"), torch.randn((T, k), device="cuda", generator=gen)
            lib, dl = capi.load_library(), torch.zeros((T, E), device="cuda")
            check(lib.ts2_op_moe_route_forward(0, stream(), 0, SCORE[score], ptr(l), E, T, E, k, None, 1, 1, 1, renorm, 1.0, None, ptr(ids), ptr(w)))
            check(lib.ts2_op_moe_route_backward(0, stream(), 0, SCORE[score], ptr(l), E, T, E, k, renorm, 1.0, None, ptr(ids), ptr(d), ptr(dl), E, 0))
            v = torch.randn((T, E), device="cuda", generator=gen, dtype=torch.float64)
            f = lambda x: (weights_of(x, ids, score, renorm, 1.0) * d.double()).sum()
            want = (f(l.double() + 1e-6 * v) - f(l.double() - 1e-6 * v)) / 2e-6
            assert abs((dl.double() * v).sum() - want) < 1e-5 * (1 + abs(want))


def test_no_tokens_and_many():
    lib = capi.load_library()
    check(lib.ts2_op_moe_route_forward(0, stream(), 0, 0, None, 8, 0, 8, 2, None, 1, 1, 1, 1, 1.0, None, None, None))
    check(lib.ts2_op_moe_route_backward(0, stream(), 0, 0, None, 8, 0, 8, 2, 1, 1.0, None, None, None, None, 8, 0))
    T, E, k = 300_000, 8, 2  # more rows than the device holds at once
    l = torch.randn((T, E), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    ids, w = torch.zeros((T, k), device="cuda", dtype=torch.int32), torch.zeros((T, k), device="cuda")
    check(lib.ts2_op_moe_route_forward(0, stream(), 0, 0, ptr(l), E, T, E, k, None, 1, 1, 1, 1, 1.0, None, ptr(ids), ptr(w)))
    assert torch.equal(ids, torch.sort(l, dim=1, descending=True, stable=True).indices[:, :k].int())


def test_beyond_32_bit_offsets():
    T, E, pitch = 2300, 16, 1_000_003
    flat = torch.zeros(T * pitch, device="cuda", dtype=torch.float16)
    l, dl = flat.as_strided((T, E), (pitch, 1), 0), flat.as_strided((T, E), (pitch, 1), 100)
    l.copy_(torch.randn((T, E), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)))
    ids, w, d = torch.zeros((T, 2), device="cuda", dtype=torch.int32), torch.zeros((T, 2), device="cuda"), torch.ones((T, 2), device="cuda")
    d[:, 1] = -1
    lib = capi.load_library()
    check(lib.ts2_op_moe_route_forward(0, stream(), 2, 0, ptr(l), pitch, T, E, 2, None, 1, 1, 1, 1, 1.0, None, ptr(ids), ptr(w)))
    check(lib.ts2_op_moe_route_backward(0, stream(), 2, 0, ptr(l), pitch, T, E, 2, 1, 1.0, None, ptr(ids), ptr(d), ptr(dl), pitch, 0))
    assert torch.equal(ids, torch.sort(l.float(), dim=1, descending=True, stable=True).indices[:, :2].int())
    g = 2 * w[:, 0] * w[:, 1]
    assert (dl.gather(1, ids.long()).float() - torch.stack([g, -g], 1)).abs().max() < 3e-4


def test_same_bits_on_another_stream_and_replayed():
    T, E, k = 5000, 64, 6
    gen = torch.Generator(device="cuda").manual_seed(1)
    l, d, b = torch.randn((T, E), device="cuda", generator=gen), torch.randn((T, k), device="cuda", generator=gen), torch.randn(E, device="cuda", generator=gen)
    lib = capi.load_library()

    def step(o):
        check(lib.ts2_op_moe_route_forward(0, stream(), 0, 1, ptr(l), E, T, E, k, ptr(b), 8, 4, 2, 1, 1.0, None, ptr(o[0]), ptr(o[1])))
        check(lib.ts2_op_moe_route_backward(0, stream(), 0, 1, ptr(l), E, T, E, k, 1, 1.0, None, ptr(o[0]), ptr(d), ptr(o[2]), E, 0))

    outs = [(torch.zeros((T, k), device="cuda", dtype=torch.int32), torch.zeros((T, k), device="cuda"), torch.zeros((T, E), device="cuda")) for _ in range(3)]
    step(outs[0])
    torch.cuda.synchronize()
    other, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(other):
        step(outs[1])
    with torch.cuda.graph(g, stream=other):
        step(outs[2])
    g.replay()
    g.replay()
    torch.cuda.synchronize()
    for o in outs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(outs[0], o))
