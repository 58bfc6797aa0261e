"""Dropout, layer norm, action log-probabilities and the clipped policy loss against their definitions in 64 bits.

Tolerances.  EPS is fp32's unit roundoff; an output of 16 bits may be off by its own rounding U (half a unit in the last
place) on top of the fp32 error.  A sum of k terms in a tree over threads with at most s additions in a row is off by at most
about (s + 10) EPS times the sum of the terms' magnitudes; the kernels keep s below 32 + k / 128, so STEPS(k) = 48 + k / 64
bounds it and the few roundings around it.  The exponential and the logarithm add at most 4 EPS relative to their values,
and an argument x of the exponential carries its own rounding, |x| EPS."""
import math

import numpy as np
import pytest
import torch

import compactlogic_b200 as cl
from compactlogic_b200 import _lib as L

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float64: 2.0 ** -53}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24, torch.float64: 1e-300}
LOW = [torch.float32, torch.bfloat16, torch.float16]
ALL = LOW + [torch.float64]


def steps(k):
    return 48 + k / 64


def near(got, want, slack, dtype, what=""):
    """|got - want| <= U |want| + slack elementwise (slack: tensor or number, absolute); NaN and infinities in place."""
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    slack = slack.detach().double().cpu() if isinstance(slack, torch.Tensor) else torch.tensor(float(slack), dtype=torch.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got)), what
    assert torch.equal(torch.isnan(want), torch.isnan(got)), what
    assert torch.equal(want[~fine & ~torch.isnan(want)], got[~fine & ~torch.isnan(got)]), what
    bound = U[dtype] * want.abs() * 1.01 + slack + TINY[dtype]
    bad = fine & ~((got - want).abs() <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} off, worst {float(((got - want).abs() / bound)[fine].max()):.3g} of the bound"


def eps_of(dtype):
    return 2.0 ** -53 if dtype == torch.float64 else EPS


def laid(t, layout):
    """The values of ``t`` [n, d] in a given storage."""
    n, d = t.shape
    if layout == "rows":
        return t.contiguous()
    if layout == "features":
        return t.t().contiguous().t()
    if layout == "padded":  # rows of a wider matrix, which do not start on 16 bytes
        w = torch.zeros(n, d + 3, dtype=t.dtype, device=t.device)
        w[:, 1:1 + d] = t
        return w[:, 1:1 + d]
    if layout == "padded_features":
        w = torch.zeros(d, n + 5, dtype=t.dtype, device=t.device)
        w[:, 2:2 + n] = t.t()
        return w[:, 2:2 + n].t()
    assert layout == "strided"
    w = torch.zeros(n, 2 * d, dtype=t.dtype, device=t.device)
    w[:, ::2] = t
    return w[:, ::2]


def rand(shape, seed, dtype=torch.float32, scale=1.0, shift=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float64) * scale + shift).to(dtype)


LAYOUTS = ["rows", "features", "padded", "padded_features", "strided"]


# ------------------------------------------------------------------------------------------------------------- dropout
def words(n, d, seed, offset, first=0):
    """Philox4x32-10 as in its paper, in numpy: [n, d] words, from the (even) row `first` on."""
    c = [np.zeros(((n + 1) // 2, (d + 1) // 2), dtype=np.uint64) for _ in range(4)]
    c[0] += np.arange((d + 1) // 2, dtype=np.uint64)[None, :]
    c[1] += np.arange(first // 2, first // 2 + (n + 1) // 2, dtype=np.uint64)[:, None]
    c[2] += np.uint64(offset & 0xFFFFFFFF)
    c[3] += np.uint64(offset >> 32)
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    m = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & m, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & m]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    out = np.zeros((2 * c[0].shape[0], 2 * c[0].shape[1]), np.uint64)
    for w in range(4):
        out[w // 2::2, w % 2::2] = c[w]
    return out[:n, :d]


def test_the_generator_is_philox():
    """The paper's known answers for Philox4x32-10: counter and key of zeros, and of ones."""
    w = words(2, 2, 0, 0)
    assert [int(w[0, 0]), int(w[0, 1]), int(w[1, 0]), int(w[1, 1])] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]


def dropped(x, p, seed, offset, rescale):
    n, d = x.shape
    keep = torch.from_numpy(words(n, d, seed, offset).astype(np.int64)).cuda() >= round(p * 2 ** 32)
    work = torch.float64 if x.dtype == torch.float64 else torch.float32
    scale = torch.tensor(1.0 / (1.0 - p) if rescale and p < 1 else 1.0, dtype=work, device="cuda")
    return torch.where(keep, x.to(work) * scale, torch.zeros((), dtype=work, device="cuda")).to(x.dtype)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n,d", [(1, 1), (2, 3), (1, 4096), (33, 1), (48, 96), (129, 777), (1000, 513)])
def test_dropout_values_and_gradient(n, d, dtype, layout):
    x = laid(rand((n, d), 1, dtype), layout).requires_grad_()
    gy = laid(rand((n, d), 2, dtype), "features" if (n + d) % 2 else "rows")
    y = cl.dropout(x, 0.3, seed=0x1234567890ABCDEF, offset=(1 << 33) + 5)
    gx, = torch.autograd.grad(y, x, gy)
    assert y.dtype == dtype and gx.dtype == dtype
    assert torch.equal(y, dropped(x.detach(), 0.3, 0x1234567890ABCDEF, (1 << 33) + 5, True))
    assert torch.equal(gx, dropped(gy, 0.3, 0x1234567890ABCDEF, (1 << 33) + 5, True))


@pytest.mark.parametrize("p", [0.0, 1e-9, 0.5, 1 - 1e-12, 1.0])
@pytest.mark.parametrize("rescale", [True, False])
def test_dropout_rates(p, rescale):
    x = rand((64, 200), 3)
    x[0, :100] = float("nan")
    x[1, :100] = float("inf")
    y = cl.dropout(x, p, seed=9, rescale=rescale)
    if p == 1.0:
        assert torch.equal(y, torch.zeros_like(x))
    elif p < 1e-6:
        assert torch.equal(torch.nan_to_num(y), torch.nan_to_num(x * torch.tensor(1 / (1 - p) if rescale else 1.0)))
    else:
        want = dropped(x, p, 9, 0, rescale)
        assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(y[2:], want[2:])
        assert torch.equal(y == 0, want == 0)


def test_dropout_rates_that_round_to_one_keep_nothing():
    """p 2^32 rounds to 2^32, which no word reaches, not even the largest."""
    for seed, offset, i, j in [(11, 1686893, 18, 48), (11, 3385604, 33, 13)]:
        assert int(words(64, 64, seed, offset)[i, j]) == 0xFFFFFFFF
        for dtype in ALL:
            for layout in LAYOUTS:
                x = laid(torch.ones(64, 64, device="cuda", dtype=dtype), layout)
                for p in (1.0, 1 - 2.0 ** -34, 1 - 2.0 ** -33, 1 - 2.0 ** -50):  # round(p 2^32) goes to the even one
                    assert not cl.dropout(x, p, seed=seed, offset=offset).any()
                for p in (1 - 2.0 ** -32, 0.5):
                    y = cl.dropout(x, p, seed=seed, offset=offset, rescale=False)
                    assert torch.equal(y, dropped(x, p, seed, offset, False)) and y[i, j] == 1


def test_dropout_shapes_and_refusals():
    for shape in [(0, 5), (5, 0), (7,), (), (3, 4, 5), (2, 3, 4, 5)]:
        x = rand(shape, 4)
        y = cl.dropout(x, 0.5, seed=1)
        assert y.shape == x.shape
        if x.numel():
            flat = x.reshape(x.shape[0], -1) if x.dim() > 1 else x.reshape(1, -1)
            assert torch.equal(y.reshape(flat.shape), dropped(flat, 0.5, 1, 0, True))
    x = rand((4, 4), 5)
    for bad in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError):
            cl.dropout(x, bad, seed=1)
    with pytest.raises(ValueError):
        cl.dropout(x, 0.5, seed=-1)
    with pytest.raises(ValueError):
        cl.dropout(x, 0.5, seed=1, offset=1 << 64)
    with pytest.raises(RuntimeError):
        cl.dropout(x.long(), 0.5, seed=1)
    with pytest.raises(RuntimeError):
        cl.dropout(x.cpu(), 0.5, seed=1)


def test_dropout_module_draws_a_mask_per_pass_and_resumes():
    m = cl.LogicDropout(0.5, seed=77).cuda()
    x = torch.ones(64, 64, device="cuda", requires_grad=True)
    y0, y1 = m(x), m(x)
    g0, = torch.autograd.grad(y0, x, torch.ones_like(y0))  # after the state has moved on
    assert torch.equal(y0, dropped(torch.ones_like(x), 0.5, 77, 0, True)) and torch.equal(g0, y0)
    assert torch.equal(y1, dropped(torch.ones_like(x), 0.5, 77, 1, True))
    other = cl.LogicDropout(0.5, seed=1).cuda()
    other.load_state_dict(m.state_dict())
    assert torch.equal(other(x), m(x))
    assert m.eval()(x) is x


def test_dropout_module_under_a_graph():
    m = cl.LogicDropout(0.5, seed=5).cuda()
    x = torch.ones(32, 64, device="cuda")
    m(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = m(x)
    seen = []
    for _ in range(3):
        graph.replay()
        seen.append(y.clone())
    for k, t in enumerate(seen):
        assert torch.equal(t, dropped(x, 0.5, 5, 1 + k, True))


def checkpointed(reentrant):
    from torch.utils.checkpoint import checkpoint
    return (lambda f, *a: f(*a)) if reentrant is None else (lambda f, *a: checkpoint(f, *a, use_reentrant=reentrant))


@pytest.mark.parametrize("shape", [(48, 64), (6, 4, 5, 7)])
@pytest.mark.parametrize("reentrant", [True, False])
def test_dropout_module_recomputed_by_activation_checkpointing(reentrant, shape):
    """A recomputed pass draws the mask of the pass that it repeats: several passes of one module in a block, several
    blocks in flight, an input that needs no gradient, and passes outside."""
    def run(how):
        torch.manual_seed(0)
        torch.cuda.manual_seed(1)
        wrap = checkpointed(how)
        m = cl.LogicDropout(0.4, seed=9).cuda()
        w = rand(shape[1:], 1).requires_grad_()
        xs = [rand(shape, 2 + k).requires_grad_(k > 0) for k in range(3)]
        with torch.no_grad():
            m(xs[0])                                                   # a rollout
        ys = [wrap(lambda x, w: m(torch.tanh(m(x) * w) * 2), x, w) for x in xs]
        last = m(ys[0] * ys[1])
        noise = torch.rand(4, device="cuda")                           # torch's own sequence
        ((last ** 2).sum() + sum((y ** 2).sum() for y in ys)).backward()
        after = m(xs[0].detach())
        return ys + [last, after] + [x.grad for x in xs[1:]] + [m.rng_state], w.grad, noise

    want, gw, _ = run(None)
    got, gw2, noise = run(reentrant)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert want[-1].tolist() == [9, 9]
    assert (gw - gw2).abs().max() <= 1e-6 * gw.abs().max()             # summed over the blocks in another order


@pytest.mark.parametrize("reentrant", [True, False])
def test_dropout_module_refuses_a_recomputation_that_it_cannot_repeat(reentrant):
    """Without torch's generator put back, or where it stood at the same place in two passes, a recomputed pass cannot
    tell which one it repeats."""
    from torch.utils.checkpoint import checkpoint
    m = cl.LogicDropout(0.5, seed=3).cuda()
    x = rand((8, 8), 1).requires_grad_()
    y = checkpoint(m, x, use_reentrant=reentrant, preserve_rng_state=False)
    torch.rand(8, 8, device="cuda")
    if reentrant:
        with pytest.raises(RuntimeError, match="recomput"):
            (y * y).sum().backward()
    else:  # dropout alone saves nothing that would have to be computed again
        gx, = torch.autograd.grad((y * y).sum(), x)
        assert torch.equal(gx, 4 * dropped(x.detach(), 0.5, 3, 0, True))
    y = checkpoint(lambda t: m(t) * t, x, use_reentrant=reentrant, preserve_rng_state=False)
    torch.rand(8, 8, device="cuda")
    with pytest.raises(RuntimeError, match="recomput"):
        (y * y).sum().backward()
    torch.cuda.manual_seed(5)
    a = checkpoint(lambda t: m(t) * t, x, use_reentrant=reentrant)
    torch.cuda.manual_seed(5)
    b = checkpoint(lambda t: m(t) * t, x, use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match="recomput"):
        (a + b).sum().backward()


def test_dropout_module_copies_and_pickles():
    import copy
    import io
    import pickle
    m = cl.LogicDropout(0.5, seed=3).cuda()
    x = torch.ones(8, 64, device="cuda", requires_grad=True)
    with torch.no_grad():
        m(x)
    y = m(x)
    file = io.BytesIO()
    torch.save(m, file)
    file.seek(0)
    for other in (copy.deepcopy(m), pickle.loads(pickle.dumps(m)), torch.load(file, weights_only=False)):
        assert torch.equal(other(x), dropped(torch.ones_like(x), 0.5, 3, 2, True))
    assert torch.equal(y, dropped(torch.ones_like(x), 0.5, 3, 1, True))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_dropout_between_logic_layers(dtype):
    """The layers' gradients through dropout equal those of the same network with the mask multiplied in by torch; with
    bf16 activations the gradient passes in fp32, so only the activations' rounding is left (they are 0 or equal)."""
    torch.manual_seed(0)
    a, b = cl.LogicLayer(64, 96).cuda(), cl.LogicLayer(96, 80).cuda()
    x = torch.rand(40, 64, device="cuda").to(dtype)
    y = b(cl.dropout(a(x), 0.25, seed=3, rescale=False))
    gy = rand(y.shape, 6, dtype)
    got = torch.autograd.grad(y, [a.weights, b.weights], gy)
    h = a(x)
    slot = getattr(h, "_clb_slot", None)
    mask = dropped(torch.ones_like(h), 0.25, 3, 0, False)
    mid = (h.detach() * mask).requires_grad_()
    y2 = b(mid)
    assert torch.equal(y, y2)
    if slot is None:
        gmid, gwb = torch.autograd.grad(y2, [mid, b.weights], gy)
        gwa, = torch.autograd.grad(h, a.weights, gmid * mask)
        tol = 1e-5
    else:  # fp32 hand-over past autograd: take it out of a slot of our own
        from compactlogic_b200.functional import GradSlot
        mid._clb_slot = GradSlot()
        y2 = b(mid)
        gwb, _ = torch.autograd.grad(y2, [b.weights, mid], gy)
        slot.add(mid._clb_slot.grad * mask.t().float())
        gwa, = torch.autograd.grad(h, a.weights, torch.zeros((), dtype=dtype, device="cuda").expand(h.shape))
        tol = 1e-5
    for g, w in zip(got, (gwa, gwb)):
        assert (g - w).abs().max() <= tol * w.abs().max()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_dropout_between_conv_layers(dtype):
    """As between dense layers: with 16-bit activations the gradient passes in fp32."""
    torch.manual_seed(0)
    a = cl.ConvLayer((3, 8, 8), 1, 8, 3, 2, num_gates=4).cuda()
    b = cl.ConvLayer((8, 4, 4), 1, 16, 3, 2, num_gates=4).cuda()
    x = torch.rand(20, 3, 8, 8, device="cuda").to(dtype)
    drop = lambda h: cl.dropout(h, 0.25, seed=3, rescale=False)  # noqa: E731
    h = drop(a(x))
    assert h.shape == (20, 8, 4, 4)
    y = b(h)
    gy = rand(y.shape, 6, dtype)
    got = torch.autograd.grad(y, [a.weights, b.weights], gy)
    h = a(x)
    mask = dropped(torch.ones(20, 128, device="cuda", dtype=dtype), 0.25, 3, 0, False).reshape(h.shape)
    mid = (h.detach() * mask).requires_grad_()
    if dtype == torch.float32:
        y2 = b(mid)
        gmid, gwb = torch.autograd.grad(y2, [mid, b.weights], gy)
        gwa, = torch.autograd.grad(h, a.weights, gmid * mask)
    else:
        from compactlogic_b200.functional import GradSlot
        mid._clb_slot = GradSlot()
        y2 = b(mid)
        gwb, _ = torch.autograd.grad(y2, [b.weights, mid], gy)
        h._clb_slot.add(mid._clb_slot.grad * mask.reshape(20, -1).t().float())
        gwa, = torch.autograd.grad(h, a.weights, torch.zeros((), dtype=dtype, device="cuda").expand(h.shape))
    assert torch.equal(y, y2)
    for g, w in zip(got, (gwa, gwb)):
        assert (g - w).abs().max() <= 1e-5 * w.abs().max()
    # another consumer beside the layer: its share comes through autograd
    h = drop(a(x))
    both, = torch.autograd.grad([b(h), h], a.weights, [gy, torch.ones_like(h)])
    h = drop(a(x))
    alone, = torch.autograd.grad(h, a.weights, torch.ones_like(h))
    assert (both - (got[0] + alone)).abs().max() <= 1e-5 * both.abs().max()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("reentrant", [True, False])
def test_logic_layers_and_dropout_recomputed(reentrant, dtype):
    """Layers and dropout in checkpointed blocks: the gradients of the plain network."""
    def run(how):
        torch.manual_seed(0)
        wrap = checkpointed(how)
        a, b, c = cl.LogicLayer(64, 96).cuda(), cl.LogicLayer(96, 80).cuda(), cl.LogicLayer(80, 60).cuda()
        m = cl.LogicDropout(0.25, rescale=False, seed=4).cuda()
        x = rand((40, 64), 1).sigmoid().to(dtype).requires_grad_()
        y = cl.GroupSum(6, tau=2.0)(c(wrap(lambda t: b(m(a(t))), x)))
        (y * rand(y.shape, 2, dtype)).sum().backward()
        return y, [x.grad] + [t.weights.grad for t in (a, b, c)]

    want, grads = run(None)
    got, again = run(reentrant)
    assert torch.equal(want, got)
    # the gradient that a recomputed block is given is autograd's, rounded to the activations' type: 40 samples' terms, U each
    tol = 40 * U[dtype] if reentrant and dtype != torch.float32 else 1e-5
    for g, w in zip(again, grads):
        assert (g.double() - w.double()).abs().max() <= tol * w.double().abs().max()


# ---------------------------------------------------------------------------------------------------------- layer norm
def norm64(x, w, b, eps, gy=None):
    x = x.detach().double()
    mu = x.mean(1, keepdim=True)
    r = 1 / torch.sqrt(((x - mu) ** 2).mean(1, keepdim=True) + eps)
    h = (x - mu) * r
    w64 = w.detach().double() if w is not None else torch.ones(x.shape[1], dtype=torch.float64, device=x.device)
    y = h * w64 + (b.detach().double() if b is not None else 0)
    if gy is None:
        return y, h, mu, r, w64
    g = gy.double()
    t = g * w64
    gx = r * (t - t.mean(1, keepdim=True) - h * (t * h).mean(1, keepdim=True))
    return y, h, mu, r, w64, t, gx, (g * h).sum(0), g.sum(0)


def check_norm(n, d, dtype, layout, affine=True, gy_layout=None, seed=10, scale=1.5, shift=0.5, eps=1e-5):
    acc = torch.float64 if dtype == torch.float64 else torch.float32
    x = laid(rand((n, d), seed, dtype, scale, shift), layout).requires_grad_()
    w = rand((d,), seed + 1, acc, 0.2, 1.0).requires_grad_() if affine else None
    b = rand((d,), seed + 2, acc, 0.2).requires_grad_() if affine else None
    gy = laid(rand((n, d), seed + 3, dtype), gy_layout or layout)
    y = cl.layer_norm(x, w, b, eps=eps)
    with torch.no_grad():
        assert torch.equal(cl.layer_norm(x, w, b, eps=eps), y)
    got = torch.autograd.grad(y, [x] + ([w, b] if affine else []), gy)
    y64, h, mu, r, w64, t, gx, gw, gb = norm64(x, w, b, eps, gy)
    e = eps_of(dtype)
    k = steps(d)
    spread = 1 + (mu.abs() + x.detach().double().abs().mean(1, keepdim=True)) * r + h.abs()  # what an EPS of x - mu becomes in h
    near(y, y64, e * k * spread * w64.abs() + e * y64.abs() + (e * b.double().abs() if affine else 0), dtype, "y")
    big = t.abs() + t.abs().mean(1, keepdim=True) + (1 + h.abs()) * ((t * h).abs().mean(1, keepdim=True) +
                                                                  (t.abs() * spread).mean(1, keepdim=True))
    near(got[0], gx, 2 * e * k * r * big, dtype, "gx")
    if affine:
        near(got[1], gw, e * ((steps(n) + k) * (gy.double().abs() * spread).sum(0)), acc, "gw")
        near(got[2], gb, e * steps(n) * gy.double().abs().sum(0), acc, "gb")
    return x, w, b, gy, y, got


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n,d", [(1, 1), (1, 784), (3, 2), (65, 33), (100, 257), (37, 1000), (300, 96)])
def test_layer_norm(n, d, dtype, layout):
    check_norm(n, d, dtype, layout)


@pytest.mark.parametrize("dtype", LOW)
@pytest.mark.parametrize("n,d,layout", [(5, 4096, "rows"), (700, 4096, "rows"), (3, 5001, "rows"), (3, 16384, "rows"),
                                        (4, 16385, "rows"), (2, 64000, "rows"), (2, 65536, "rows"), (3, 65537, "padded"),
                                        (2, 300000, "rows"), (64, 16384, "features"), (40, 5001, "features"),
                                        (1030, 300, "features"), (5000, 40, "features"), (5000, 40, "rows"),
                                        (3, 100000, "features"), (2048, 2000, "rows"), (1, 1000000, "features")])
def test_layer_norm_sizes(n, d, layout, dtype):
    check_norm(n, d, dtype, layout)


@pytest.mark.parametrize("layout", ["rows", "features"])
def test_layer_norm_variants(layout):
    check_norm(50, 130, torch.float32, layout, affine=False)
    check_norm(50, 130, torch.float32, layout, gy_layout="features" if layout == "rows" else "rows")
    check_norm(50, 130, torch.bfloat16, layout, gy_layout="strided")
    check_norm(50, 130, torch.float32, layout, scale=1e-3, shift=100.0)  # a mean far above the spread
    x = laid(rand((20, 64), 1), layout)
    w = rand((64,), 2).requires_grad_()
    y = cl.layer_norm(x, w)  # only the weight learns
    gy = rand((20, 64), 3)
    gw, = torch.autograd.grad(y, w, gy)
    _, h, mu, r, *_ = norm64(x, w, None, 1e-5, gy)
    near(gw, (gy.double() * h).sum(0), EPS * 200 * (gy.double().abs() * (2 + h.abs())).sum(0), torch.float32)
    const = laid(torch.full((4, 100), 3.25, device="cuda"), layout).requires_grad_()
    y = cl.layer_norm(const)
    assert torch.equal(y, torch.zeros_like(y))
    bad = rand((4, 100), 5)
    bad[1, 7] = float("nan")
    bad[2, 9] = float("inf")
    y = cl.layer_norm(laid(bad, layout))
    assert torch.isnan(y[1]).all() and torch.isnan(y[2]).all() and torch.isfinite(y[[0, 3]]).all()


@pytest.mark.parametrize("dtype", LOW)
@pytest.mark.parametrize("n,d", [(500, 1000), (300, 4096), (7, 96), (40, 2056), (3, 12000), (20, 999)])
def test_layer_norm_without_parameters(n, d, dtype):
    """No weight, no bias: nothing is read for them, at any width and form of the windows."""
    check_norm(n, d, dtype, "rows", affine=False)
    check_norm(n, d, dtype, "features", affine=False)
    x = rand((n, d), 1, dtype).requires_grad_()
    b = rand((d,), 2).requires_grad_()
    y = cl.layer_norm(x, None, b)  # a bias alone
    gy = rand((n, d), 3, dtype)
    _, gb = torch.autograd.grad(y, (x, b), gy)
    near(gb, gy.double().sum(0), EPS * steps(n) * gy.double().abs().sum(0), torch.float32)


def test_layer_norm_parameters_at_odd_places():
    """Parameters that are slices, off the boundaries of wide reads."""
    for dtype, d, at in [(torch.bfloat16, 1024, 1), (torch.bfloat16, 1024, 4), (torch.float32, 512, 2), (torch.float16, 1001, 3)]:
        big = rand((2, d + 8), 5)
        w, b = big[0, at:at + d], big[1, at:at + d]
        x, gy = rand((33, d), 6, dtype).requires_grad_(), rand((33, d), 7, dtype)
        y = cl.layer_norm(x, w, b)
        gx, = torch.autograd.grad(y, x, gy)
        want = cl.layer_norm(x, w.clone(), b.clone())
        gwant, = torch.autograd.grad(want, x, gy)
        near(y, want.double(), 1e-5, dtype)
        near(gx, gwant.double(), 1e-5 * float(gwant.double().abs().max()), dtype)


def test_layer_norm_shapes_and_refusals():
    for shape in [(0, 5), (7,), (3, 4, 5)]:
        x = rand(shape, 4).requires_grad_()
        w = torch.ones(shape[-1], device="cuda", requires_grad=True)
        y = cl.layer_norm(x, w)
        assert y.shape == x.shape
        gx, gw = torch.autograd.grad(y.sum(), [x, w])
        assert gx.shape == x.shape and (x.numel() or torch.equal(gw, torch.zeros_like(gw)))
        near(y.reshape(-1, shape[-1]), norm64(x.reshape(-1, shape[-1]), w, None, 1e-5)[0], 1e-5, torch.float32)
    x = rand((4, 8), 5)
    w = torch.ones(8, device="cuda")
    for bad in (w[:7], w.double(), w.half()):
        with pytest.raises(RuntimeError):
            cl.layer_norm(x, bad)
        with pytest.raises(RuntimeError):
            cl.layer_norm(x, None, bad)
    with pytest.raises(RuntimeError):
        cl.layer_norm(x, w.cpu())
    with pytest.raises(RuntimeError):
        cl.layer_norm(x.long())
    with pytest.raises(RuntimeError):
        cl.layer_norm(rand((4, 0), 1))
    with pytest.raises(ValueError):
        cl.layer_norm(x, w, eps=-1.0)
    with pytest.raises(RuntimeError):
        cl.LogicLayerNorm(9).cuda()(x)


@pytest.mark.parametrize("layout", ["rows", "features"])
def test_layer_norm_gradient_by_differences(layout):
    x = laid(rand((5, 37), 1, torch.float64), layout).requires_grad_()
    w, b = rand((37,), 2, torch.float64).requires_grad_(), rand((37,), 3, torch.float64).requires_grad_()
    assert torch.autograd.gradcheck(lambda *a: cl.layer_norm(*a), (x, w, b), eps=1e-6, atol=1e-7, rtol=1e-6)


@pytest.mark.parametrize("layout", ["rows", "features"])
def test_layer_norm_repeats_its_bits(layout):
    a = check_norm(513, 700, torch.bfloat16, layout)
    b = check_norm(513, 700, torch.bfloat16, layout)
    assert torch.equal(a[4], b[4]) and all(torch.equal(p, q) for p, q in zip(a[5], b[5]))


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n,d", [(1, 1), (1, 2), (1, 8), (1, 784), (1, 5001), (5, 1)])
def test_layer_norm_of_one_row_or_one_feature(n, d, dtype, layout):
    """Where an axis has one entry its stride says nothing: every storage of the input with every one of the gradient."""
    for gy_layout in LAYOUTS:
        check_norm(n, d, dtype, layout, gy_layout=gy_layout)


def test_layer_norm_of_one_row_between_stack_and_cat():
    """Gradients of one row as autograd hands them over: columns of a wider matrix."""
    d = 96
    x, w, b = rand((1, d), 1).requires_grad_(), rand((d,), 2, shift=1.0).requires_grad_(), rand((d,), 3).requires_grad_()
    for join, g in [(lambda y: torch.stack([y, 2 * y.detach()], -1), rand((1, d, 2), 4)),
                    (lambda y: torch.cat([y.t(), y.detach().t(), y.detach().t()], 1), rand((d, 3), 5))]:
        y = cl.layer_norm(x, w, b)
        got = torch.autograd.grad(join(y), (x, w, b), g)
        gy = g[..., 0].reshape(1, d).clone()
        want = torch.autograd.grad(cl.layer_norm(x, w, b), (x, w, b), gy)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        *_, gx, gw, gb = norm64(x, w, b, 1e-5, gy)
        for p, q in zip(got, (gx, gw, gb)):
            assert (p.double() - q).abs().max() <= EPS * 16 * steps(d) * (1 + q.abs().max())


# -------------------------------------------------------------------------------------------------------------- losses
def logits64(z, actions, live, temperature):
    z = z.detach().double() / temperature
    full = torch.log_softmax(z, 1)
    a = torch.where(live, actions, 0)
    return full, full.gather(1, a[:, None])[:, 0]


def row_slack(z, lp, temperature, dtype):
    """Absolute error of a log-probability: the sum of v exponentials, its logarithm, and the differences to the maximum."""
    e = eps_of(dtype)
    z = z.detach().double()
    span = ((z - z.max(1, keepdim=True).values).nan_to_num(neginf=0.0).abs() / temperature)
    p = torch.softmax(z / temperature, 1).nan_to_num()
    return e * (steps(z.shape[1]) + 8 + 4 * (p * span).sum(1) + lp.nan_to_num(neginf=0.0).abs() * 2)


def grad_slack(full, c, lp_slack, dtype):
    p = full.exp()
    return (c.abs()[:, None] * (p * (lp_slack[:, None] + eps_of(dtype) * (8 + 4 * full.nan_to_num(neginf=0.0).abs()))) +
            eps_of(dtype) * 8 * c.abs()[:, None])


CASES = [(1, 1), (1, 2), (1, 10), (7, 3), (64, 10), (1000, 10), (33, 100), (5, 1000), (1025, 47), (3, 4099), (40, 2048)]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n,v", CASES)
def test_action_log_probs(n, v, dtype, layout):
    check_logp(n, v, dtype, layout)


@pytest.mark.parametrize("dtype", LOW)
@pytest.mark.parametrize("n,v,layout", [(9, 32768, "rows"), (3, 50001, "rows"), (4, 131072, "rows"), (2, 262144, "rows"),
                                        (2, 600001, "padded"), (300, 5000, "rows"), (2000, 129, "rows"), (100, 8192, "rows"),
                                        (31, 3000, "features"), (2, 40000, "features"), (3000, 1000, "features")])
def test_action_log_probs_sizes(n, v, layout, dtype):
    check_logp(n, v, dtype, layout)


def check_logp(n, v, dtype, layout, temperature=0.7):
    acc = torch.float64 if dtype == torch.float64 else torch.float32
    z = laid(rand((n, v), 20, dtype, 3.0), layout).requires_grad_()
    g = torch.Generator(device="cuda").manual_seed(3)
    act = torch.randint(0, v, (n,), generator=g, device="cuda")
    up = rand((n,), 21, acc)
    lp = cl.action_log_probs(z, act, temperature=temperature)
    with torch.no_grad():
        assert torch.equal(lp, cl.action_log_probs(z, act, temperature=temperature))
    assert lp.dtype == acc
    gz, = torch.autograd.grad(lp, z, up)
    full, want = logits64(z, act, torch.ones(n, dtype=torch.bool, device="cuda"), temperature)
    slack = row_slack(z, want, temperature, dtype)
    near(lp, want, slack, acc, "logp")
    c = up.double() / temperature
    grad = -c[:, None] * full.exp()
    grad[torch.arange(n, device="cuda"), act] += c
    near(gz, grad, grad_slack(full, c, slack, dtype), dtype, "gz")


def policy64(z, act, adv, old, ref, mask, clip, beta, temperature, reduction):
    n = z.shape[0]
    live = mask if mask is not None else torch.ones(n, dtype=torch.bool, device="cuda")
    full, lp = logits64(z, act, live, temperature)
    lp = torch.where(live, lp, 0.0)
    adv, old = adv.double(), old.double()
    ratio = torch.where(live, torch.exp(lp - old), 0.0)
    lo, hi = 1 - clip[0], 1 + clip[1]
    a, b = ratio * adv, ratio.clamp(lo, hi) * adv
    rows, slope = -torch.minimum(a, b), torch.where(a <= b, -a, 0.0)
    kl = None
    if ref is not None:
        q = ref.double() - lp
        kl = torch.where(live, torch.expm1(q) - q, 0.0)
        rows, slope = rows + beta * kl, slope - beta * torch.expm1(q)
    rows, slope = torch.where(live, rows, 0.0), torch.where(live, slope, 0.0)
    count = max(1, int(live.sum()))
    f = 1.0 / count if reduction == "mean" else 1.0
    c = slope * f / temperature
    gz = -c[:, None] * full.exp()
    at = torch.nonzero(live)[:, 0]
    gz[at, act[at]] += c[at]
    gz = torch.where(live[:, None], gz, 0.0)
    loss = rows if reduction == "none" else rows.sum() * f
    return loss, lp, ratio, kl, gz, rows, c, full, f


def policy_inputs(n, v, dtype, layout, masked=0.0, ref=True, seed=30, temperature=1.0, scale=2.0):
    acc = torch.float64 if dtype == torch.float64 else torch.float32
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = laid(rand((n, v), seed, dtype, scale), layout)
    act = torch.randint(0, v, (n,), generator=g, device="cuda")
    lp = torch.log_softmax(z.double() / temperature, 1).gather(1, act[:, None])[:, 0]
    # ratios inside the clip range and beyond it, none within 2 % of an edge
    step = torch.rand(n, generator=g, device="cuda", dtype=torch.float64) * 0.15
    step = torch.where(torch.rand(n, generator=g, device="cuda") < 0.4, step + 0.27, step)
    old = (lp + torch.where(torch.rand(n, generator=g, device="cuda") < 0.5, step, -step)).to(acc)
    adv = rand((n,), seed + 1, acc, 1.0, 0.3)
    refs = (lp + rand((n,), seed + 2, torch.float64, 0.5)).to(acc) if ref else None
    mask = torch.rand(n, generator=g, device="cuda") >= masked if masked else None
    return z, act, adv, old, refs, mask


def check_policy(n, v, dtype, layout, masked=0.0, ref=True, reduction="mean", temperature=1.0, upstream=None, clip=0.2,
                 beta=0.1, inputs=None):
    acc = torch.float64 if dtype == torch.float64 else torch.float32
    z, act, adv, old, refs, mask = inputs or policy_inputs(n, v, dtype, layout, masked, ref, temperature=temperature)
    if mask is not None:
        act = torch.where(mask, act, -100)
    z = z.detach().requires_grad_()
    r = cl.policy_loss(z, act, adv, old, ref_log_probs=refs, mask=mask, clip=clip, kl_coef=beta, temperature=temperature,
                       reduction=reduction)
    both = clip if isinstance(clip, tuple) else (clip, clip)
    loss, lp, ratio, kl, gz, rows, c, full, f = policy64(z, act, adv, old, refs, mask, both, beta, temperature, reduction)
    e = eps_of(dtype)
    lps = row_slack(z, lp, temperature, dtype)
    near(r.log_probs, lp, lps, acc, "logp")
    at = lps + e * (old.double().abs() + 8)
    near(r.ratio, ratio, ratio * at, acc, "ratio")
    row = ratio * (at + 4 * e) * adv.double().abs()
    dslope = row
    if refs is not None:
        q = refs.double() - lp
        kls = torch.expm1(q).abs() * (lps + e * (refs.double().abs() + 8)) + 8 * e * (torch.exp(q) + q.abs())
        kls = torch.where(kl == 0, torch.zeros_like(kls) if mask is None else kls * mask, kls)
        near(r.kl, kl, kls, acc, "kl")
        row = row + beta * kls
        dslope = dslope + beta * torch.exp(q) * (lps + e * (refs.double().abs() + 8))
    else:
        assert r.kl is None
    row = row + 4 * e * rows.abs()
    near(r.loss, loss, row if reduction == "none" else f * (row.sum() + e * steps(n) * rows.abs().sum()), acc, "loss")
    if upstream is None:
        upstream = torch.ones_like(r.loss) if reduction != "none" else rand((n,), 50, acc)
    gr, = torch.autograd.grad(r.loss, z, upstream, retain_graph=True)
    u = upstream.double()
    want = gz * (u[:, None] if reduction == "none" else u)
    cu = c * u
    slack = grad_slack(full, cu, lps, dtype) + (dslope * f / temperature * u.abs())[:, None] * 1.0
    if mask is not None:
        slack = slack * mask[:, None]
    near(gr, want, slack, dtype, "gz")
    again, = torch.autograd.grad(r.loss, z, upstream)
    near(again, want, slack, dtype, "gz again")
    with torch.no_grad():
        bare = cl.policy_loss(z, act, adv, old, ref_log_probs=refs, mask=mask, clip=clip, kl_coef=beta,
                              temperature=temperature, reduction=reduction)
    assert torch.equal(bare.loss, r.loss) and torch.equal(bare.log_probs, r.log_probs)
    return r, gr


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n,v", CASES)
def test_policy_loss(n, v, dtype, layout):
    check_policy(n, v, dtype, layout, masked=0.3 if n > 5 else 0.0)


@pytest.mark.parametrize("dtype", LOW)
@pytest.mark.parametrize("n,v,layout", [(9, 32768, "rows"), (3, 50001, "rows"), (4, 131072, "rows"), (2, 262144, "rows"),
                                        (2, 600001, "padded"), (300, 5000, "rows"), (2000, 129, "rows"), (100, 8192, "rows"),
                                        (31, 3000, "features"), (3000, 1000, "features"), (70000, 5, "features")])
def test_policy_loss_sizes(n, v, layout, dtype):
    check_policy(n, v, dtype, layout, masked=0.2 if n > 8 else 0.0)


@pytest.mark.parametrize("layout", ["rows", "features"])
@pytest.mark.parametrize("n,v", [(200, 10), (20, 3000)])
def test_policy_loss_variants(n, v, layout):
    check_policy(n, v, torch.float32, layout, ref=False)
    check_policy(n, v, torch.float32, layout, reduction="sum", masked=0.5)
    check_policy(n, v, torch.float32, layout, reduction="none", masked=0.5)
    check_policy(n, v, torch.bfloat16, layout, reduction="none")
    check_policy(n, v, torch.float32, layout, temperature=1.7)
    check_policy(n, v, torch.float32, layout, clip=(0.2, 0.25))
    check_policy(n, v, torch.float32, layout, upstream=torch.tensor(0.37, device="cuda"), masked=0.2)
    check_policy(n, v, torch.bfloat16, layout, upstream=torch.tensor(1024.0, device="cuda"))


@pytest.mark.parametrize("layout", ["rows", "features"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [10, 5000])
def test_masked_logits(v, dtype, layout):
    """Forbidden classes: -inf or the type's lowest value, up to rows where one class is left, or none."""
    n = 12
    z, act, adv, old, refs, _ = policy_inputs(n, v, dtype, "rows")
    low = torch.finfo(dtype).min
    for fill in (float("-inf"), low):
        y = z.clone()
        y[0, :] = fill
        y[0, act[0]] = 1.0                       # one class left
        y[1, ::2] = fill
        y[1, act[1]] = 0.5
        y[2, act[2]] = fill                      # the chosen one forbidden
        others = torch.arange(n, device="cuda") != 2
        y = laid(y, layout).requires_grad_()
        lp = cl.action_log_probs(y, act)
        full, want = logits64(y, act, torch.ones(n, dtype=torch.bool, device="cuda"), 1.0)
        near(lp[others], want[others], row_slack(y, want, 1.0, dtype)[others], torch.float32)
        assert lp[2] == float("-inf") if fill != low else lp[2] < -1e37
        assert lp[0] == 0.0
        gz, = torch.autograd.grad(lp.sum(), y)
        assert torch.isfinite(gz).all()
        assert (gz[0] == 0).all()
    y = z.clone()
    y[3, :] = low                                # every class at the lowest value: uniform
    y = laid(y, layout)
    lp = cl.action_log_probs(y, act)
    assert abs(float(lp[3]) + math.log(v)) <= EPS * (steps(v) + 4 * math.log(v))
    y = z.clone()
    y[4, :] = float("-inf")                      # nothing left: no distribution
    y[5, 0] = float("nan")
    y[6, 1] = float("inf")
    y = laid(y, layout).requires_grad_()
    lp = cl.action_log_probs(y, act)
    gz, = torch.autograd.grad(lp.sum(), y)
    for i in (4, 5, 6):
        assert torch.isnan(lp[i]) and torch.isnan(gz[i]).all()
    assert torch.isfinite(lp[[0, 1, 2, 3, 7]]).all() and torch.isfinite(gz[[0, 1, 2, 3, 7]]).all()
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[4:7] = False                            # rows that do not count may hold anything
    old[5] = float("nan")
    adv[6] = float("inf")
    r = cl.policy_loss(y, act, adv, old, ref_log_probs=refs, mask=keep, kl_coef=0.1)
    gz, = torch.autograd.grad(r.loss, y)
    assert torch.isfinite(r.loss) and torch.isfinite(gz).all() and (gz[4:7] == 0).all()
    assert (r.log_probs[4:7] == 0).all() and (r.ratio[4:7] == 0).all() and (r.kl[4:7] == 0).all()


# A row's form by its length: lanes of a warp, a warp, a block, a cluster, and beyond a cluster (read twice).
LENGTHS = [3, 17, 47, 300, 1777, 3000, 20000, 50001, 131072, 600001]


def loss_inputs(z, seed=30, temperature=1.0):
    """What ``policy_inputs`` makes, for given logits."""
    n, v = z.shape
    acc = torch.float64 if z.dtype == torch.float64 else torch.float32
    g = torch.Generator(device="cuda").manual_seed(seed)
    act = torch.randint(0, v, (n,), generator=g, device="cuda")
    act[0] = z[0].argmax()
    lp = torch.log_softmax(z.double() / temperature, 1).gather(1, act[:, None])[:, 0]
    step = torch.rand(n, generator=g, device="cuda", dtype=torch.float64) * 0.15
    step = torch.where(torch.rand(n, generator=g, device="cuda") < 0.4, step + 0.27, step)
    old = (lp + torch.where(torch.rand(n, generator=g, device="cuda") < 0.5, step, -step)).to(acc)
    refs = (lp + rand((n,), seed + 2, torch.float64, 0.5)).to(acc)
    return z, act, rand((n,), seed + 1, acc, 1.0, 0.3), old, refs, None


@pytest.mark.parametrize("layout", ["rows", "padded", "features"])
@pytest.mark.parametrize("v", LENGTHS)
@pytest.mark.parametrize("shift,scale,temperature", [(1e3, 2.0, 1.0), (-1e5, 2.0, 1.0), (1e6, 2.0, 1.0), (0.0, 3.0, 0.01),
                                                     (30.0, 0.05, 0.01)])
def test_losses_of_logits_far_from_zero(v, shift, scale, temperature, layout):
    """What the logits have in common cancels exactly, in the sum, in the gradient and in the action's own entry, whatever
    the row's form, and a small temperature does not magnify its rounding."""
    n = 5
    z = laid(rand((n, v), 40, torch.float32, scale, shift), layout)
    z, act, *_ = inputs = loss_inputs(z, temperature=temperature)
    check_policy(n, v, torch.float32, layout, temperature=temperature, inputs=inputs)
    z = z.detach().requires_grad_()
    lp = cl.action_log_probs(z, act, temperature=temperature)
    up = rand((n,), 21)
    gz, = torch.autograd.grad(lp, z, up)
    full, want = logits64(z, act, torch.ones(n, dtype=torch.bool, device="cuda"), temperature)
    slack = row_slack(z, want, temperature, torch.float32)
    near(lp, want, slack, torch.float32, "logp")
    c = up.double() / temperature
    grad = -c[:, None] * full.exp()
    grad[torch.arange(n, device="cuda"), act] += c
    near(gz, grad, grad_slack(full, c, slack, torch.float32), torch.float32, "gz")


@pytest.mark.parametrize("layout", ["rows", "padded", "features"])
@pytest.mark.parametrize("dtype", LOW)
@pytest.mark.parametrize("v", LENGTHS)
def test_rows_filled_with_one_value(v, dtype, layout):
    """A mask by a large finite value that leaves nothing: every class has probability 1 / v, at any temperature."""
    fills = [-1e4, 6e4] if dtype == torch.float16 else [-1e4, -1e9, 1e30, -1e37, -3e38]
    z = laid(torch.tensor(fills, device="cuda", dtype=dtype)[:, None].expand(-1, v), layout).requires_grad_()
    n = len(fills)
    act = torch.arange(n, device="cuda") * 7 % v
    for temperature in (1.0, 0.02):
        lp = cl.action_log_probs(z, act, temperature=temperature)
        assert (lp.double() + math.log(v)).abs().max() <= EPS * (steps(v) + 4 * math.log(v))
        gz, = torch.autograd.grad(lp.sum(), z)
        want = torch.full((n, v), -1.0 / v, dtype=torch.float64, device="cuda")
        want[torch.arange(n, device="cuda"), act] += 1.0
        near(gz, want / temperature, EPS * (steps(v) + 16) * (want.abs() + 1 / v) / temperature, dtype, "gz")
        r = cl.policy_loss(z, act, torch.full((n,), -2.0, device="cuda"), lp.detach(), temperature=temperature)
        gz, = torch.autograd.grad(r.loss, z)     # ratios of 1: the slope is the negative advantage
        near(gz, want * 2 / n / temperature, EPS * (steps(v) + 16) * (want.abs() + 1 / v) * 2 / n / temperature, dtype,
             "policy gz")


@pytest.mark.parametrize("layout", ["rows", "features"])
@pytest.mark.parametrize("v", [10, 3000])
def test_policy_loss_edges(v, layout):
    z, act, adv, old, refs, _ = policy_inputs(6, v, torch.float32, layout)
    none = torch.zeros(6, dtype=torch.bool, device="cuda")
    z = z.requires_grad_()
    r = cl.policy_loss(z, act, adv, old, ref_log_probs=refs, mask=none, kl_coef=0.1)
    gz, = torch.autograd.grad(r.loss, z)
    assert r.loss == 0 and (gz == 0).all()       # nothing counts
    act2 = act.clone()
    act2[2] = v                                  # no such class
    act2[3] = -1
    r = cl.policy_loss(z, act2, adv, old, reduction="none")
    gz, = torch.autograd.grad(r.loss.nan_to_num().sum(), z)
    assert torch.isnan(r.loss[2:4]).all() and torch.isfinite(r.loss[[0, 1, 4, 5]]).all()
    assert torch.isnan(gz[2:4]).all() and torch.isfinite(gz[[0, 1, 4, 5]]).all()
    empty = cl.policy_loss(z[:0], act[:0], adv[:0], old[:0])
    assert empty.loss == 0 and empty.log_probs.shape == (0,)
    ge, = torch.autograd.grad(empty.loss, z)
    assert (ge == 0).all()
    # the ratio's branches, both signs of the advantage: gradient only where the unclipped term is the smaller
    lp = cl.action_log_probs(z.detach(), act)
    old = lp - torch.tensor([0.5, 0.5, -0.5, -0.5, 0.0, 0.0], device="cuda")
    adv = torch.tensor([1.0, -1.0, 1.0, -1.0, 1.0, -1.0], device="cuda")
    r = cl.policy_loss(z, act, adv, old, reduction="none")
    gz, = torch.autograd.grad(r.loss.sum(), z)
    assert (gz.abs().sum(1) > 0).tolist() == [False, True, True, False, True, True]


def test_losses_take_leading_axes():
    z, act, adv, old, refs, mask = policy_inputs(24, 7, torch.float32, "rows", masked=0.3)
    flat = cl.policy_loss(z, act, adv, old, ref_log_probs=refs, mask=mask, kl_coef=0.1)
    s = (2, 3, 4)
    deep = cl.policy_loss(z.view(*s, 7), act.view(s).int(), adv.view(s), old.view(s), ref_log_probs=refs.view(s),
                          mask=mask.view(s), kl_coef=0.1)
    assert torch.equal(flat.loss, deep.loss) and deep.log_probs.shape == s and torch.equal(flat.kl, deep.kl.reshape(-1))
    assert cl.action_log_probs(z.view(*s, 7), act.view(s)).shape == s
    one = cl.action_log_probs(z[0], act[0])
    assert one.shape == () and torch.allclose(one, flat.log_probs.new_tensor(float(cl.action_log_probs(z, act)[0])))


@pytest.mark.parametrize("layout", ["rows", "features"])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_loss_gradients_by_differences(layout, reduction):
    z, act, adv, old, refs, mask = policy_inputs(8, 5, torch.float64, layout, masked=0.3)
    z = z.requires_grad_()
    assert torch.autograd.gradcheck(
        lambda t: cl.policy_loss(t, act, adv, old, ref_log_probs=refs, mask=mask, kl_coef=0.2, temperature=1.3,
                                 reduction=reduction).loss, (z,), eps=1e-6, atol=1e-7, rtol=1e-6)
    assert torch.autograd.gradcheck(lambda t: cl.action_log_probs(t, act, mask=mask, temperature=1.3), (z,), eps=1e-6,
                                    atol=1e-7, rtol=1e-6)


def test_losses_repeat_their_bits():
    for n, v, layout in [(999, 10, "features"), (50, 50001, "rows"), (700, 333, "rows")]:
        inputs = policy_inputs(n, v, torch.float32, layout, masked=0.2)
        a = check_policy(n, v, torch.float32, layout, inputs=inputs)
        b = check_policy(n, v, torch.float32, layout, inputs=inputs)
        assert torch.equal(a[0].loss, b[0].loss) and torch.equal(a[1], b[1])


def test_loss_refusals():
    z, act, adv, old, refs, mask = policy_inputs(6, 5, torch.float32, "rows", masked=0.3)
    for bad in (act[:5], act.float(), act[:, None], act.bool()):
        with pytest.raises(RuntimeError):
            cl.action_log_probs(z, bad)
        with pytest.raises(RuntimeError):
            cl.policy_loss(z, bad, adv, old)
    for bad in (mask[:5], mask.float()):
        with pytest.raises(RuntimeError):
            cl.action_log_probs(z, act, mask=bad)
    with pytest.raises(RuntimeError):
        cl.policy_loss(z, act, adv[:5], old)
    with pytest.raises(RuntimeError):
        cl.policy_loss(z, act, adv, old.cpu())
    with pytest.raises(RuntimeError):
        cl.policy_loss(z.cpu(), act, adv, old)
    with pytest.raises(RuntimeError):
        cl.policy_loss(z.long(), act, adv, old)
    with pytest.raises(RuntimeError):
        cl.action_log_probs(z[:, :0], act)
    for t in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError):
            cl.action_log_probs(z, act, temperature=t)
        with pytest.raises(ValueError):
            cl.policy_loss(z, act, adv, old, temperature=t)
    with pytest.raises(ValueError):
        cl.policy_loss(z, act, adv, old, clip=-0.1)
    with pytest.raises(ValueError):
        cl.policy_loss(z, act, adv, old, reduction="average")


# --------------------------------------------------------------------------------------------------- second derivatives
@pytest.mark.parametrize("layout", ["rows", "features"])
def test_dropout_second_derivatives(layout):
    x = laid(rand((9, 14), 1, torch.float64), layout).requires_grad_()
    assert torch.autograd.gradgradcheck(lambda t: cl.dropout(t ** 3, 0.3, seed=2), (x,), eps=1e-6, atol=1e-7, rtol=1e-6)
    assert torch.autograd.gradgradcheck(lambda t: cl.dropout((t ** 3).reshape(9, 2, 7), 0.3, seed=2), (x,), eps=1e-6,
                                        atol=1e-7, rtol=1e-6)
    g, = torch.autograd.grad(cl.dropout(x, 0.3, seed=2).sum(), x, create_graph=True)
    again, = torch.autograd.grad((g * x).sum(), x)  # a gradient that is constant
    assert torch.equal(again, g)


@pytest.mark.parametrize("layout", ["rows", "features", "strided"])
@pytest.mark.parametrize("name", ["layer_norm", "action_log_probs", "policy_loss", "policy_loss none"])
def test_second_derivatives_are_refused(name, layout):
    """A first derivative under create_graph is right; differentiated again it raises instead of leaving its term out."""
    z, act, adv, old, refs, mask = policy_inputs(6, 20, torch.float32, layout)
    w, b = rand((20,), 1).requires_grad_(), rand((20,), 2).requires_grad_()
    z = z.requires_grad_()
    calls = {"layer_norm": (lambda: cl.layer_norm(z, w, b), (z, w)),
             "action_log_probs": (lambda: cl.action_log_probs(z, act), (z,)),
             "policy_loss": (lambda: cl.policy_loss(z, act, adv, old, ref_log_probs=refs, kl_coef=0.1).loss, (z,)),
             "policy_loss none": (lambda: cl.policy_loss(z, act, adv, old, reduction="none").loss, (z,))}
    call, inputs = calls[name]
    plain = torch.autograd.grad(call().sum(), inputs)
    for up in (torch.ones_like(call()), torch.ones_like(call()).requires_grad_()):
        for k, at in enumerate(inputs):
            grads = torch.autograd.grad(call(), inputs, up, create_graph=True)
            assert all(torch.equal(p, q) for p, q in zip(plain, grads))
            with pytest.raises(RuntimeError, match="second derivative"):
                torch.autograd.grad((grads[k] ** 2).sum() + (z ** 2).sum(), z)
    # the bias's gradient is a sum of the incoming one: constant where that is
    if name == "layer_norm":
        gb, = torch.autograd.grad(call().sum(), b, create_graph=True)
        assert torch.equal(torch.autograd.grad((gb * b).sum(), b)[0], gb)


def test_operators_on_a_side_stream():
    """Work is enqueued on the current stream: results there equal those on the default one."""
    z, act, adv, old, refs, mask = policy_inputs(500, 1000, torch.bfloat16, "rows", masked=0.2)
    x = rand((500, 1000), 3, torch.bfloat16)
    want = (cl.policy_loss(z, act, adv, old, ref_log_probs=refs, mask=mask).loss, cl.layer_norm(x), cl.dropout(x, 0.5, seed=1))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = (cl.policy_loss(z, act, adv, old, ref_log_probs=refs, mask=mask).loss, cl.layer_norm(x),
               cl.dropout(x, 0.5, seed=1))
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_training_step_under_a_graph():
    """Norm, layers, dropout and the loss captured as one step replay to the eager step's gradients."""
    torch.manual_seed(0)
    norm, a, b = cl.LogicLayerNorm(32).cuda(), cl.LogicLayer(32, 64).cuda(), cl.LogicLayer(64, 60).cuda()
    x = torch.randn(48, 32, device="cuda")
    z, act, adv, old, refs, mask = policy_inputs(48, 6, torch.float32, "features", masked=0.2)
    params = [norm.weight, norm.bias, a.weights, b.weights]

    def body():
        h = b(cl.dropout(a(torch.sigmoid(norm(x))), 0.1, seed=4, rescale=False))
        logits = cl.GroupSum(6, tau=2.0)(h)
        r = cl.policy_loss(logits, act, adv, old, ref_log_probs=refs, mask=mask, kl_coef=0.1)
        grads = torch.autograd.grad(r.loss, params)
        return (r.loss.detach(),) + grads

    want = body()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = body()
    graph.replay()
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert (w - g).abs().max() <= 1e-5 * w.abs().max()


@pytest.mark.parametrize("layout", ["rows", "features"])
def test_offsets_past_32_bits(layout):
    """Tensors of more than 2^31 elements: the last rows are right."""
    n, d = (33000, 65536) if layout == "rows" else (65536, 33000)
    free, _ = torch.cuda.mem_get_info()
    if free < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    base = torch.empty(n, d, dtype=torch.bfloat16, device="cuda") if layout == "rows" else \
        torch.empty(d, n, dtype=torch.bfloat16, device="cuda").t()
    base.fill_(0.5)
    tail = rand((6, d), 1, torch.bfloat16)
    base[-6:] = tail
    x = base.requires_grad_()
    y = cl.dropout(x, 0.25, seed=3, rescale=False)
    keep = torch.from_numpy(words(6, d, 3, 0, first=n - 6).astype(np.int64)).cuda() >= round(0.25 * 2 ** 32)
    assert torch.equal(y[-6:], torch.where(keep, tail, torch.zeros((), dtype=tail.dtype, device="cuda")))
    del y
    gy = torch.zeros_like(base)
    gy[-6:] = rand((6, d), 2, torch.bfloat16)
    y = cl.layer_norm(x)
    gx, = torch.autograd.grad(y, x, gy)
    y64, h, mu, r, w64, t, gx64, *_ = norm64(tail, None, None, 1e-5, gy[-6:])
    spread = 1 + (mu.abs() + tail.double().abs().mean(1, keepdim=True)) * r + h.abs()
    near(y[-6:], y64, EPS * steps(d) * spread, torch.bfloat16, "y")
    big = t.abs() + t.abs().mean(1, keepdim=True) + (1 + h.abs()) * ((t * h).abs().mean(1, keepdim=True) +
                                                                  (t.abs() * spread).mean(1, keepdim=True))
    near(gx[-6:], gx64, 2 * EPS * steps(d) * r * big, torch.bfloat16, "gx")
    del y, gx, gy
    act = torch.zeros(n, dtype=torch.int64, device="cuda")
    act[-6:] = torch.tensor([0, 5, d - 1, d // 2, 7, d - 3], device="cuda")
    up = torch.zeros(n, device="cuda")
    up[-6:] = 1.5
    lp = cl.action_log_probs(x, act)
    gz, = torch.autograd.grad(lp, x, up)
    full, want = logits64(tail, act[-6:], torch.ones(6, dtype=torch.bool, device="cuda"), 1.0)
    slack = row_slack(tail, want, 1.0, torch.bfloat16)
    near(lp[-6:], want, slack, torch.float32, "logp")
    grad = -1.5 * full.exp()
    grad[torch.arange(6, device="cuda"), act[-6:]] += 1.5
    near(gz[-6:], grad, grad_slack(full, up[-6:].double(), slack, torch.bfloat16), torch.bfloat16, "gz")
    assert (gz[:-6:997] == 0).all()
    del gz
    r = cl.policy_loss(x, act, up, lp.detach(), reduction="sum")
    gz, = torch.autograd.grad(r.loss, x)
    # ratios of exactly 1: the slope is -1.5
    near(gz[-6:], -grad, grad_slack(full, up[-6:].double(), slack, torch.bfloat16), torch.bfloat16, "policy gz")


def test_status_codes():
    lib = L.lib()
    t = torch.zeros(64, device="cuda")
    p = t.data_ptr()
    assert lib.clb_dropout(0, p, 3, 4, 4, 0, 0.5, 1, 0, 0, None, p, 4, None) == L.CLB_ERR_INVALID  # ldx < row
    assert lib.clb_layer_norm_forward(0, p, 4, 4, 4, 0, None, None, 1e-5, p, 3, None, None, None, 0, None) == L.CLB_ERR_INVALID
    assert lib.clb_action_logp(0, p, 4, 4, 5, 0, p, None, 1.0, p, None, None) == L.CLB_ERR_INVALID
