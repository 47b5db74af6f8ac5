"""Residual sums with their norms against the definition in 64 bits, forward and
gradients.  Tolerances: an output's own rounding (half a step), and 2^-24 of the
absolute terms for each fp32 operation on the way: 48 of them cover the chains of a
row (sums over the hidden size in parts of at most 24 by a thread, then pairs), sums
over rows count each row."""
import pytest
import torch

from ananta_ocr_b200 import norms
from ananta_ocr_b200 import _lib as L
from step_testutil import DT, U, half_step, norm_forward, norm_grads

pytestmark = pytest.mark.gpu
OPS = 48


def make(rows, hidden, dt, groups=0, post=False, wt="fp32", gt=None, seed=0, grad=False):
    g = torch.Generator().manual_seed(seed + rows * 7 + hidden)
    dt, wt = DT[dt], DT[wt]
    rnd = lambda *s, dtype=dt, std=1.0, mean=0.0: (torch.randn(*s, generator=g) * std + mean).to(dtype).cuda()  # noqa: E731
    t = dict(y=rnd(rows, hidden), residual=rnd(rows, hidden, std=2.0), weight=rnd(hidden, dtype=wt, std=0.3, mean=1.0),
             gate=rnd(groups, hidden, dtype=DT[gt] if gt else dt) if groups else None,
             post=rnd(hidden, dtype=wt, std=0.3, mean=1.0) if post else None)
    if grad:
        for v in t.values():
            if v is not None:
                v.requires_grad_()
    return t, rnd(rows, hidden), rnd(rows, hidden)


def up(t):
    return {k: None if v is None else v.detach().double().cpu() for k, v in t.items()}


def check_forward(t, stream, normed, eps, scale):
    r = up(t)
    dt = t["y"].dtype
    s, h = norm_forward(r["y"], r["residual"], r["weight"], r["gate"], r["post"], eps, scale)
    z = s if r["residual"] is None else s - r["residual"]
    size = z.abs() + (0 if r["residual"] is None else r["residual"].abs())
    r2 = (s.square().mean(-1, keepdim=True) + eps).rsqrt()
    # fp16 numbers below 2^-14 are multiples of 2^-24: rounded, they are off by up to 2^-25 whatever their size
    least = 2.0 ** -25 if dt == torch.float16 else 1e-38
    if stream is not None:
        tol = half_step(dt) * s.abs() + OPS * U * size + least
        assert ((stream.double().cpu() - s).abs() <= tol).all()
    tol = half_step(dt) * h.abs() + OPS * U * size * r2 * r["weight"].abs() + least
    assert ((normed.double().cpu() - h).abs() <= tol).all()


def check_grads(t, ds, dh, got, eps, scale):
    r = up(t)
    dt, rows = t["y"].dtype, t["y"].shape[0]
    zero = torch.zeros_like(r["y"])
    want = norm_grads(r["y"], r["residual"], r["weight"], r["gate"], r["post"], eps, scale,
                      zero if ds is None else ds.double().cpu(), dh.double().cpu())
    for name, g in got.items():
        if g is None:
            continue
        w, terms = want[name]
        w, terms = w.reshape(g.shape), terms.reshape(g.shape)
        n = OPS + (rows if name in ("weight", "gate", "post") else 0)
        tol = half_step(g.dtype) * w.abs() + n * U * terms + (2.0 ** -25 if g.dtype == torch.float16 else 1e-38)
        off = (g.double().cpu() - w).abs()
        assert (off <= tol).all(), (name, (off / tol).max())


SHAPES = [(1, 1), (1, 8), (3, 24), (8, 1280), (5, 1283), (2, 2048), (7, 2056), (3, 4104), (2, 8191), (3, 8192), (130, 72)]


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,hidden", SHAPES)
def test_forward(rows, hidden, dt):
    for groups, post, wt, scale in ((0, False, "fp32", 1.0), (1, True, dt, 0.5), (rows, False, dt, -0.25)):
        t, _, _ = make(rows, hidden, dt, groups, post, wt)
        s, h = norms.add_rms_norm(t["y"], t["residual"], t["weight"], 1e-5, gate=t["gate"], post_weight=t["post"], scale=scale)
        check_forward(t, s, h, 1e-5, scale)
    t, _, _ = make(rows, hidden, dt)
    t["residual"] = None
    check_forward(t, None, norms.rms_norm(t["y"], t["weight"], 1e-5), 1e-5, 1.0)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,hidden", SHAPES[1:])
def test_gradients(rows, hidden, dt):
    for groups, post, wt, gt, scale in ((0, False, "fp32", None, 1.0), (1, True, dt, "fp32", 0.5), (rows, True, "fp32", dt, 2.0)):
        t, ds, dh = make(rows, hidden, dt, groups, post, wt, gt, grad=True)
        out = norms.add_rms_norm(t["y"], t["residual"], t["weight"], 1e-5, gate=t["gate"], post_weight=t["post"], scale=scale)
        names = [k for k, v in t.items() if v is not None]
        got = torch.autograd.grad(out, [t[k] for k in names], [ds, dh])
        check_grads(t, ds, dh, dict(zip(names, got)), 1e-5, scale)


@pytest.mark.parametrize("rows,groups", [(2000, 4), (1500, 500), (997, 1)])
def test_gradients_of_many_rows(rows, groups):
    """Groups of more rows than a CTA takes, and of fewer."""
    t, ds, dh = make(rows, 136, "bf16", groups, True, grad=True)
    out = norms.add_rms_norm(t["y"], t["residual"], t["weight"], 1e-6, gate=t["gate"], post_weight=t["post"], scale=0.5)
    names = list(t)
    check_grads(t, ds, dh, dict(zip(names, torch.autograd.grad(out, list(t.values()), [ds, dh]))), 1e-6, 0.5)


@pytest.mark.parametrize("hidden,groups,post,dt", [(264, 5, True, "bf16"), (4104, 1, False, "fp16"), (512, 0, True, "fp32"), (520, 7000, True, "bf16")])
def test_forward_of_many_rows(hidden, groups, post, dt):
    """Rows enough for a CTA to take several, whatever the hidden size."""
    rows = 14000 if hidden < 4000 else 2000
    t, _, _ = make(rows, hidden, dt, groups, post)
    check_forward(t, *norms.add_rms_norm(t["y"], t["residual"], t["weight"], 1e-6, gate=t["gate"], post_weight=t["post"],
                                         scale=0.5), 1e-6, 0.5)


@pytest.mark.parametrize("hidden,dt", [(656, "fp32"), (768, "fp32"), (1536, "bf16"), (1544, "bf16"), (2048, "fp16")])
def test_rings_around_48_kb(hidden, dt):
    """The fetched rows and the static part together pass the default limit of shared memory."""
    t, ds, dh = make(5, hidden, dt, 1, True, grad=True)
    out = norms.add_rms_norm(t["y"], t["residual"], t["weight"], 1e-5, gate=t["gate"], post_weight=t["post"])
    check_grads(t, ds, dh, dict(zip(t, torch.autograd.grad(out, list(t.values()), [ds, dh]))), 1e-5, 1.0)
    t, _, _ = make(16000, hidden, dt, 1, True)
    check_forward(t, *norms.add_rms_norm(t["y"], t["residual"], t["weight"], 1e-5, gate=t["gate"], post_weight=t["post"]), 1e-5, 1.0)


def test_gradients_against_differences():
    """Along random directions: the 64-bit definition's central difference with a step of
    1e-6 is off by 1e-9 of the values here; the gradients are fp32."""
    t, ds, dh = make(6, 40, "fp32", 2, True, grad=True)
    out = norms.add_rms_norm(t["y"], t["residual"], t["weight"], 1e-5, gate=t["gate"], post_weight=t["post"], scale=0.7)
    grads = dict(zip(t, torch.autograd.grad(out, list(t.values()), [ds, dh])))
    r = up(t)
    wants = norm_grads(**r, eps=1e-5, scale=0.7, ds=ds.double().cpu(), dh=dh.double().cpu())
    gen = torch.Generator().manual_seed(9)
    for name in t:
        v = torch.randn(r[name].shape, generator=gen, dtype=torch.float64)

        def loss(h):
            q = dict(r)
            q[name] = q[name] + h * v
            s, n = norm_forward(**q, eps=1e-5, scale=0.7)
            return (s * ds.double().cpu()).sum() + (n * dh.double().cpu()).sum()

        diff = (loss(1e-6) - loss(-1e-6)) / 2e-6
        got = (grads[name].double().cpu() * v).sum()
        terms = (wants[name][1].reshape(v.shape) * v.abs()).sum()
        assert abs(got - diff) <= (OPS + 6) * U * terms + 1e-6, name


def test_rms_norm_gradients():
    t, _, dh = make(9, 200, "bf16", grad=True)
    h = norms.rms_norm(t["y"], t["weight"], 1e-6)
    dy, dw = torch.autograd.grad(h, [t["y"], t["weight"]], dh)
    t["residual"] = None
    check_grads(t, None, dh, {"y": dy, "weight": dw}, 1e-6, 1.0)


def test_leaves_keep_gradients_of_their_own():
    """The plain sum's two gradients are one tensor; the leaves' are not."""
    t, ds, dh = make(4, 64, "fp32", grad=True)
    for _ in range(2):
        s, h = norms.add_rms_norm(t["y"], t["residual"], t["weight"], 1e-6)
        torch.autograd.backward([s, h], [ds, dh])
    t["y"].grad.zero_()
    check_grads({**t}, ds, dh, {"residual": t["residual"].grad / 2, "weight": t["weight"].grad / 2}, 1e-6, 1.0)
    got = norms.add_rms_norm_backward(ds, dh, t["y"].detach(), t["residual"].detach(), t["weight"].detach(), 1e-6, scale=0.5)
    check_grads(t, ds, dh, {"y": got.y, "residual": got.residual}, 1e-6, 0.5)


def test_second_derivatives_are_refused():
    t, ds, dh = make(4, 64, "fp32", grad=True)
    h = norms.rms_norm(t["y"], t["weight"], 1e-6)
    (dy,) = torch.autograd.grad(h.square().sum(), [t["y"]], create_graph=True)
    with pytest.raises(RuntimeError):
        dy.sum().backward()


def test_only_one_output_is_used():
    t, ds, dh = make(4, 64, "fp32", grad=True)
    s, h = norms.add_rms_norm(t["y"], t["residual"], t["weight"], 1e-6)
    (dy,) = torch.autograd.grad(s, [t["y"]], ds, retain_graph=True)
    assert torch.equal(dy, ds)
    (dy,) = torch.autograd.grad(h, [t["y"]], dh)
    check_grads(t, None, dh, {"y": dy}, 1e-6, 1.0)


def test_shapes_and_strides():
    """Rows out of a wider tensor, an odd offset, more dimensions, a transposed gradient."""
    g = torch.Generator().manual_seed(1)
    wide = torch.randn(6, 3 * 80 + 1, generator=g).bfloat16().cuda()
    for y, res in ((wide[:, 80:160], wide[:, :80]), (wide[:, 81:161], wide[:, 1:81]), (wide[::2, :80], wide[1::2, 160:240]),
                   (wide[:, :160:2], wide[:, 1:161:2])):
        t = dict(y=y, residual=res, weight=torch.ones(80).cuda(), gate=None, post=None)
        check_forward(t, *norms.add_rms_norm(y, res, t["weight"], 1e-6), 1e-6, 1.0)
    y, res = (torch.randn(2, 3, 48, generator=g).cuda().requires_grad_() for _ in range(2))
    w = torch.ones(48, device="cuda", requires_grad=True)
    s, h = norms.add_rms_norm(y, res, w, 1e-6)
    assert s.shape == h.shape == (2, 3, 48)
    up = torch.randn(48, 3, 2, generator=g).cuda().permute(2, 1, 0)
    dy, dr, dw = torch.autograd.grad([s, h], [y, res, w], [up, up])
    assert dy.shape == y.shape and dw.shape == w.shape
    t = dict(y=y.reshape(6, 48), residual=res.reshape(6, 48), weight=w, gate=None, post=None)
    check_grads(t, up.reshape(6, 48), up.reshape(6, 48), {"y": dy.reshape(6, 48), "residual": dr.reshape(6, 48), "weight": dw},
                1e-6, 1.0)


def test_rows_that_are_one_row():
    """A broadcast residual and broadcast gradients."""
    t, ds, dh = make(5, 88, "bf16")
    t["residual"] = t["residual"][:1].expand(5, 88)
    check_forward(t, *norms.add_rms_norm(t["y"], t["residual"], t["weight"], 1e-6), 1e-6, 1.0)
    ds, dh = ds[:1].expand(5, 88), dh[:1, :1].expand(5, 88)
    got = norms.add_rms_norm_backward(ds, dh, t["y"], t["residual"], t["weight"], 1e-6)
    check_grads(t, ds, dh, {"y": got.y, "residual": got.residual, "weight": got.weight}, 1e-6, 1.0)


def test_zero_rows_and_zero_values():
    w = torch.ones(16, device="cuda", requires_grad=True)
    y = torch.zeros(0, 16, device="cuda", requires_grad=True)
    s, h = norms.add_rms_norm(y, y, w, 1e-6)
    assert s.shape == (0, 16)
    (dw,) = torch.autograd.grad([s, h], [w], [s.detach(), h.detach()])
    assert torch.equal(dw, torch.zeros_like(dw))
    z = torch.zeros(3, 16, device="cuda")
    s, h = norms.add_rms_norm(z, z, w.detach(), 1e-6, post_weight=w.detach())
    assert torch.equal(s, z) and torch.equal(h, z)


def test_a_bad_row_stays_alone():
    t, ds, dh = make(6, 1280, "bf16")
    want = norms.add_rms_norm(t["y"], t["residual"], t["weight"], 1e-6)
    t["y"][2, 5], t["residual"][4, 7] = float("nan"), float("inf")
    got = norms.add_rms_norm(t["y"], t["residual"], t["weight"], 1e-6)
    for a, b in zip(got, want):
        for r in (0, 1, 3, 5):
            assert torch.equal(a[r], b[r])
    assert got[1][2].isnan().all() and got[0][2].isnan().sum() == 1


def test_streams_and_graphs():
    """A captured forward and backward call, replayed on new values, on a stream of its own."""
    t, ds, dh = make(33, 1280, "bf16", 3, True)
    run = lambda: (*norms.add_rms_norm(t["y"], t["residual"], t["weight"], 1e-6, gate=t["gate"], post_weight=t["post"]),  # noqa: E731
                   *norms.add_rms_norm_backward(ds, dh, t["y"], t["residual"], t["weight"], 1e-6, gate=t["gate"],
                                                post_weight=t["post"]))
    run()
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        out = run()
    for seed in (1, 2):
        n, ds2, dh2 = make(33, 1280, "bf16", 3, True, seed=seed)
        for a, b in ((t["y"], n["y"]), (t["residual"], n["residual"]), (ds, ds2), (dh, dh2)):
            a.copy_(b)
        g.replay()
        for a, b in zip(out, run()):
            assert torch.equal(a, b)


def test_refusals():
    t, ds, dh = make(4, 64, "bf16")
    y, res, w = t["y"], t["residual"], t["weight"]
    f = norms.add_rms_norm
    for bad in (lambda: f(y, res.float(), w, 1e-6), lambda: f(y, res[:3], w, 1e-6), lambda: f(y, res, w[:63], 1e-6),
                lambda: f(y, res, w.double(), 1e-6), lambda: f(y, res, w, 1e-6, gate=w[None].repeat(3, 1)),
                lambda: f(y, res, w, 1e-6, gate=w[None, None]), lambda: f(y.long(), res.long(), w, 1e-6),
                lambda: f(y, res, w, 1e-6, post_weight=w.half())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        f(y.cpu(), res.cpu(), w.cpu(), 1e-6)
    wide = torch.zeros(1, 8200, device="cuda")
    with pytest.raises(L.DashError, match="8192"):
        f(wide, wide, torch.ones(8200, device="cuda"), 1e-6)
