"""Tokens and distributions against the definition in 64 bits.  The weights are exact
to 2^-43 of the largest, so tokens are equal unless a border lies within some 10^-11 of the
random number; the inputs here have none but exact ones, which are decided alike."""
import numpy as np
import pytest
import torch

from ananta_ocr_b200 import drafts, sampling
from step_testutil import DT, distribution, draw, kept

pytestmark = pytest.mark.gpu

SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (0.8, 0, 0.9, 0.0), (1.3, 0, 1.0, 0.03), (0.9, 40, 0.8, 0.01), (0.0, 5, 0.5, 0.1),
            (1.0, 1, 0.3, 0.0), (2.0, 1000000, 0.999, 0.0), (0.6, 7, 0.0, 0.0), (1.0, 3, 0.7, 1.0), (50.0, 0, 0.5, 0.0)]


def logits_of(rows, vocab, dt, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(rows, vocab, generator=g) * spread
    return z.to(DT[dt]), torch.rand(rows, generator=g)


def same(z, u, settings, **kw):
    """Token and distribution of every row; settings: one per row."""
    z64 = z.double().cpu().numpy()
    got = sampling.sample(z, u, **kw).cpu().numpy()
    p = sampling.probs(z, **kw).double().cpu().numpy()
    f32 = lambda v: float(np.float32(v))  # noqa: E731
    for i, s in enumerate(settings):
        s = (f32(s[0]), s[1], f32(s[2]), f32(s[3]))
        want = distribution(z64[i], *s)
        assert (want > 0).sum() - (p[i] > 0).sum() in range(0, 1 + int((want < 1e-12).sum() - (want == 0).sum())), (i, s)
        # a probability is rounded once; its weight and the sum are off by 2^-43 of the largest weight each
        np.testing.assert_allclose(p[i], want, rtol=2.0 ** -23, atol=2.0 ** -40, err_msg=str((i, s)))
        assert got[i] == draw(z64[i], float(u[i]), *s), (i, s)


def columns(settings):
    t, k, p, m = zip(*settings)
    f = lambda v: torch.tensor(v, dtype=torch.float32, device="cuda")  # noqa: E731
    return dict(temperature=f(t), top_k=torch.tensor(k, dtype=torch.int32, device="cuda"), top_p=f(p), min_p=f(m))


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("vocab", [1, 2, 31, 1003, 4096, 50257])
def test_every_setting(vocab, dt):
    z, u = logits_of(len(SETTINGS), vocab, dt, vocab)
    same(z.cuda(), u.cuda(), SETTINGS, **columns(SETTINGS))


@pytest.mark.parametrize("setting", SETTINGS)
def test_one_setting_for_all_rows(setting):
    z, u = logits_of(5, 777, "fp32", 3)
    t, k, p, m = setting
    same(z.cuda(), u.cuda(), [setting] * 5, temperature=t, top_k=k, top_p=p, min_p=m)


@pytest.mark.parametrize("vocab,dt", [(129280, "bf16"), (129280, "fp32"), (1 << 20, "fp32"), (1 << 20, "bf16"), (300001, "fp32")])
def test_large_vocabularies(vocab, dt):
    """Up to the largest, whose slices do not fit shared memory."""
    settings = SETTINGS[:6]
    z, u = logits_of(len(settings), vocab, dt, 11, spread=2.0)
    same(z.cuda(), u.cuda(), settings, **columns(settings))


def test_flat_rows():
    """Equal logits: every border is exact, and the lowest indices are kept."""
    V = 1000
    z = torch.zeros(8, V)
    z[1], z[2], z[3] = -3.4028234663852886e38, 5.0, -0.0
    z[3, ::2] = 0.0
    z[4] = float("inf")
    u = torch.tensor([0.0, 0.25, 0.5, 0.999, 0.1, 0.7, 0.3, 0.99999994])
    for setting in ((1.0, 0, 1.0, 0.0), (1.0, 10, 1.0, 0.0), (1.0, 0, 0.5, 0.0), (0.5, 300, 0.1, 0.0), (1.0, 0, 1.0, 1.0)):
        t, k, p, m = setting
        same(z.cuda(), u.cuda(), [setting] * 8, temperature=t, top_k=k, top_p=p, min_p=m)
    assert sampling.sample(z.cuda(), u.cuda()).tolist() == [int(x * V) for x in u.tolist()]


def test_ties_across_slices():
    """A few values only, over a whole vocabulary: the cutoff splits thousands of equal ones."""
    g = torch.Generator().manual_seed(2)
    z = torch.randint(0, 4, (6, 60000), generator=g).float()
    u = torch.rand(6, generator=g)
    settings = [(1.0, 17000, 1.0, 0.0), (1.0, 0, 0.55, 0.0), (1.0, 40001, 0.77, 0.0), (0.5, 1, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 2, 0.6, 0.0)]
    same(z.bfloat16().cuda(), u.cuda(), settings, **columns(settings))


def test_masks_and_odd_values():
    """Rows with nothing, one token, masks of -inf or of the type's lowest value, NaN."""
    V, inf, nan = 5000, float("inf"), float("nan")
    for dt in DT:
        z, u = logits_of(7, V, dt, 5)
        low = torch.finfo(DT[dt]).min
        z[0] = -inf
        z[1] = -inf
        z[1, 4321] = -7.0
        z[2, 100:] = low
        z[3, ::3] = nan
        z[4] = nan
        z[5, :4990] = -inf
        z[6, 17] = inf
        settings = [(0.8, 30, 0.9, 0.01)] * 7
        same(z.cuda(), u.cuda(), settings, temperature=0.8, top_k=30, top_p=0.9, min_p=0.01)
        same(z.cuda(), u.cuda(), [(1.0, 0, 1.0, 0.0)] * 7)
        same(z.cuda(), u.cuda(), [(0.0, 0, 1.0, 0.0)] * 7, temperature=0.0)
        tok = sampling.sample(z.cuda(), u.cuda()).tolist()
        assert tok[0] == tok[4] == -1 and tok[1] == 4321 and tok[6] == 17


def test_random_numbers_at_the_borders():
    """u = running sum / total exactly: the next token, as the sum has to exceed it."""
    z = torch.tensor([[0.0] * 4 + [float("-inf")] + [0.0] * 4]).repeat(8, 1)
    u = torch.arange(8).float() / 8
    assert sampling.sample(z.cuda(), u.cuda()).tolist() == [0, 1, 2, 3, 5, 6, 7, 8]


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_strides_and_offsets(dt):
    z, u = logits_of(6, 2051, dt, 8)
    big = torch.full((6, 3, 2100), 9.0, dtype=DT[dt]).cuda()
    for view in (big[:, 1, 3:2054], big[:, 0, 16:2067], big.transpose(1, 2)[:, 5:2056, 2]):
        view.copy_(z)
        s = (0.9, 100, 0.9, 0.0)
        same(view, u.cuda(), [s] * 6, temperature=0.9, top_k=100, top_p=0.9)
        same(view[1:2], u[1:2].cuda(), [s], temperature=0.9, top_k=100, top_p=0.9)
    same(z.cuda(), torch.stack([u, u], 1).cuda()[:, 0], [(1.0, 0, 1.0, 0.0)] * 6)


def test_the_distribution_is_sampled():
    """Tokens of 4,096 evenly spread numbers have the distribution's counts (each
    within one, as the numbers are 1 / 4096 apart)."""
    z, _ = logits_of(1, 300, "fp32", 1)
    n = 4096
    u = (torch.arange(n).float() + 0.5) / n
    kw = dict(temperature=1.2, top_k=40, top_p=0.95)
    tok = sampling.sample(z.cuda().expand(n, 300), u.cuda(), **kw)
    p = sampling.probs(z.cuda(), **kw)[0].double().cpu()
    count = torch.bincount(tok.cpu(), minlength=300).double()
    assert ((count - p * n).abs() <= 1 + 1e-3).all()


def test_targets_of_the_verification():
    """probs of a filtered row is a target of verify_drafts: a draft that was cut off is never kept."""
    z, _ = logits_of(4, 500, "fp32", 4)
    target = sampling.probs(z.cuda(), temperature=0.9, top_k=10)
    cut = (target[0] == 0).nonzero()[0]
    best = z[2].argmax().item()
    tokens = torch.tensor([1, int(cut), 1, best]).cuda()
    cu = torch.tensor([0, 2, 4], dtype=torch.int32).cuda()
    kept_ = drafts.verify_drafts(tokens, None, cu, target, max_nodes=2, u_accept=torch.zeros(4).cuda(),
                                 u_sample=torch.tensor([0.5, 0.5]).cuda())
    assert kept_.n_accept.tolist() == [0, 1]
    assert target[0, kept_.next_token[0]] > 0 and target[3, kept_.next_token[1]] > 0


def test_graph_and_streams():
    z, u = (t.cuda() for t in logits_of(9, 4099, "bf16", 6))
    kw = columns([SETTINGS[i % len(SETTINGS)] for i in range(9)])
    run = lambda: (sampling.sample(z, u, **kw), sampling.probs(z, **kw))  # noqa: E731
    run()
    torch.cuda.synchronize()
    g, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=st):
        out = run()
    for seed in (7, 8):
        z2, u2 = logits_of(9, 4099, "bf16", seed)
        z.copy_(z2), u.copy_(u2)
        g.replay()
        for a, b in zip(out, run()):
            assert torch.equal(a, b)
    # several calls at once on streams of their own
    torch.cuda.synchronize()
    want, got = run(), []
    for _ in range(4):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            got.append(run())
    torch.cuda.synchronize()
    for r in got:
        for a, b in zip(r, want):
            assert torch.equal(a, b)


def test_empty_and_refusals():
    z, u = (t.cuda() for t in logits_of(3, 10, "fp32", 1))
    assert sampling.sample(z[:0], u[:0]).shape == (0,) and sampling.probs(z[:0]).shape == (0, 10)
    for bad in (lambda: sampling.sample(z, u[:2]), lambda: sampling.sample(z, u.double()), lambda: sampling.sample(z[0], u),
                lambda: sampling.sample(z.double(), u), lambda: sampling.sample(z, u, temperature=u[:2]),
                lambda: sampling.sample(z, u, top_p=u.half()), lambda: sampling.probs(z, top_k=u)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        sampling.probs(z.cpu())
    with pytest.raises(NotImplementedError):
        sampling.probs(z.clone().requires_grad_())
    assert sampling.sample(z.clone().requires_grad_(), u).shape == (3,)
    assert len(kept(z[0].double().cpu().numpy(), 1.0, 3, 1.0, 0.0)[0]) == 3
