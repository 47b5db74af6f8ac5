"""The few-token mixture-of-experts layer against the definition in 64 bits: outputs within
a bound that is added up from the arithmetic (step_testutil.moe), picks equal, weights
within two roundings."""
import pytest
import torch

from ananta_ocr_b200 import _lib as L
from ananta_ocr_b200 import moe
from step_testutil import DT
from step_testutil import moe as definition

pytestmark = pytest.mark.gpu


def make(tokens, hidden, ffn, experts, shared=0, dt="bf16", gate="same", seed=0):
    g = torch.Generator().manual_seed(seed + tokens * 31 + hidden)
    d = DT[dt]
    rnd = lambda *s, std, dtype=d: (torch.randn(*s, generator=g) * std).to(dtype).cuda()  # noqa: E731
    t = dict(x=rnd(tokens, hidden, std=1.0), residual=rnd(tokens, hidden, std=1.0),
             gate=rnd(experts, hidden, std=hidden ** -0.5, dtype=torch.float32 if gate == "fp32" else d),
             gu=rnd(experts, 2 * ffn, hidden, std=hidden ** -0.5), down=rnd(experts, hidden, ffn, std=ffn ** -0.5), sgu=None, sd=None)
    if shared:
        t["sgu"], t["sd"] = rnd(2 * shared, hidden, std=hidden ** -0.5), rnd(hidden, shared, std=shared ** -0.5)
    return t, moe.MoeWeights(t["gate"], t["gu"], t["down"], t["sgu"], t["sd"])


def check(t, r, topk, renorm=False, scale=1.0, residual=True):
    up = {k: None if v is None else v.double().cpu() for k, v in t.items()}
    out, ids, w, tol = definition(up["x"], up["gate"], up["gu"], up["down"], up["sgu"], up["sd"], topk, renorm, scale,
                                  up["residual"] if residual else None, t["x"].dtype)
    assert torch.equal(r.ids.cpu(), ids)
    assert ((r.weights.double().cpu() - w).abs() <= w.abs() * 2.0 ** -23).all()
    off = (r.out.double().cpu() - out).abs()
    assert (off <= tol).all(), (off / tol).max()


CASES = [  # tokens, hidden, ffn, experts, topk, shared ffn
    (1, 8, 8, 1, 1, 0), (1, 256, 128, 8, 2, 128), (2, 64, 72, 8, 3, 8), (5, 200, 136, 7, 7, 0), (16, 256, 128, 8, 2, 256),
    (17, 1280, 896, 16, 6, 1792), (33, 136, 264, 40, 8, 40), (64, 320, 64, 64, 6, 64), (65, 72, 200, 3, 2, 0),
    (128, 128, 128, 256, 16, 0), (200, 72, 24, 5, 1, 16), (256, 64, 40, 9, 4, 24), (3, 4096, 16, 2, 1, 0), (4, 16, 4104, 2, 2, 8),
]


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("case", CASES)
def test_layer(case, dt):
    tokens, hidden, ffn, experts, topk, shared = case
    t, w = make(tokens, hidden, ffn, experts, shared, dt)
    check(t, moe.moe_layer(t["x"], w, topk, residual=t["residual"]), topk)


@pytest.mark.parametrize("tokens", [1, 9, 40])
def test_options(tokens):
    t, w = make(tokens, 264, 136, 12, 48, gate="fp32")
    check(t, moe.moe_layer(t["x"], w, 3, renormalize=True, scale=2.5), 3, True, 2.5, residual=False)
    check(t, moe.moe_layer(t["x"], w, 12, scale=-0.5, residual=t["residual"]), 12, False, -0.5)


def test_equal_scores_take_the_lowest_index():
    t, w = make(6, 64, 32, 10)
    t["gate"][3:8] = t["gate"][2]
    t["gate"][9] = 0
    t["gate"][0] = 0
    check(t, moe.moe_layer(t["x"], w, 4, residual=t["residual"]), 4)
    t["gate"].zero_()
    r = moe.moe_layer(t["x"], w, 4, residual=t["residual"])
    assert r.ids.tolist() == [[0, 1, 2, 3]] * 6
    check(t, r, 4)


def test_near_scores_are_told_apart():
    """Scores that differ by less than fp32 sums do: 2^-9 in 2^20, decided in 64 bits."""
    t, w = make(4, 512, 16, 6, gate="fp32")
    t["x"].fill_(1.0)
    t["gate"].zero_()
    t["gate"][:, 0] = 2.0 ** 20
    t["gate"][:, 1:100] = 1.0 + 2.0 ** -20
    t["gate"][4, 500] = 2.0 ** -9
    t["gate"][:, 501] = -2.0 ** 20
    t["gate"][2, 300] = 2.0 ** -10
    r = moe.moe_layer(t["x"], w, 3, residual=t["residual"])
    assert r.ids[:, :3].tolist() == [[4, 2, 0]] * 4
    check(t, r, 3)


def test_all_tokens_on_one_expert():
    t, w = make(256, 64, 72, 6)
    t["gate"].zero_()
    t["gate"][4, 0] = 8.0
    t["x"][:, 0] = 1.0 + torch.rand(256).cuda()
    r = moe.moe_layer(t["x"], w, 1, residual=t["residual"])
    assert (r.ids == 4).all()
    check(t, r, 1)


def test_rows_do_not_depend_on_the_others():
    """A row's output is that of the same row in another batch of the same size, bit for bit;
    a row of NaN or infinities stays alone."""
    t, w = make(24, 256, 136, 16, 64)
    a = moe.moe_layer(t["x"], w, 4, residual=t["residual"])
    x = t["x"].clone()
    x[5], x[6, 3] = float("nan"), float("inf")
    x[20:] = t["x"][:4]
    b = moe.moe_layer(x, w, 4, residual=t["residual"])
    rows = [i for i in range(20) if i not in (5, 6)]
    assert torch.equal(a.out[rows], b.out[rows]) and torch.equal(a.ids[rows], b.ids[rows])
    assert b.out[5].isnan().all()
    assert ((b.ids >= 0) & (b.ids < 16)).all()


def test_unpicked_experts_are_not_read():
    t, w = make(7, 128, 64, 32, 16)
    want = moe.moe_layer(t["x"], w, 2, residual=t["residual"])
    unused = torch.ones(32, dtype=torch.bool, device="cuda").scatter(0, want.ids.flatten().long(), False)
    t["gu"][unused], t["down"][unused] = float("nan"), float("inf")
    assert torch.equal(moe.moe_layer(t["x"], w, 2, residual=t["residual"]).out, want.out)


def test_strides_and_weights_in_place():
    t, w = make(9, 96, 40, 6, 8)
    want = moe.moe_layer(t["x"], w, 2, residual=t["residual"])
    wide = torch.zeros(9, 300, dtype=torch.bfloat16).cuda()
    for at in (0, 8, 5):
        x, res = wide[:, at:at + 96], wide[:, 150 + at:246 + at]
        x.copy_(t["x"]), res.copy_(t["residual"])
        assert torch.equal(moe.moe_layer(x, w, 2, residual=res).out, want.out)
    assert torch.equal(moe.moe_layer(t["x"].t().contiguous().t(), w, 2, residual=t["residual"]).out, want.out)
    t["gu"].mul_(0.5)
    check(t, moe.moe_layer(t["x"], w, 2, residual=t["residual"]), 2)


def test_two_runs_are_equal():
    t, w = make(40, 640, 320, 32, 320)
    a = moe.moe_layer(t["x"], w, 6, residual=t["residual"])
    for _ in range(3):
        assert torch.equal(moe.moe_layer(t["x"], w, 6, residual=t["residual"]).out, a.out)


def test_graphs_and_streams():
    """Two captured layers that share their weights, replayed at once on two streams."""
    t, w = make(8, 256, 136, 16, 64)
    run = lambda: moe.moe_layer(t["x"], w, 4, residual=t["residual"])  # noqa: E731
    run()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, run()))
    for seed in (1, 2):
        n, _ = make(8, 256, 136, 16, 64, seed=seed)
        t["x"].copy_(n["x"]), t["residual"].copy_(n["residual"])
        want = run()
        torch.cuda.synchronize()
        for g, _ in graphs:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    g.replay()
        torch.cuda.synchronize()
        for _, r in graphs:
            for a, b in zip(r, want):
                assert torch.equal(a, b)


def test_empty_and_refusals():
    t, w = make(4, 64, 32, 6, 8)
    r = moe.moe_layer(t["x"][:0], w, 2)
    assert r.out.shape == (0, 64) and r.ids.shape == (0, 2)
    with pytest.raises(NotImplementedError):
        moe.moe_layer(t["x"].clone().requires_grad_(), w, 2)
    with torch.no_grad():
        moe.moe_layer(t["x"].clone().requires_grad_(), w, 2)
    with pytest.raises(ValueError):
        moe.moe_layer(t["x"][:, :56], w, 2)
    with pytest.raises(ValueError):
        moe.moe_layer(t["x"].half(), w, 2)
    with pytest.raises(ValueError):
        moe.moe_layer(t["x"], w, 2, residual=t["residual"][:3])
    with pytest.raises(L.DashError, match="topk"):
        moe.moe_layer(t["x"], w, 7)
    with pytest.raises(L.DashError, match="256"):
        moe.moe_layer(torch.zeros(257, 64, dtype=torch.bfloat16, device="cuda"), w, 2)
    with pytest.raises(ValueError):
        moe.MoeWeights(t["gate"], t["gu"], t["down"].transpose(1, 2))
    with pytest.raises(ValueError):
        moe.MoeWeights(t["gate"], t["gu"].float(), t["down"].float())
    with pytest.raises(ValueError):
        moe.MoeWeights(t["gate"], t["gu"], t["down"], t["sgu"])
    odd, ow = make(4, 60, 32, 6)
    with pytest.raises(L.DashError, match="multiples of 8"):
        moe.moe_layer(odd["x"], ow, 2)
