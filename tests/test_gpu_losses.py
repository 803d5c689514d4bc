"""The loss operators on the GPU against their definitions in 64 bits.

Tolerances (relative in the 2-norm, fixed before the first run):

* 16-bit gradients carry two roundings to the type (dZ, then the result), each
  at most u = 2^-9 (bf16) or 2^-12 (fp16's half ulp is 2^-12 of a value in
  [1, 2); its unit roundoff 2^-11) of a value; sums of both signs keep that
  relation on average and not for each value, so four times the sum of both is
  allowed: 2^-6 for bf16 (8 u), 2^-8 for fp16.
* fp32 gradients come from tf32 pairs (2^-21 of each product) summed in fp32
  over up to thousands of terms: 2^-17.
* Losses are differences of numbers up to the largest logit in size: per row
  2^-19 of (1 + max |z|) for fp32 operands and for 16-bit ones alike (their
  products are exact in fp32), logits themselves being sums of D products in
  fp32, whose rounding grows with sum |h w|: 2^-21 of that is added.
"""

import math

import pytest
import torch

from pytorch_opt_b200 import _lib, losses

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
GRAD_TOL = {torch.bfloat16: 2.0**-6, torch.float16: 2.0**-8, torch.float32: 2.0**-17}


@pytest.fixture(autouse=True)
def _no_device_error(cuda):
    yield
    assert _lib.device_error(reset=True) == 0


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _head(T, D, V, dtype, seed=0, scale=1.0):
    g = _gen(seed)
    h = (scale * torch.randn(T, D, generator=g, device="cuda")).to(dtype)
    w = (torch.randn(V, D, generator=g, device="cuda") / math.sqrt(D)).to(dtype)
    y = torch.randint(0, V, (T,), generator=g, device="cuda")
    return h, w, y


def _loss_bound(h, w, temperature=1.0):
    """Per row: what the loss may be off by (see the head of this file)."""
    h, w = h.double(), w.double()
    z = (h @ w.t()).abs().amax(1)
    s = (h.abs() @ w.abs().t()).amax(1)
    return temperature * (2.0**-19 * (1 + z) + 2.0**-21 * s)


def _rel(got, want):
    got, want = got.double(), want.double()
    return float((got - want).norm() / want.norm().clamp_min(1e-300))


def ref_ce(h, w, y, smoothing=0.0, z_loss=0.0, ignore=-100, up=None):
    """(row losses, dH, dW) of sum_t up_t l_t in 64 bits, from log-probabilities."""
    counts = y != ignore
    h64, w64 = torch.where(counts[:, None], h.double(), 0.0), w.double()
    z = h64 @ w64.t()
    V = z.shape[1]
    lse = torch.logsumexp(z, 1)
    logp = z - lse[:, None]
    goal = torch.zeros_like(z)
    goal.scatter_(1, y.clamp(0, V - 1)[:, None], 1 - smoothing)
    goal += smoothing / V
    rows = torch.where(counts, -(goal * logp).sum(1) + z_loss * lse**2, 0.0)
    dz = (1 + 2 * z_loss * lse[:, None]) * logp.exp() - goal
    dz *= (counts.double() * (1.0 if up is None else up.double()))[:, None]
    return rows, dz @ w64, dz.t() @ h64


def ref_distill(z, index, teacher, a, up=None):
    """(row losses, dz) in 64 bits."""
    there = index >= 0
    t = torch.where(there, teacher.double() / a, -math.inf)
    counts = (t > -math.inf).any(1)
    t = torch.where(counts[:, None], t, 0.0)
    t = t - t.amax(1, keepdim=True)  # equal entries of any size: their logarithms would not show beside 1e38
    logq = t - torch.logsumexp(t, 1, keepdim=True)
    q = torch.where(counts[:, None], logq.exp(), 0.0)
    z = torch.where(counts[:, None], z.double(), 0.0)
    top = z.amax(1, keepdim=True)
    z = torch.where(top > -math.inf, z - top, z)  # as above: a row of the lowest value, 64 bits or not
    logp = (z / a) - torch.logsumexp(z / a, 1, keepdim=True)
    at = index.clamp(min=0)
    each = torch.where(q > 0, q * (logq - logp.gather(1, at)), 0.0)
    rows = a * a * each.sum(1)
    goal = torch.zeros_like(z).scatter_add_(1, at, q)
    dz = a * (logp.exp() - goal) * counts[:, None]
    if up is not None:
        dz = dz * up.double()[:, None]
    return rows, dz, counts


def _grads(loss, *inputs, up=None):
    return torch.autograd.grad(loss, inputs, up)


# ------------------------------------------------------- linear cross entropy
SIZES = [(1, 8, 1), (1, 64, 5000), (2, 1, 3), (3, 77, 33), (127, 64, 128), (128, 128, 129), (255, 64, 257),
         (257, 200, 1000), (300, 136, 513), (131, 1000, 2049), (513, 256, 255), (5, 320, 20011)]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("T,D,V", SIZES)
def test_linear_cross_entropy_rows_and_mean(T, D, V, dtype):
    h, w, y = _head(T, D, V, DTYPES[dtype], seed=T + D + V, scale=3.0)
    if T > 3:
        y[torch.rand(T, generator=_gen(1), device="cuda") < 0.3] = -100
        y[0] = 0
    want, dh, dw = ref_ce(h, w, y)
    n = int((y != -100).sum())
    rows = losses.linear_cross_entropy(h, w, y, reduction="none")
    assert rows.dtype == torch.float32 and rows.shape == (T,)
    assert ((rows - want).abs() <= _loss_bound(h, w)).all()
    assert (rows[y == -100] == 0).all()
    h.requires_grad_(), w.requires_grad_()
    loss = losses.linear_cross_entropy(h, w, y)
    assert abs(float(loss) - float(want.sum() / n)) <= float(_loss_bound(h.detach(), w.detach()).max())
    gh, gw = _grads(loss, h, w)
    assert gh.dtype == h.dtype and gw.dtype == w.dtype
    if V > 1:
        assert _rel(gh, dh / n) <= GRAD_TOL[h.dtype]
        assert _rel(gw, dw / n) <= GRAD_TOL[h.dtype]
    else:  # one class: probability 1 and nothing to learn
        assert float(gh.abs().max()) <= 1e-5 and float(gw.abs().max()) <= 1e-5
    assert (gh[y == -100] == 0).all()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("reduction", ["sum", "none"])
@pytest.mark.parametrize("smoothing,z_loss", [(0.0, 0.0), (0.1, 1e-3), (1.0, 0.0)])
def test_linear_cross_entropy_terms_and_upstream(dtype, reduction, smoothing, z_loss):
    T, D, V = 201, 96, 777
    h, w, y = _head(T, D, V, DTYPES[dtype], seed=7, scale=2.0)
    y[::5] = 3  # a value of its own as ignore_index
    up = torch.randn(T, generator=_gen(3), device="cuda") * 1e-3 if reduction == "none" else torch.full((T,), 0.37, device="cuda")
    want, dh, dw = ref_ce(h, w, y, smoothing, z_loss, 3, up)
    h.requires_grad_(), w.requires_grad_()
    loss = losses.linear_cross_entropy(h, w, y, ignore_index=3, label_smoothing=smoothing, z_loss=z_loss,
                                       reduction=reduction)
    bound = _loss_bound(h.detach(), w.detach()) * 4  # z_loss lse^2 adds a few roundings of numbers below 100
    if reduction == "none":
        assert ((loss - want).abs() <= bound).all()
        gh, gw = _grads(loss, h, w, up=up)
    else:
        assert abs(float(loss) - float(want.sum())) <= float(bound.sum())
        gh, gw = _grads(loss, h, w, up=torch.tensor(0.37, device="cuda"))
    tol = GRAD_TOL[h.dtype] * (1 if reduction == "none" else 1.5)  # the upstream scalar rounds once more
    assert _rel(gh, dh) <= tol
    assert _rel(gw, dw) <= tol


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_linear_cross_entropy_chunks_of_rows(dtype):
    T, D, V = 900, 200, 300
    h, w, y = _head(T, D, V, DTYPES[dtype], seed=11, scale=2.0)
    y[torch.rand(T, generator=_gen(2), device="cuda") < 0.5] = -100  # the later chunks hold few rows or none
    want, dh, dw = ref_ce(h, w, y)
    n = int((y != -100).sum())
    h.requires_grad_(), w.requires_grad_()
    for chunk in (256, 512, 0):
        loss = losses.linear_cross_entropy(h, w, y, chunk_rows=chunk)
        gh, gw = _grads(loss, h, w)
        assert abs(float(loss) - float(want.sum() / n)) <= float(_loss_bound(h.detach(), w.detach()).max())
        assert _rel(gh, dh / n) <= GRAD_TOL[h.dtype]
        assert _rel(gw, dw / n) <= GRAD_TOL[h.dtype]


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_linear_cross_entropy_few_tiles_split_their_long_axis(dtype):
    # dH: one tile of rows over a long vocabulary; dW: one tile of the vocabulary over many rows.
    for T, D, V in ((9, 64, 30011), (5003, 64, 65)):
        h, w, y = _head(T, D, V, DTYPES[dtype], seed=T, scale=2.0)
        y[1] = -100
        want, dh, dw = ref_ce(h, w, y)
        n = T - 1
        h.requires_grad_(), w.requires_grad_()
        gh, gw = _grads(losses.linear_cross_entropy(h, w, y), h, w)
        assert _rel(gh, dh / n) <= GRAD_TOL[h.dtype]
        assert _rel(gw, dw / n) <= GRAD_TOL[h.dtype]


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_linear_cross_entropy_nothing_counts(dtype):
    h, w, y = _head(70, 64, 100, DTYPES[dtype])
    y.fill_(-100)
    h.fill_(math.nan)
    h.requires_grad_(), w.requires_grad_()
    for reduction in ("mean", "sum"):
        loss = losses.linear_cross_entropy(h, w, y, reduction=reduction)
        gh, gw = _grads(loss, h, w)
        assert float(loss) == 0.0 and (gh == 0).all() and (gw == 0).all()
    rows = losses.linear_cross_entropy(h, w, y, reduction="none")
    gh, gw = _grads(rows, h, w, up=torch.ones_like(rows))
    assert (rows == 0).all() and (gh == 0).all() and (gw == 0).all()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("counted", [1, 200, 257, 1100])
def test_linear_cross_entropy_few_of_many_rows_count(dtype, counted):
    # How dH's long axis is split goes by the rows that count, on the device.
    T, D, V = 1100, 264, 6001
    h, w, y = _head(T, D, V, DTYPES[dtype], seed=counted)
    drop = torch.randperm(T, generator=_gen(2), device="cuda")[counted:]
    y[drop] = -100
    want, dh, dw = ref_ce(h, w, y)
    h.requires_grad_(), w.requires_grad_()
    loss = losses.linear_cross_entropy(h, w, y, reduction="sum")
    assert abs(float(loss.detach() - want.sum())) <= float(_loss_bound(h.detach(), w.detach())[y != -100].sum())
    gh, gw = _grads(loss, h, w)
    assert _rel(gh, dh) < GRAD_TOL[DTYPES[dtype]] and _rel(gw, dw) < GRAD_TOL[DTYPES[dtype]]
    assert (gh[drop] == 0).all()


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_linear_cross_entropy_masked_rows_hold_anything(dtype):
    T, D, V = 140, 72, 300
    h, w, y = _head(T, D, V, DTYPES[dtype], seed=5)
    y[10:40] = -100
    h[10:25] = math.nan
    h[25:40] = math.inf
    want, dh, dw = ref_ce(h, w, y)
    n = T - 30
    h.requires_grad_(), w.requires_grad_()
    loss = losses.linear_cross_entropy(h, w, y)
    gh, gw = _grads(loss, h, w)
    assert math.isclose(float(loss), float(want.sum() / n), rel_tol=1e-4)
    assert (gh[10:40] == 0).all()
    assert _rel(gh, dh / n) <= GRAD_TOL[h.dtype]
    assert _rel(gw, dw / n) <= GRAD_TOL[h.dtype]


def test_linear_cross_entropy_bad_targets_are_loud_and_contained():
    h, w, y = _head(64, 64, 100, torch.bfloat16, seed=6)
    y[3], y[60] = 100, -5
    rows = losses.linear_cross_entropy(h, w, y, reduction="none")
    bad = torch.zeros(64, dtype=torch.bool, device="cuda")
    bad[3] = bad[60] = True
    assert torch.isnan(rows[bad]).all() and torch.isfinite(rows[~bad]).all()
    h.requires_grad_(), w.requires_grad_()
    loss = losses.linear_cross_entropy(h, w, y)
    gh, gw = _grads(loss, h, w)
    assert math.isnan(float(loss))
    assert (gh[bad] == 0).all() and torch.isfinite(gh).all() and torch.isfinite(gw).all()
    h2, y2 = h.detach()[~bad], y[~bad]
    _, dh, dw = ref_ce(h2, w.detach(), y2)
    assert _rel(gw, dw / 64) <= GRAD_TOL[h.dtype]


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_linear_cross_entropy_large_logits(dtype):
    """Confident and wrong rows: logits of hundreds, probabilities that underflow."""
    T, D, V = 64, 64, 500
    h, w, y = _head(T, D, V, DTYPES[dtype], seed=8, scale=100.0)
    want, dh, dw = ref_ce(h, w, y)
    h.requires_grad_(), w.requires_grad_()
    rows = losses.linear_cross_entropy(h, w, y, reduction="none")
    assert ((rows - want).abs() <= _loss_bound(h.detach(), w.detach())).all()
    gh, gw = _grads(losses.linear_cross_entropy(h, w, y, reduction="sum"), h, w)
    # Softmax of logits that carry an error d has one of d: 2^-19 of 400 more than elsewhere.
    assert _rel(gh, dh) <= GRAD_TOL[h.dtype] + 2.0**-10
    assert _rel(gw, dw) <= GRAD_TOL[h.dtype] + 2.0**-10


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_linear_cross_entropy_strides_and_offsets(dtype):
    dt = DTYPES[dtype]
    B, S, D, V = 3, 41, 64, 211
    g = _gen(12)
    big_h = torch.randn(B, S, D + 3, generator=g, device="cuda").to(dt)
    big_w = torch.randn(V + 1, D + 5, generator=g, device="cuda").to(dt)
    h, w = big_h[..., 1:D + 1], big_w[1:, 3:D + 3]  # odd pitches, odd starts
    y = torch.randint(0, V, (S, B), generator=g, device="cuda").t()
    want, dh, dw = ref_ce(h.reshape(-1, D), w, y.reshape(-1))
    got = losses.linear_cross_entropy(h, w, y.int(), reduction="none")
    assert got.shape == (B, S)
    assert ((got.reshape(-1) - want).abs() <= _loss_bound(h.reshape(-1, D), w)).all()
    big_h.requires_grad_(), big_w.requires_grad_()
    loss = losses.linear_cross_entropy(big_h[..., 1:D + 1], big_w[1:, 3:D + 3], y)
    gh, gw = _grads(loss, big_h, big_w)
    assert _rel(gh[..., 1:D + 1].reshape(-1, D), dh / (B * S)) <= GRAD_TOL[dt]
    assert _rel(gw[1:, 3:D + 3], dw / (B * S)) <= GRAD_TOL[dt]
    # transposed storage: no row is contiguous
    ht = h.detach().reshape(-1, D).t().contiguous().t()
    wt = w.detach().t().contiguous().t()
    got = losses.linear_cross_entropy(ht, wt, y.reshape(-1), reduction="none")
    assert ((got - want).abs() <= _loss_bound(h.reshape(-1, D), w)).all()
    # one hidden state for all tokens (stride 0), gradient summed over its uses
    one = h.detach().reshape(-1, D)[:1].clone().requires_grad_()
    loss = losses.linear_cross_entropy(one.expand(B * S, D), w.detach(), y.reshape(-1), reduction="sum")
    _, dh1, _ = ref_ce(one.detach().expand(B * S, D), w, y.reshape(-1))
    assert _rel(_grads(loss, one)[0], dh1.sum(0, keepdim=True)) <= 2 * GRAD_TOL[dt]


def test_linear_cross_entropy_one_gradient_alone():
    h, w, y = _head(50, 64, 300, torch.bfloat16, seed=13)
    _, dh, dw = ref_ce(h, w, y)
    a = h.clone().requires_grad_()
    assert _rel(_grads(losses.linear_cross_entropy(a, w, y, reduction="sum"), a)[0], dh) <= GRAD_TOL[h.dtype]
    b = w.clone().requires_grad_()
    assert _rel(_grads(losses.linear_cross_entropy(h, b, y, reduction="sum"), b)[0], dw) <= GRAD_TOL[h.dtype]
    rows = losses.linear_cross_entropy(h, b, y, reduction="none")
    assert _rel(_grads(rows, b, up=torch.ones_like(rows))[0], dw) <= GRAD_TOL[h.dtype]


def test_linear_cross_entropy_backward_runs_once_per_loss():
    h, w, y = _head(20, 64, 300, torch.bfloat16, seed=14)
    h.requires_grad_()
    loss = losses.linear_cross_entropy(h, w, y)
    loss.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="one backward pass"):
        loss.backward()


def test_losses_differentiate_once():
    """A graph of the gradient may be asked for; going through it a second time is refused."""
    h, w, y = _head(20, 64, 300, torch.float32, seed=14)
    index, teacher = y[:, None], torch.zeros(20, 1, device="cuda")
    for reduction in ("mean", "none"):
        for call in (lambda a: losses.linear_cross_entropy(a, w, y, reduction=reduction),
                     lambda a: losses.distillation(a, index, teacher, reduction=reduction)):
            a = h.clone().requires_grad_()
            loss = call(a).sum()
            g, = torch.autograd.grad(loss, a, create_graph=True)
            b = h.clone().requires_grad_()
            assert torch.equal(g.detach(), torch.autograd.grad(call(b).sum(), b)[0])
            with pytest.raises(RuntimeError):
                g.sum().backward()


@pytest.mark.parametrize("fn", ["ce", "distil"])
def test_gradient_agrees_with_differences(fn):
    """(l(h + e d) - l(h - e d)) / 2e along random directions, fp32: e = 2^-6 leaves a term of e^2 |d|^3 of third
    derivatives (each below 1/2 for softmax, |W d| ~ 1) and the losses' rounding over e: 2^-8 of the largest."""
    T, D, V = 37, 48, 401
    h, w, y = _head(T, D, V, torch.float32, seed=15, scale=2.0)
    index = torch.randint(0, V, (T, 5), generator=_gen(4), device="cuda")
    teacher = torch.randn(T, 5, generator=_gen(5), device="cuda")
    call = {"ce": lambda a, b: losses.linear_cross_entropy(a, b, y, label_smoothing=0.1, z_loss=1e-3, reduction="none"),
            "distil": lambda a, b: losses.linear_distillation(a, b, index, teacher, temperature=1.5,
                                                             reduction="none")}[fn]
    e = 2.0**-6
    d = torch.randn(T, D, generator=_gen(6), device="cuda")
    hg, wg = h.clone().requires_grad_(), w.clone().requires_grad_()
    rows = call(hg, wg)
    gh, gw = _grads(rows, hg, wg, up=torch.ones_like(rows))
    diff = (call(h + e * d, w) - call(h - e * d, w)).double() / (2 * e)
    want = (gh.double() * d.double()).sum(1)
    assert float((diff - want).abs().max()) <= 2.0**-8 * float(want.abs().max().clamp_min(1))
    dwd = torch.randn(V, D, generator=_gen(7), device="cuda") / math.sqrt(D)
    diff = (call(h, w + e * dwd) - call(h, w - e * dwd)).double().sum() / (2 * e)
    want = (gw.double() * dwd.double()).sum()
    assert abs(float(diff - want)) <= 2.0**-8 * max(1.0, abs(float(want)), T)


def test_linear_cross_entropy_on_a_side_stream_is_ordered():
    h, w, y = _head(300, 256, 4000, torch.bfloat16, seed=16)
    want, dh, dw = ref_ce(h, w, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
        loss = losses.linear_cross_entropy(a, b, y)
        gh, gw = _grads(loss, a, b)
    torch.cuda.current_stream().wait_stream(side)
    assert _rel(gh, dh / 300) <= GRAD_TOL[h.dtype] and _rel(gw, dw / 300) <= GRAD_TOL[h.dtype]


def test_losses_repeat_to_the_bit():
    h, w, y = _head(700, 192, 5001, torch.bfloat16, seed=17)
    y[::3] = -100
    outs = []
    for _ in range(3):
        a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
        loss = losses.linear_cross_entropy(a, b, y)
        outs.append((loss.detach(), *_grads(loss, a, b)))
    for o in outs[1:]:
        assert all(torch.equal(x, z) for x, z in zip(o, outs[0]))


def test_linear_cross_entropy_under_graph_capture():
    h, w, y = _head(100, 128, 1000, torch.bfloat16, seed=18)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        losses.linear_cross_entropy(h, w, y, reduction="none")
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        rows = losses.linear_cross_entropy(h, w, y, reduction="none")
    h2, _, y2 = _head(100, 128, 1000, torch.bfloat16, seed=19)
    y2[4] = -100
    h.copy_(h2), y.copy_(y2)
    g.replay()
    want, _, _ = ref_ce(h, w, y)
    assert ((rows - want).abs() <= _loss_bound(h, w)).all()


def test_linear_cross_entropy_empty():
    w = torch.randn(10, 8, device="cuda").requires_grad_()
    h = torch.empty(0, 8, device="cuda").requires_grad_()
    y = torch.empty(0, dtype=torch.long, device="cuda")
    assert losses.linear_cross_entropy(h, w, y, reduction="none").shape == (0,)
    loss = losses.linear_cross_entropy(h, w, y)
    gh, gw = _grads(loss, h, w)
    assert float(loss) == 0.0 and gh.shape == (0, 8) and (gw == 0).all()


def test_losses_refuse(cuda):
    h, w, y = _head(4, 8, 16, torch.bfloat16)
    i, t = torch.zeros(4, 2, dtype=torch.long, device=cuda), torch.zeros(4, 2, device=cuda)
    for bad, word in [((h, w.float(), y), "both be"), ((h.double(), w.double(), y), "both be"),
                      ((h, w[:, :7], y), "expects hidden"), ((h, w, y[:3]), "target"), ((h, w, y.float()), "target"),
                      ((h, w[:0], y), "expects hidden"), ((h, w, y.cpu()), "CUDA tensors only")]:
        with pytest.raises(RuntimeError, match=word):
            losses.linear_cross_entropy(*bad)
    for kw, word in [(dict(reduction="avg"), "reduction"), (dict(label_smoothing=1.1), "label_smoothing"),
                     (dict(z_loss=math.nan), "z_loss"), (dict(chunk_rows=-1), "chunk_rows")]:
        with pytest.raises(RuntimeError, match=word):
            losses.linear_cross_entropy(h, w, y, **kw)
    for fn, first in ((losses.linear_distillation, (h, w)), (losses.distillation, (torch.randn(4, 16, device=cuda),))):
        for bad, word in [((i.float(), t), "teacher_index"), ((i, t.double()), "teacher_logits"), ((i[:3], t[:3]), "top"),
                          ((i, t[:, :1]), "top"), ((i[:, :0], t[:, :0]), "entries"),
                          ((i.new_zeros(4, 1025), t.new_zeros(4, 1025)), "entries")]:
            with pytest.raises(RuntimeError, match=word):
                fn(*first, *bad)
        for a in (0.0, -1.0, math.nan, math.inf):
            with pytest.raises(RuntimeError, match="temperature"):
                fn(*first, i, t, temperature=a)
        with pytest.raises(RuntimeError, match="reduction"):
            fn(*first, i, t, reduction="batchmean")
    with pytest.raises(RuntimeError, match="logits must be"):
        losses.distillation(torch.randn(4, 16, device=cuda).double(), i, t)


# --------------------------------------------------------------- distillation
def _teacher(T, V, K, seed, dtype=torch.float32, holes=True):
    g = _gen(seed)
    index = torch.stack([torch.randperm(V, generator=g, device="cuda")[:K] for _ in range(T)])
    teacher = (3 * torch.randn(T, K, generator=g, device="cuda")).to(dtype)
    if holes and T > 4:
        gone = torch.rand(T, K, generator=g, device="cuda") < 0.3
        gone[1] = True   # a row with no entry
        gone[2] = False  # a full one
        index[gone] = -1
        teacher[gone] = math.nan
    return index, teacher


DSIZES = [(1, 1, 1), (1, 50257, 16), (2, 7, 7), (3, 4099, 1), (40, 1000, 64), (33, 33333, 130), (9, 130001, 1000),
          (300, 255, 3)]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("T,V,K", DSIZES)
def test_distillation_of_logits(T, V, K, dtype):
    dt = DTYPES[dtype]
    g = _gen(T + V)
    z = (3 * torch.randn(T, V, generator=g, device="cuda")).to(dt)
    index, teacher = _teacher(T, V, K, K, torch.float32 if dtype == "fp32" else dt)
    for a in (1.0, 2.5):
        want, dz, counts = ref_distill(z, index, teacher, a)
        rows = losses.distillation(z, index, teacher, temperature=a, reduction="none")
        # Sums of at most 1024 terms and logarithms in fp32 of numbers below 32, times a^2.
        assert ((rows - want).abs() <= a * a * 2.0**-17).all()
        assert (rows[~counts] == 0).all()
        x = z.clone().requires_grad_()
        n = int(counts.sum())
        loss = losses.distillation(x, index, teacher, temperature=a)
        assert abs(float(loss) - float(want.sum()) / max(n, 1)) <= a * a * 2.0**-17
        got, = _grads(loss, x)
        u = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-17}[dt]
        if V > 1:
            floor = 2.0**-24 if dt == torch.float16 else 0.0  # fp16 gradients of a mean reach its subnormals
            err = (got.double() - dz / max(n, 1)).norm()
            assert float(err) <= u * float((dz / max(n, 1)).norm()) + floor * math.sqrt(z.numel())
        assert (got[~counts] == 0).all()
        up = torch.randn(T, generator=_gen(9), device="cuda")
        x = z.clone().requires_grad_()
        got, = _grads(losses.distillation(x, index, teacher, temperature=a, reduction="none"), x, up=up)
        _, dz, _ = ref_distill(z, index, teacher, a, up)
        if V > 1:
            floor = 2.0**-24 if dt == torch.float16 else 0.0
            assert float((got.double() - dz).norm()) <= u * float(dz.norm()) + floor * math.sqrt(z.numel())


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("T,D,V,K", [(1, 64, 3000, 5), (40, 72, 1000, 64), (260, 64, 300, 130), (9, 100, 5001, 1000),
                                     (600, 96, 513, 2)])
def test_linear_distillation(T, D, V, K, dtype):
    dt = DTYPES[dtype]
    h, w, _ = _head(T, D, V, dt, seed=T + K, scale=3.0)
    index, teacher = _teacher(T, V, K, K, dt)
    for a, chunk in ((1.0, 0), (2.0, 256)):
        z = h.double() @ w.double().t()
        want, dz, counts = ref_distill(z, index, teacher, a)
        n = max(1, int(counts.sum()))
        bound = _loss_bound(h, w, a) + a * a * 2.0**-17
        rows = losses.linear_distillation(h, w, index, teacher, temperature=a, reduction="none")
        assert ((rows - want).abs() <= bound).all()
        x, v = h.clone().requires_grad_(), w.clone().requires_grad_()
        loss = losses.linear_distillation(x, v, index, teacher, temperature=a, chunk_rows=chunk)
        assert abs(float(loss) - float(want.sum()) / n) <= float(bound.max())
        gh, gw = _grads(loss, x, v)
        assert _rel(gh, dz @ w.double() / n) <= GRAD_TOL[dt]
        assert _rel(gw, dz.t() @ h.double() / n) <= GRAD_TOL[dt]
        up = torch.randn(T, generator=_gen(9), device="cuda")
        rows = losses.linear_distillation(x, v, index, teacher, temperature=a, reduction="none")
        gh, gw = _grads(rows, x, v, up=up)
        _, dz, _ = ref_distill(z, index, teacher, a, up)
        assert _rel(gh, dz @ w.double()) <= GRAD_TOL[dt]
        assert _rel(gw, dz.t() @ h.double()) <= GRAD_TOL[dt]


def _both_forms(z, index, teacher, **kw):
    """Row losses and dz by the logits' form and, through an identity head, by the linear one."""
    V = z.shape[1]
    x = z.clone().requires_grad_()
    rows = losses.distillation(x, index, teacher, reduction="none", **kw)
    yield rows.detach(), _grads(rows, x, up=torch.ones_like(rows))[0]
    x = z.clone().requires_grad_()
    eye = torch.eye(V, device="cuda", dtype=z.dtype)
    rows = losses.linear_distillation(x, eye, index, teacher, reduction="none", **kw)
    yield rows.detach(), _grads(rows, x, up=torch.ones_like(rows))[0]


def test_distillation_entries_at_the_edge():
    """Repeated indices add up, -inf has no mass, the type's lowest value has, one-sided rows stay exact."""
    T, V, K = 7, 96, 6
    z = 2 * torch.randn(T, V, generator=_gen(21), device="cuda")
    index = torch.stack([torch.randperm(V, generator=_gen(s), device="cuda")[:K] for s in range(T)])
    teacher = torch.randn(T, K, generator=_gen(22), device="cuda")
    low = torch.finfo(torch.float32).min
    index[0] = torch.tensor([5, 5, 5, 9, 9, 95])
    teacher[1, :3] = -math.inf
    teacher[2] = -math.inf                      # no mass at all: counts for nothing
    teacher[3] = low                            # equal mass
    teacher[4, 1:] = low                        # one entry has it all
    index[5, 1:] = -1
    teacher[5, 1:] = math.inf                   # beside no entry: not looked at
    index[6] = -1
    want, dz, counts = ref_distill(z, index, teacher, 1.0)
    assert counts.tolist() == [True, True, False, True, True, True, False]
    for rows, grad in _both_forms(z, index, teacher):
        assert ((rows - want).abs() <= 2.0**-16).all()
        assert (grad[~counts] == 0).all()
        assert _rel(grad, dz) <= 2.0**-16
        assert _lib.device_error(reset=True) == 0


def test_distillation_masked_vocabulary():
    """A student's -inf logits have probability 0; an entry there makes the row's loss infinite, unless it has no mass."""
    T, V = 3, 64
    z = torch.randn(T, V, generator=_gen(23), device="cuda")
    z[:, 40:] = -math.inf
    index = torch.tensor([[1, 2, 50], [1, 50, 2], [3, 4, 5]], device="cuda")
    teacher = torch.tensor([[0.0, 1.0, -math.inf], [0.0, 1.0, 2.0], [0.0, 0.0, 0.0]], device="cuda")
    x = z.clone().requires_grad_()
    rows = losses.distillation(x, index, teacher, reduction="none")
    want, dz, _ = ref_distill(z, index, teacher, 1.0)
    assert math.isinf(float(rows[1])) and math.isclose(float(rows[0]), float(want[0]), rel_tol=1e-5)
    grad, = _grads(rows, x, up=torch.ones_like(rows))
    assert _rel(grad, dz) <= 2.0**-16
    x = torch.full((1, V), -math.inf, device="cuda")  # nothing to put mass on
    assert math.isnan(float(losses.distillation(x, index[:1], teacher[:1], reduction="none")))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("temperature", [1.0, 0.5, 4.0])
def test_distillation_masked_by_the_lowest_value(dtype, temperature):
    """Logits masked by the type's lowest finite value: probability 0 beside others, equal shares alone."""
    dt = DTYPES[dtype]
    T, V = 4, 300
    z = torch.randn(T, V, generator=_gen(31), device="cuda").to(dt)
    low = torch.finfo(dt).min
    z[0, 5:] = low
    z[1] = low
    z[2, ::2] = low
    index = torch.tensor([[0, 3], [7, 299], [1, 3], [0, 1]], device="cuda")
    teacher = torch.tensor([[0.0, 1.0]] * T, device="cuda")
    want, dz, _ = ref_distill(z, index, teacher, temperature)
    x = z.clone().requires_grad_()
    rows = losses.distillation(x, index, teacher, temperature=temperature, reduction="none")
    assert ((rows - want).abs() <= max(1.0, temperature**2) * 2.0**-17).all()
    grad, = _grads(rows, x, up=torch.ones_like(rows))
    assert torch.isfinite(grad).all()
    assert _rel(grad, dz) <= {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-10, torch.float32: 2.0**-17}[dt]


def test_distillation_bad_index_is_loud_and_contained():
    T, V = 5, 64
    z = torch.randn(T, V, generator=_gen(24), device="cuda")
    index = torch.randint(0, V, (T, 3), generator=_gen(25), device="cuda")
    teacher = torch.zeros(T, 3, device="cuda")
    index[2, 1] = V
    keep = torch.tensor([0, 1, 3, 4], device="cuda")
    want, dz, _ = ref_distill(z[keep], index[keep], teacher[keep], 1.0)
    for rows, grad in _both_forms(z, index, teacher):
        assert math.isnan(float(rows[2])) and (grad[2] == 0).all()
        assert ((rows[keep] - want).abs() <= 2.0**-16).all() and _rel(grad[keep], dz) <= 2.0**-16


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_distillation_strides_and_in_place(dtype):
    dt = DTYPES[dtype]
    T, V, K = 19, 1021, 12
    big = torch.randn(T, V + 6, generator=_gen(26), device="cuda").to(dt)
    index, teacher = _teacher(T, V, K, 3)
    wide_i, wide_t = torch.full((T, K + 2), -1, device="cuda"), torch.zeros(T, K + 1, device="cuda")
    wide_i[:, 1:K + 1], wide_t[:, :K] = index, teacher
    want, dz, counts = ref_distill(big[:, 5:V + 5], index, teacher, 1.0)
    x = big.clone().requires_grad_()
    rows = losses.distillation(x[:, 5:V + 5], wide_i[:, 1:K + 1].int(), wide_t[:, :K], reduction="none")
    assert ((rows - want).abs() <= 2.0**-17).all()
    got, = _grads(rows, x, up=torch.ones_like(rows))
    tol = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-10, torch.float32: 2.0**-17}[dt]
    assert _rel(got[:, 5:V + 5], dz) <= tol and (got[:, :5] == 0).all()
    t = torch.empty(V, T, device="cuda", dtype=dt).t().copy_(big[:, 5:V + 5])  # no row is contiguous
    assert ((losses.distillation(t, index, teacher, reduction="none") - want).abs() <= 2.0**-17).all()
    # the C entry may write the gradient over the logits
    buf = big.clone()
    view = buf[:, 5:V + 5]
    out = torch.empty(T, device="cuda")
    ones = torch.ones(T, device="cuda")
    _lib.check(_lib.load().po_distill_logits(
        view.data_ptr(), V + 6, _lib.DTYPE_CODE[dt], T, V, index.data_ptr(), K, teacher.data_ptr(), K, 0, K, 1.0, 0,
        ones.data_ptr(), out.data_ptr(), None, view.data_ptr(), V + 6, None, 0, _lib.stream_ptr(buf.device)), "in place")
    assert torch.equal(out, rows) and torch.equal(view, got[:, 5:V + 5])
    assert torch.equal(buf[:, :5], big[:, :5]) and torch.equal(buf[:, V + 5:], big[:, V + 5:])


def test_distillation_past_32_bit_offsets():
    T, V = 16800, 128256  # 2^31 elements and more
    z = torch.zeros(T, V, device="cuda", dtype=torch.bfloat16)
    z[-3:] = torch.randn(3, V, generator=_gen(27), device="cuda").to(z.dtype)
    index = torch.full((T, 2), -1, device="cuda")
    index[-3:] = torch.tensor([[0, 128255], [5, 6], [128254, 3]], device="cuda")
    teacher = torch.zeros(T, 2, device="cuda")
    want, dz, _ = ref_distill(z[-3:], index[-3:], teacher[-3:], 1.0)
    z.requires_grad_()
    loss = losses.distillation(z, index, teacher)
    assert math.isclose(float(loss), float(want.mean()), rel_tol=1e-5)
    got, = _grads(loss, z)
    assert _rel(got[-3:], dz / 3) <= 2.0**-8
    assert float(got[:100].abs().max()) == 0 and float(got[-40:-3].abs().max()) == 0


def test_linear_cross_entropy_past_32_bit_offsets():
    T, D, V = 17000, 64, 128256  # one chunk of 2^31 exponentials and more
    h, w, y = _head(T, D, V, torch.bfloat16, seed=28, scale=2.0)
    h.requires_grad_()
    loss = losses.linear_cross_entropy(h, w, y, reduction="sum", chunk_rows=1 << 20)
    gh, = _grads(loss, h)
    want, dh, _ = ref_ce(h.detach()[-300:], w, y[-300:])
    assert _rel(gh[-300:], dh) <= GRAD_TOL[h.dtype]


def test_distillation_empty():
    z = torch.empty(0, 10, device="cuda").requires_grad_()
    i, t = torch.empty(0, 2, dtype=torch.long, device="cuda"), torch.empty(0, 2, device="cuda")
    loss = losses.distillation(z, i, t)
    assert float(loss) == 0.0 and _grads(loss, z)[0].shape == (0, 10)
    assert losses.distillation(z, i, t, reduction="none").shape == (0,)


def test_fp16_gradients_of_a_mean_keep_their_digits_under_a_loss_scale():
    """p / n is far below fp16's smallest value; a loss scale lifts it back, as with gradients made after it."""
    T, D, V, K, up = 600, 64, 40000, 4, 2.0**14
    h, w, y = _head(T, D, V, torch.float16)
    want, dh, dw = ref_ce(h, w, y, up=torch.full((T,), up / T, device="cuda"))
    h.requires_grad_(), w.requires_grad_()
    gh, gw = _grads(losses.linear_cross_entropy(h, w, y) * up, h, w)
    rare = torch.ones(V, dtype=torch.bool, device="cuda")
    rare[y] = False  # rows of W that are nobody's target: p alone
    assert _rel(gh, dh) < GRAD_TOL[h.dtype] and _rel(gw, dw) < GRAD_TOL[h.dtype]
    assert float(dw[rare].abs().max()) / up < 2.0**-14 and _rel(gw[rare], dw[rare]) < 2.0**-7
    z, index, teacher = (torch.randn(T, V, generator=_gen(5), device="cuda").half(), *_teacher(T, V, K, 6))
    want, dz, counts = ref_distill(z, index, teacher, 2.0)
    dz *= up / int(counts.sum())
    z.requires_grad_()
    gz, = _grads(losses.distillation(z, index, teacher, temperature=2.0) * up, z)
    rest = torch.ones_like(z, dtype=torch.bool).scatter_(1, index.clamp(min=0), False)
    assert _rel(gz, dz) < 2.0**-9 and _rel(gz[rest], dz[rest]) < 2.0**-8


@pytest.mark.parametrize("size", [1.0, 40.0, 3000.0])
def test_fp16_gradients_of_a_mean_stay_in_range(size):
    """Every row the same large state and target: the largest gradients that states of this size can have."""
    T, D, V = 500, 64, 300
    h = torch.full((T, D), size, device="cuda", dtype=torch.float16)
    w = torch.zeros(V, D, device="cuda", dtype=torch.float16)
    w[1] = -0.25  # unlikely
    y = torch.ones(T, dtype=torch.long, device="cuda")
    want, dh, dw = ref_ce(h, w, y, up=torch.full((T,), 1 / T, device="cuda"))
    h.requires_grad_(), w.requires_grad_()
    gh, gw = _grads(losses.linear_cross_entropy(h, w, y), h, w)
    assert _rel(gh, dh) < GRAD_TOL[h.dtype] and _rel(gw, dw) < GRAD_TOL[h.dtype]


def test_scale_of_gradients_is_skipped_for_one():
    x = torch.randn(1001, device="cuda")
    lib = _lib.load()
    for dt in DTYPES.values():
        for off in (0, 1):  # on a 16-byte boundary, and not
            v, u = x.to(dt).clone()[off:], x.to(dt).clone()[off:off + 77]
            for a, b in ((v, u), (u, None)):
                for f in (0.3, 1.0):
                    factor = torch.tensor(f, device="cuda")
                    want = [(t.float() * f).to(dt) for t in (a, b) if t is not None]
                    _lib.check(lib.po_scale_inplace(a.data_ptr(), a.numel(), None if b is None else b.data_ptr(),
                                                    0 if b is None else b.numel(), _lib.DTYPE_CODE[dt],
                                                    factor.data_ptr(), _lib.stream_ptr(a.device)), "scale")
                    assert torch.equal(a, want[0])
                    assert b is None or torch.equal(b, want[1])


def test_example_trains_and_distills():
    """Losses and Muon together: the example's losses fall, and both forms of the divergence agree (the logits'
    form reads logits rounded to bf16: 2^-9 of logits of order 10)."""
    import importlib.util
    import os

    from tests.conftest import ROOT

    spec = importlib.util.spec_from_file_location("distill_lm", os.path.join(ROOT, "examples", "distill_lm.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    out = example.run(steps=60, vocab=1000, dim=128, rows=32, length=32, say=lambda *_: None)
    assert out["teacher last"] < 0.8 * out["teacher first"]
    assert out["student last"] < 0.8 * out["student first"]
    assert math.isclose(out["divergence, linear"], out["divergence, logits"], rel_tol=0.05)
