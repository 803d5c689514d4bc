"""The loss operators at the edges of their arguments: empty and expanded
inputs, forward-mode derivatives, temperatures below 1, values near the types'
limits, upstream gradients of rows that count for nothing.

Definitions and tolerances are those of ``test_gpu_losses``; where a test has a
bound of its own, the reason stands beside it.
"""

import math

import pytest
import torch

from pytorch_opt_b200 import _lib, losses
from tests.test_gpu_losses import DTYPES, GRAD_TOL, _gen, _grads, _head, _loss_bound, _rel, _teacher, ref_ce, ref_distill

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_device_error(cuda):
    yield
    assert _lib.device_error(reset=True) == 0


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("top,temperature", [(1, 1.0), (3, 1.0), (1, 2.0), (5, 0.5)])
def test_linear_distillation_empty(top, temperature, reduction):
    w = torch.randn(10, 8, device="cuda").requires_grad_()
    h = torch.empty(0, 8, device="cuda").requires_grad_()
    i, t = torch.empty(0, top, dtype=torch.long, device="cuda"), torch.empty(0, top, device="cuda")
    loss = losses.linear_distillation(h, w, i, t, temperature=temperature, reduction=reduction)
    gh, gw = _grads(loss, h, w, up=torch.ones_like(loss))
    assert gh.shape == (0, 8) and (gw == 0).all()
    if reduction == "none":
        assert loss.shape == (0,)
    else:
        assert float(loss.detach()) == 0.0


def test_forward_mode_is_refused():
    """No tangent is lost silently: a dual tensor without requires_grad is refused like any other."""
    h, w, y = _head(20, 64, 300, torch.float32, seed=1)
    index, teacher = _teacher(20, 300, 3, 2)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(h, torch.ones_like(h))
        for reduction in ("mean", "none"):
            for call in (lambda a: losses.linear_cross_entropy(a, w, y, reduction=reduction),
                         lambda a: losses.linear_cross_entropy(h, torch.autograd.forward_ad.make_dual(w, w), y),
                         lambda a: losses.linear_distillation(a, w, index, teacher, reduction=reduction),
                         lambda a: losses.distillation(a, index.clamp(max=63), teacher, reduction=reduction)):
                with pytest.raises(RuntimeError):  # (NotImplementedError is one)
                    call(dual)
                with torch.no_grad(), pytest.raises(RuntimeError):  # which does not stop forward mode
                    call(dual)
        plain = losses.linear_cross_entropy(h, w, y)  # no dual among its inputs
    assert torch.equal(plain, losses.linear_cross_entropy(h, w, y))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("temperature", [0.5, 0.125, 2.0])
def test_teacher_entries_of_the_lowest_value(dtype, temperature):
    """Entries of the type's lowest value alone share equally at every temperature, and the row counts; beside
    others they have no mass; -inf has none. Both forms agree on what a mean divides by."""
    dt = DTYPES[dtype]
    T, V, K = 6, 64, 4
    z = torch.randn(T, V, generator=_gen(41), device="cuda")
    index = torch.stack([torch.randperm(V, generator=_gen(s), device="cuda")[:K] for s in range(T)])
    teacher = torch.randn(T, K, generator=_gen(42), device="cuda").to(dt)
    teacher[0] = torch.finfo(dt).min
    teacher[1, 1:] = torch.finfo(dt).min
    teacher[2] = -math.inf
    teacher[3, :2] = -math.inf
    teacher[3, 2:] = torch.finfo(dt).min
    teacher[4] = torch.finfo(dt).max
    want, dz, counts = ref_distill(z, index, teacher, temperature)
    assert counts.tolist() == [True, True, False, True, True, True]
    n, eye = int(counts.sum()), torch.eye(V, device="cuda")
    for form in (lambda a, r: losses.distillation(a, index, teacher, temperature=temperature, reduction=r),
                 lambda a, r: losses.linear_distillation(a, eye, index, teacher, temperature=temperature, reduction=r)):
        a = z.clone().requires_grad_()
        rows = form(a, "none")
        assert ((rows - want).abs() <= max(1.0, temperature**2) * 2.0**-16).all()
        assert _rel(_grads(rows, a, up=torch.ones_like(rows))[0], dz) <= 2.0**-16
        loss = form(a, "mean")
        assert abs(float(loss.detach()) - float(want.sum()) / n) <= max(1.0, temperature**2) * 2.0**-16
        assert _rel(_grads(loss, a)[0], dz / n) <= 2.0**-16


def test_targets_of_one_value_expanded():
    """A target that is a broadcast view, as a constant one often is."""
    T, D, V = 37, 64, 300
    h, w, _ = _head(T, D, V, torch.bfloat16, seed=3)
    y = torch.full((1,), 7, device="cuda").expand(T)
    want, dh, dw = ref_ce(h, w, y)
    rows = losses.linear_cross_entropy(h, w, y, reduction="none")
    assert ((rows - want).abs() <= _loss_bound(h, w)).all()
    a = h.reshape(1, T, D).expand(2, T, D)
    both = losses.linear_cross_entropy(a, w, y.expand(2, T).int(), reduction="none")
    assert torch.equal(both[0], rows) and torch.equal(both[1], rows)
    index, teacher = y[:1, None].expand(T, 1), torch.zeros(1, 1, device="cuda").expand(T, 1)
    same = losses.linear_distillation(h, w, index, teacher, reduction="none")  # all mass on one entry
    assert ((same - want).abs() <= _loss_bound(h, w) + 2.0**-17).all()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan, 1e30])
@pytest.mark.parametrize("form", ["ce", "distil"])
def test_upstream_of_rows_that_count_for_nothing_is_not_looked_at(form, value, dtype):
    """A division by a masked row's weight leaves anything as its upstream gradient."""
    T, D, V = 70, 64, 300
    dt = DTYPES[dtype]
    h, w, y = _head(T, D, V, dt, seed=4)
    up = 100.0 * torch.rand(T, generator=_gen(5), device="cuda")
    index, teacher = _teacher(T, V, 4, 6, holes=False)
    off = torch.zeros(T, dtype=torch.bool, device="cuda")
    off[3::4] = True
    y[off], index[off] = -100, -1
    if form == "ce":
        _, dh, dw = ref_ce(h, w, y, up=up)
    else:
        _, dz, _ = ref_distill(h.double() @ w.double().t(), index, teacher, 1.0, up)
        dh, dw = dz @ w.double(), dz.t() @ h.double()
    up[off] = value
    h.requires_grad_(), w.requires_grad_()
    rows = (losses.linear_cross_entropy(h, w, y, reduction="none") if form == "ce" else
            losses.linear_distillation(h, w, index, teacher, reduction="none"))
    gh, gw = _grads(rows, h, w, up=up)
    assert _rel(gh, dh) <= GRAD_TOL[dt] and _rel(gw, dw) <= GRAD_TOL[dt]


def test_upstream_of_one_row_that_is_infinite_stays_there():
    T, D, V = 70, 64, 300
    h, w, y = _head(T, D, V, torch.float16, seed=4)
    up = 100.0 + torch.rand(T, generator=_gen(5), device="cuda")
    _, dh, _ = ref_ce(h, w, y, up=up)
    up[9] = math.inf
    rest = torch.arange(T, device="cuda") != 9
    h.requires_grad_()
    gh, = _grads(losses.linear_cross_entropy(h, w, y, reduction="none"), h, up=up)
    assert _rel(gh[rest], dh[rest]) <= GRAD_TOL[h.dtype] and not torch.isfinite(gh[9]).any()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("copies", [1, 5])  # up to two rows (eight in fp32) go to the CUDA cores
@pytest.mark.parametrize("temperature", [1.0, 0.5])
def test_linear_logits_near_the_largest_value(temperature, copies, dtype):
    """Finite logits of 3e38 at temperature 1 and 1.5e38 at 0.5: only differences from the row's maximum are scaled."""
    dt = DTYPES[dtype]
    V = 96
    big = 3e38 * temperature
    z = torch.zeros(2, V, device="cuda")
    z[0] = -big                                  # masked throughout: equal shares
    z[1, :4], z[1, 4:] = big, torch.randn(V - 4, generator=_gen(51), device="cuda")
    z = z.repeat(copies, 1).to(dt)
    y = torch.tensor([3, 1], device="cuda").repeat(copies)
    want = torch.tensor([math.log(V), math.log(4.0)], dtype=torch.float64, device="cuda").repeat(copies)
    p = torch.zeros(2, V, dtype=torch.float64, device="cuda")
    p[0], p[1, :4] = 1 / V, 0.25
    dz = p.repeat(copies, 1)
    dz[torch.arange(2 * copies), y] -= 1
    eye = torch.eye(V, device="cuda", dtype=dt)
    index, teacher = y[:, None], torch.zeros(2 * copies, 1, device="cuda")  # all mass on the target
    calls = [lambda a, r: losses.linear_distillation(a, eye, index, teacher, temperature=temperature, reduction=r)]
    if temperature == 1.0:
        calls.append(lambda a, r: losses.linear_cross_entropy(a, eye, y, reduction=r))
    for call in calls:
        a = z.clone().requires_grad_()
        rows = call(a, "none")
        # log and exponentials of equal logits: a few roundings of numbers below 8, times a^2.
        assert ((rows - temperature**2 * want).abs() <= 2.0**-20).all()
        assert _rel(_grads(rows, a, up=torch.ones_like(rows))[0], temperature * dz) <= GRAD_TOL[dt]
        assert _rel(_grads(call(a, "sum"), a)[0], temperature * dz) <= GRAD_TOL[dt]


def test_temperatures_whose_square_has_no_fp32():
    """Losses have the factor a^2 and exponents 1 / a: beyond 2^-60 .. 2^60 one of them leaves fp32's range."""
    h, w, _ = _head(4, 8, 16, torch.bfloat16)
    i, t = torch.zeros(4, 2, dtype=torch.long, device="cuda"), torch.zeros(4, 2, device="cuda")
    for a in (1e-39, 2.0**-61, 2.0**61, 1e30):
        with pytest.raises(RuntimeError, match="temperature"):
            losses.linear_distillation(h, w, i, t, temperature=a)
        with pytest.raises(RuntimeError, match="temperature"):
            losses.distillation(torch.randn(4, 16, device="cuda"), i, t, temperature=a)
    for a in (2.0**-60, 2.0**60):
        assert torch.isfinite(losses.linear_distillation(h, w, i, t, temperature=a))
        assert torch.isfinite(losses.distillation(torch.randn(4, 16, device="cuda"), i, t, temperature=a))


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("T,chunk", [(2, 0), (300, 0), (900, 0), (900, 256)])
@pytest.mark.parametrize("z_loss,top,shared", [(0.5, 120.0, 0.25), (2.0, 250.0, 4.0), (-0.5, 120.0, 0.25)])
def test_fp16_gradients_of_a_large_z_loss(z_loss, top, shared, T, chunk, reduction):
    """(1 + 2 c lse) softmax reaches a thousand times softmax, later rows the most; the gradients fit fp16."""
    D, V = 64, 500
    h, w, y = _head(T, D, V, torch.float16, seed=T, scale=0.5)
    w[:, 0] = shared
    h[:, 0] = torch.linspace(2.0, top, T, device="cuda") / shared  # adds 2 .. top to every logit of a row
    w[:, 1] = 0
    w[:7, 1] = 2.0
    h[:, 1] = 4.0                                             # and 8 to seven of them: some p are large
    y[5::9] = -100
    n = int((y != -100).sum())
    up = torch.full((T,), 1 / n if reduction == "mean" else 2.0**-6, device="cuda")
    want, dh, dw = ref_ce(h, w, y, 0.0, z_loss, -100, up)
    assert max(float(dh.abs().max()), float(dw.abs().max())) < 60000
    h.requires_grad_(), w.requires_grad_()
    loss = losses.linear_cross_entropy(h, w, y, z_loss=z_loss, reduction=reduction, chunk_rows=chunk)
    if reduction == "none":
        gh, gw = _grads(loss, h, w, up=up)
    else:
        gh, gw = _grads(loss, h, w, up=torch.tensor(1.0 if reduction == "mean" else 2.0**-6, device="cuda"))
    assert _rel(gh, dh) <= GRAD_TOL[h.dtype] and _rel(gw, dw) <= GRAD_TOL[h.dtype]


def test_fp16_gradients_of_a_large_z_loss_under_a_loss_scale():
    """As without z-loss, rare rows of W keep their digits until the loss scale comes, in chunks or not."""
    T, D, V, up = 600, 64, 20000, 2.0**10
    h, w, y = _head(T, D, V, torch.float16)
    w[:, 0] = 1.0
    h[:, 0] = torch.linspace(0.0, 90.0, T, device="cuda")
    _, dh, dw = ref_ce(h, w, y, 0.0, 0.5, -100, torch.full((T,), up / T, device="cuda"))
    h.requires_grad_(), w.requires_grad_()
    for chunk in (0, 256):
        gh, gw = _grads(losses.linear_cross_entropy(h, w, y, z_loss=0.5, chunk_rows=chunk) * up, h, w)
        assert _rel(gh, dh) < GRAD_TOL[h.dtype] and _rel(gw, dw) < GRAD_TOL[h.dtype]


@pytest.mark.parametrize("T", [1, 2])
def test_fp16_gradients_of_few_rows_keep_their_digits_under_a_loss_scale(T):
    """As those of many: rows of W that are nobody's target have p h, far below fp16's smallest normal value."""
    D, V, up = 64, 128256, 2.0**16
    h, w, y = _head(T, D, V, torch.float16, seed=9, scale=0.1)
    _, dh, dw = ref_ce(h, w, y, up=torch.full((T,), up / T, device="cuda"))
    h.requires_grad_(), w.requires_grad_()
    gh, gw = _grads(losses.linear_cross_entropy(h, w, y) * up, h, w)
    rare = torch.ones(V, dtype=torch.bool, device="cuda")
    rare[y] = False
    assert _rel(gh, dh) < GRAD_TOL[h.dtype] and _rel(gw, dw) < GRAD_TOL[h.dtype]
    assert _rel(gw[rare], dw[rare]) < 2.0**-7


@pytest.mark.parametrize("form", ["ce", "distil"])
@pytest.mark.parametrize("T", [2, 600, 4000])
def test_fp16_gradients_of_a_sum_divided_afterwards_stay_in_range(T, form):
    """loss_sum / n: the sum's own gradient of a frequent target's row may lie beyond fp16, the mean's does not."""
    D, V = 64, 100
    h = torch.full((T, D), 80000.0 / T if T > 2 else 40000.0, device="cuda", dtype=torch.float16)
    w = torch.zeros(V, D, device="cuda", dtype=torch.float16)
    y = torch.ones(T, dtype=torch.long, device="cuda")
    _, dh, dw = ref_ce(h, w, y, up=torch.full((T,), 1 / T, device="cuda"))
    assert float(dw.abs().max()) * T > 65504 > float(dw.abs().max())
    h.requires_grad_(), w.requires_grad_()
    for chunk in (0, 256):
        loss = (losses.linear_cross_entropy(h, w, y, reduction="sum", chunk_rows=chunk) if form == "ce" else
                losses.linear_distillation(h, w, y[:, None], torch.zeros(T, 1, device="cuda"), reduction="sum",
                                           chunk_rows=chunk))
        gh, gw = _grads(loss / T, h, w)
        assert torch.isfinite(gw).all() and _rel(gw, dw) <= GRAD_TOL[h.dtype]
        assert float(gh.abs().max()) == 0.0  # W is 0


def test_splits_chosen_on_the_device_have_the_whole_gpu(tmp_path):
    """Half of the rows count, so dH's 32 tiles take two splits or more: their launch has a pair of SMs for each
    unit, although the host, which knows of 60 tiles, splits nothing."""
    import json

    T, D, V = 3840, 1024, 20000
    h, w, y = _head(T, D, V, torch.bfloat16, seed=8)
    y[::2] = -100
    _, dh, _ = ref_ce(h, w, y)
    h.requires_grad_()
    loss = lambda: losses.linear_cross_entropy(h, w, y, reduction="sum")  # noqa: E731
    gh, = _grads(loss(), h)
    assert _rel(gh, dh) <= GRAD_TOL[h.dtype]
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        loss()
        torch.cuda.synchronize()
    prof.export_chrome_trace(str(tmp_path / "trace.json"))
    events = json.loads((tmp_path / "trace.json").read_text())["traceEvents"]
    heads = sorted((e["ts"], e["args"]["grid"][0]) for e in events
                   if e.get("cat") == "kernel" and "head_gemm_kernel" in e["name"])
    assert len(heads) == 2  # logits, dH
    pairs = torch.cuda.get_device_properties(0).multi_processor_count // 2
    assert heads[1][1] >= 2 * min(pairs, 64)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("form", ["ce", "linear", "logits"])
def test_gradients_under_graph_capture(form, reduction, dtype):
    """A step's loss and gradients captured once, replayed on other inputs."""
    T, D, V, K = 100, 64, 1000, 5
    dt = DTYPES[dtype]

    def inputs(seed):
        h, w, y = _head(T, D, V, dt, seed=seed)
        y[seed % 7::7] = -100
        return [h, w, y, *_teacher(T, V, K, seed), torch.rand(T, generator=_gen(seed), device="cuda")]

    at = inputs(18)
    h, w, y, index, teacher, up = at
    leaves = [h.clone().requires_grad_(), w.clone().requires_grad_()]
    z = (h @ w.t()).requires_grad_()

    def step():
        if form == "logits":
            loss, xs = losses.distillation(z, index, teacher, reduction=reduction), [z]
        elif form == "ce":
            loss, xs = losses.linear_cross_entropy(*leaves, y, reduction=reduction), leaves
        else:
            loss, xs = losses.linear_distillation(*leaves, index, teacher, reduction=reduction), leaves
        return (loss, *_grads(loss, *xs, up=up if reduction == "none" else None))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (19, 20):
        with torch.no_grad():
            for a, b in zip(at, inputs(seed)):
                a.copy_(b)
            leaves[0].copy_(h), leaves[1].copy_(w), z.copy_(h @ w.t())
        graph.replay()
        torch.cuda.synchronize()
        n = int((y != -100).sum()) if form == "ce" else int((index >= 0).any(1).sum())
        u = up if reduction == "none" else torch.full((T,), 1 / n, device="cuda")
        if form == "ce":
            want, dh, dw = ref_ce(h, w, y, up=u)
        else:
            zz = z.detach().double() if form == "logits" else h.double() @ w.double().t()
            want, dz, _ = ref_distill(zz, index, teacher, 1.0, u)
            dh, dw = dz @ w.double(), dz.t() @ h.double()
        bound = _loss_bound(h, w) + 2.0**-17
        if reduction == "none":
            assert ((got[0].detach() - want).abs() <= bound).all()
        else:
            assert abs(float(got[0].detach()) - float(want.sum()) / n) <= float(bound.max())
        grads = (dz,) if form == "logits" else (dh, dw)
        for a, b in zip(got[1:], grads):
            assert _rel(a, b) <= GRAD_TOL[dt]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("soft", [False, True])
def test_masked_rows_among_many(soft, dtype):
    """More than 16384 rows: a packing block takes several groups of eight."""
    T, D, V = 33001, 72, 130
    dt = DTYPES[dtype]
    h, w, y = _head(T, D, V, dt, seed=30, scale=2.0)
    drop = torch.rand(T, generator=_gen(31), device="cuda") < 0.4
    drop[1000:9000] = True
    drop[20000:28000] = False
    y[drop] = -100
    h[drop] = math.nan
    if soft:
        index, teacher = y[:, None].clone(), torch.zeros(T, 1, device="cuda")
        index[drop] = -1
    want, dh, dw = ref_ce(h, w, y)
    call = lambda a, b, **k: (losses.linear_distillation(a, b, index, teacher, **k) if soft else  # noqa: E731
                              losses.linear_cross_entropy(a, b, y, **k))
    rows = call(h, w, reduction="none")
    assert ((rows - want).abs() <= torch.where(drop, 0.0, _loss_bound(torch.where(drop[:, None], 0.0, h), w)) + 2.0**-17 * soft).all()
    n = int((~drop).sum())
    h.requires_grad_(), w.requires_grad_()
    for chunk in (0, 8192):
        gh, gw = _grads(call(h, w, chunk_rows=chunk), h, w)
        assert (gh[drop] == 0).all()
        assert _rel(gh, dh / n) <= GRAD_TOL[dt] and _rel(gw, dw / n) <= GRAD_TOL[dt]


@pytest.mark.parametrize("T", [1, 2, 30, 600])
def test_fp16_gradients_of_a_sum_keep_their_digits_under_a_loss_scale(T):
    """Softmax itself is below fp16's smallest normal value in a large vocabulary; loss_sum / n times a scale lifts it."""
    D, V, K, up = 64, 60000, 4, 2.0**12
    h, w, y = _head(T, D, V, torch.float16, seed=10, scale=0.1)
    _, dh, dw = ref_ce(h, w, y, up=torch.full((T,), up / T, device="cuda"))
    h.requires_grad_(), w.requires_grad_()
    gh, gw = _grads(losses.linear_cross_entropy(h, w, y, reduction="sum") / T * up, h, w)
    rare = torch.ones(V, dtype=torch.bool, device="cuda")
    rare[y] = False
    assert _rel(gh, dh) < GRAD_TOL[h.dtype] and _rel(gw, dw) < GRAD_TOL[h.dtype]
    # A division by T that is no power of two rounds once more; 2^-7 as for a mean.
    assert _rel(gw[rare], dw[rare]) < 2.0**-7
    z, index, teacher = (4 * torch.randn(T, V, generator=_gen(5), device="cuda").half(), *_teacher(T, V, K, 6))
    _, dz, _ = ref_distill(z, index, teacher, 2.0, torch.full((T,), up / T, device="cuda"))
    z.requires_grad_()
    gz, = _grads(losses.distillation(z, index, teacher, temperature=2.0, reduction="sum") / T * up, z)
    rest = torch.ones_like(z, dtype=torch.bool).scatter_(1, index.clamp(min=0), False)
    rest &= dz.abs() > 2.0**-13  # what fp16 holds to 2^-11 once it is scaled
    # Each value is rounded to 2^-11 twice.
    assert _rel(gz, dz) < 2.0**-9
    assert float(((gz.double() - dz).abs() / dz.abs().clamp_min(1e-30))[rest].max()) < 2.0**-9


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("mode", [2, 3])
def test_c_functions_report_the_factors_they_store_by(mode, dtype):
    """PO_MEAN_SCALED and PO_SUM_SCALED of every type: stored gradients times the reported factors are the gradients;
    for bf16 and fp32 the factors are 1."""
    dt, lib = DTYPES[dtype], _lib.load()
    T, D, V, K = 40, 64, 300, 3
    h, w, y = _head(T, D, V, dt, seed=12)
    index, teacher = _teacher(T, V, K, 5)
    n = T if mode == 2 else 1
    _, dh, dw = ref_ce(h, w, y)
    loss, code, stream = torch.empty((), device="cuda"), _lib.DTYPE_CODE[dt], _lib.stream_ptr(h.device)
    rows = torch.full((T + 2,), math.nan, device="cuda")
    gh, gw = torch.empty_like(h), torch.empty_like(w)
    nbytes = lib.po_linear_loss_workspace_bytes(w.data_ptr(), D, code, T, D, V, 1, 1, 1, 0)
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    _lib.check(lib.po_linear_loss(
        h.data_ptr(), D, w.data_ptr(), D, code, T, D, V, y.data_ptr(), 1, None, 0, 0, 1, -100, 0.0, 0.0, 1.0, mode, None,
        rows.data_ptr(), loss.data_ptr(), gh.data_ptr(), D, gw.data_ptr(), D, 0, ws.data_ptr(), nbytes, stream), "head")
    assert _rel(gh.double() * rows[T].double(), dh / n) <= GRAD_TOL[dt]
    assert _rel(gw.double() * rows[T + 1].double(), dw / n) <= GRAD_TOL[dt]
    assert dtype == "fp16" or (rows[T:] == 1).all()
    z = torch.randn(T, V, generator=_gen(13), device="cuda").to(dt)
    _, dz, counts = ref_distill(z, index, teacher, 1.0)
    n = int(counts.sum()) if mode == 2 else 1
    rows, gz = torch.full((T + 1,), math.nan, device="cuda"), torch.empty_like(z)
    ws = torch.empty(lib.po_distill_logits_workspace_bytes(T), dtype=torch.uint8, device="cuda")
    _lib.check(lib.po_distill_logits(
        z.data_ptr(), V, code, T, V, index.data_ptr(), K, teacher.data_ptr(), K, 0, K, 1.0, mode, None, rows.data_ptr(),
        loss.data_ptr(), gz.data_ptr(), V, ws.data_ptr(), ws.numel(), stream), "logits")
    assert _rel(gz.double() * rows[T].double(), dz / n) <= GRAD_TOL[dt]
    assert dtype == "fp16" or float(rows[T]) == 1.0
