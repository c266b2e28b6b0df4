"""Orthogonalisation and the Muon step on the CPU path, and every refusal of the entry points."""
import math

import pytest
import torch

import distributeddeeplearning_amd.torch as hvd
from distributeddeeplearning_amd.ops import functional as ops
from distributeddeeplearning_amd.optim import FusedMuon


def oracle(g, steps=5, coef=ops.ORTHO_COEFFICIENTS, eps=1e-7):
    """The steps' polynomial on the singular values, 64 bits."""
    u, s, vh = torch.linalg.svd(g.double(), full_matrices=False)
    a, b, c = coef
    s = s / max(float(g.double().norm()), eps)
    for _ in range(steps):
        s = a * s + b * s ** 3 + c * s ** 5
    return (u * s) @ vh


@pytest.mark.parametrize("shape", [(1, 1), (1, 9), (9, 1), (16, 16), (24, 40), (40, 24)])
def test_plain_steps_are_a_polynomial_of_the_singular_values(shape):
    g = torch.randn(shape, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    torch.testing.assert_close(ops.orthogonalize_plain(g), oracle(g), rtol=1e-9, atol=1e-11)


def test_cpu_forms_and_types():
    gen = torch.Generator().manual_seed(2)
    mats = [torch.randn(s, generator=gen) for s in ((8, 20), (20, 8), (5, 5))]
    outs = ops.orthogonalize(mats)
    assert [o.shape for o in outs] == [m.shape for m in mats] and all(o.dtype == torch.bfloat16 for o in outs)
    for m, o in zip(mats, outs):
        # one rounding to bf16: at most half a step, 2^-8 of the value (fp32 steps: far below)
        torch.testing.assert_close(o.double(), oracle(m), rtol=2 ** -8, atol=1e-6)
    stack = torch.randn(3, 6, 11, generator=gen)
    o = ops.orthogonalize(stack)
    for k in range(3):
        assert torch.equal(o[k], ops.orthogonalize(stack[k]))
    assert ops.orthogonalize([]) == []
    assert ops.orthogonalize(torch.zeros(0, 4)).shape == (0, 4) and ops.orthogonalize(torch.zeros(2, 4, 0)).shape == (2, 4, 0)
    assert not ops.orthogonalize(torch.zeros(4, 7)).any()


@pytest.mark.parametrize("call, text", [
    (lambda: ops.orthogonalize(torch.zeros(3)), "matrix"),
    (lambda: ops.orthogonalize(torch.zeros(2, 2, 2, 2)), "matrix"),
    (lambda: ops.orthogonalize([torch.zeros(2, 2, 2)]), "matrix"),
    (lambda: ops.orthogonalize(torch.zeros(2, 2, dtype=torch.float16)), "fp32 or bf16"),
    (lambda: ops.orthogonalize(torch.zeros(2, 2, dtype=torch.float64)), "fp32 or bf16"),
    (lambda: ops.orthogonalize([torch.zeros(2, 2), torch.zeros(2, 2, dtype=torch.bfloat16)]), "share"),
    (lambda: ops.orthogonalize(torch.zeros(2, 2, requires_grad=True)), "gradient"),
    (lambda: ops.orthogonalize(torch.zeros(2, 2), steps=0), "steps"),
    (lambda: ops.orthogonalize(torch.zeros(2, 2), steps=-1), "steps"),
    (lambda: ops.orthogonalize(torch.zeros(2, 2), steps=65), "steps"),
    (lambda: ops.orthogonalize(torch.zeros(2, 2), steps=2.5), "steps"),
    (lambda: ops.orthogonalize(torch.zeros(2, 2), coefficients=(1.0, 2.0)), "coefficients"),
    (lambda: ops.orthogonalize(torch.zeros(2, 2), eps=0.0), "eps"),
    (lambda: ops.orthogonalize(torch.zeros(2, 2), eps=float("nan")), "eps"),
    (lambda: FusedMuon([("w", torch.nn.Parameter(torch.zeros(2, 2)))], lr=-1.0), "negative"),
    (lambda: FusedMuon([("w", torch.nn.Parameter(torch.zeros(2, 2)))], vector_lr_scale=-1.0), "negative"),
    (lambda: FusedMuon([("w", torch.nn.Parameter(torch.zeros(2, 2)))], steps=100), "steps"),
])
def test_refusals(call, text):
    with pytest.raises(ValueError, match=text):
        call()


def test_no_grad_input_is_taken():
    w = torch.randn(4, 6, requires_grad=True)
    with torch.no_grad():
        assert not ops.orthogonalize(w).requires_grad


class Net(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.conv = torch.nn.Conv2d(3, 6, 3)
        self.fc = torch.nn.Linear(10, 4)
        self.up = torch.nn.Linear(4, 10, bias=False)


def reference_step(w, g, v, lr, mu, wd, nesterov, matrix, vector_scale):
    """One parameter, 64 bits."""
    v.mul_(mu).add_(g)
    u = g + mu * v if nesterov else v
    if not matrix:
        return w.sub_(u, alpha=lr * vector_scale)
    o = oracle(u.reshape(w.shape[0], -1)).reshape(w.shape)
    rows, cols = w.shape[0], w[0].numel()
    return w.mul_(1 - lr * wd).sub_(o, alpha=lr * math.sqrt(max(1.0, rows / cols)))


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("distributed", [False, True])
def test_cpu_steps_follow_the_formula(nesterov, distributed):
    torch.manual_seed(3)
    net = Net()
    net.conv.weight.data = net.conv.weight.data.contiguous(memory_format=torch.channels_last)
    opt = FusedMuon(net.named_parameters(), lr=0.03, momentum=0.9, weight_decay=0.1, nesterov=nesterov, vector_lr_scale=0.5)
    if distributed:
        hvd.init()
        opt = hvd.DistributedOptimizer(opt, named_parameters=net.named_parameters())
    ref = {n: p.detach().double().clone() for n, p in net.named_parameters()}
    vel = {n: torch.zeros_like(w) for n, w in ref.items()}
    for _ in range(4):
        opt.zero_grad()
        for n, p in net.named_parameters():
            p.grad.copy_(torch.randn(p.shape))
            reference_step(ref[n], p.grad.double(), vel[n], 0.03, 0.9, 0.1, nesterov, p.dim() > 1, 0.5)
        opt.step()
    for n, p in net.named_parameters():
        # four fp32 steps of values of order one: 2^-24 each, some hundreds of operations
        torch.testing.assert_close(p.detach().double(), ref[n], rtol=1e-4, atol=2e-5)


def test_state_round_trip_and_choice_by_name():
    from distributeddeeplearning_amd.training.loop import build_optimizer
    from distributeddeeplearning_amd.utils.config import TrainConfig

    torch.manual_seed(4)
    a, b = Net(), Net()
    b.load_state_dict(a.state_dict())
    cfg = TrainConfig(optimizer="muon", lr=0.01, momentum=0.9)
    oa, ob = build_optimizer(cfg, a, 1), build_optimizer(cfg, b, 1)
    assert type(oa) is FusedMuon

    def step(net, opt, seed):
        gen = torch.Generator().manual_seed(seed)
        for _, p in net.named_parameters():
            p.grad.copy_(torch.randn(p.shape, generator=gen))
        opt.step()

    step(a, oa, 1)
    ob.load_state_dict(oa.state_dict())
    with torch.no_grad():
        for p, q in zip(a.parameters(), b.parameters()):
            q.copy_(p)
    step(a, oa, 2)
    step(b, ob, 2)
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.equal(p, q)


def test_sizes_that_the_kernels_refuse():
    """The library's own checks: before anything is launched, so they need no GPU."""
    from distributeddeeplearning_amd.ops import kernels, native

    if not native.kernels_available():
        pytest.skip("kernel library not built")

    def row(r, c, batch=1):
        return (64, r * c, c, 1, 64, r * c, c, 1, r, c, batch)

    for rows in ([row(0, 4)], [row(4, -1)], [row(1 << 30, 1)], [row(32768, 32769)], [row(4, 4, 0)], [row(4, 4, 1 << 23)], [row(4, 4, 1 << 40)],
                 [row(300, 300, 1 << 21)], [row(4, 4)] * 65):
        table, count = kernels.ortho_table(rows)
        with pytest.raises(kernels.KernelError, match="out of range"):
            kernels.ortho_workspace(table, count)
    # a launch has at most 2^32 - 1 threads: of 1024 for each matrix's sums and for the table
    table, count = kernels.ortho_table([row(4, 4, (1 << 22) - 3), row(32704, 32704)])
    with pytest.raises(kernels.KernelError, match="out of range"):      # (the second matrix has 1024 sums)
        kernels.ortho_workspace(table, count)
    table, count = kernels.ortho_table([row(4, 4, (1 << 22) - 1026), row(32704, 32704)])
    assert kernels.ortho_workspace(table, count) > 0 and kernels.ortho_workspace(*kernels.ortho_table([row(64, 300), row(100, 256)])) == 0
    lib = kernels.lib()
    ok = (3.4445, -4.7750, 2.0315)
    assert kernels.ortho_coefficients_ok(*ok, 5) and not kernels.ortho_coefficients_ok(*ok, 65) and not kernels.ortho_coefficients_ok(*ok, 0)

    def call(steps=5, eps=1e-7, kind=0, ws=256, nbytes=1 << 40, table=kernels.ortho_table([row(300, 300)])[0], count=1, coef=ok):
        f = lib.ddl_orthogonalize
        c = __import__("ctypes")
        return f(table, c.c_int(count), c.c_int(kind), *(c.c_float(v) for v in coef), c.c_int(steps), c.c_float(eps), c.c_void_p(ws),
                 c.c_longlong(nbytes), c.c_void_p(0))

    no_source = kernels.ortho_table([(0,) + row(300, 300)[1:]])[0]
    no_stride = kernels.ortho_table([row(300, 300)[:2] + (1 << 31,) + row(300, 300)[3:]])[0]
    for kw in (dict(steps=0), dict(steps=65), dict(eps=0.0), dict(eps=float("nan")), dict(kind=2), dict(kind=-1), dict(ws=0), dict(ws=64), dict(nbytes=100),
               dict(count=-1), dict(coef=(100.0, 0.0, 0.0)), dict(table=no_source), dict(table=no_stride)):
        assert call(**kw) != 0, kw
    assert call(count=0) == 0


def test_destinations_that_are_not_dense_are_refused():
    """Every form writes dense results; refused before anything is launched, so it needs no GPU."""
    import ctypes as c

    from distributeddeeplearning_amd.ops import kernels, native

    if not native.kernels_available():
        pytest.skip("kernel library not built")
    refused = -1                                          # DDL_EINVAL
    for r, cols in ((300, 400), (20, 700), (40, 90)):
        for db, drs, dcs, batch in ((r * cols, cols + 8, 1, 1), (r * cols, 1, r, 1), (r * cols, cols, 2, 1), (r * cols + 64, cols, 1, 3),
                                    (0, cols, 1, 2), (-1, cols, 1, 2), (r * cols, -cols, 1, 1)):
            table, count = kernels.ortho_table([(64, r * cols, cols, 1, 64, db, drs, dcs, r, cols, batch)])
            rc = kernels.lib().ddl_orthogonalize(table, c.c_int(count), c.c_int(0), c.c_float(3.4445), c.c_float(-4.7750), c.c_float(2.0315), c.c_int(5),
                                                 c.c_float(1e-7), c.c_void_p(256), c.c_longlong(1 << 40), c.c_void_p(0))
            assert rc == refused, (r, cols, db, drs, dcs, batch, rc)


OUT_OF_RANGE = [(50.0, 0.0, 0.0), (3.0, 3.0, 3.0), (float("nan"), 0.0, 0.0), (1.0, -40.0, 0.0), (1e39, 0.0, 0.0), (float("inf"), 0.0, 0.0)]


@pytest.mark.parametrize("coef", OUT_OF_RANGE, ids=str)
def test_coefficients_are_refused_on_the_cpu_and_when_the_optimizer_is_made(coef):
    with pytest.raises(ValueError, match="range"):
        ops.orthogonalize(torch.zeros(4, 4), coefficients=coef)
    p = torch.nn.Parameter(torch.zeros(2, 3))
    before = p.data_ptr()
    with pytest.raises(ValueError, match="range"):
        FusedMuon([("w", p)], coefficients=coef)
    assert p.data_ptr() == before and p.grad is None
    opt = FusedMuon([("w", p)])
    opt.param_groups[0]["ortho_a"], opt.param_groups[0]["ortho_b"], opt.param_groups[0]["ortho_c"] = coef
    with pytest.raises(ValueError, match="range"):
        opt.step()


def test_the_range_of_coefficients_is_the_librarys():
    from distributeddeeplearning_amd.ops import kernels, native

    if not native.kernels_available():
        pytest.skip("kernel library not built")
    gen = torch.Generator().manual_seed(5)
    taken = 0
    for i in range(4000):
        a, b, c = (torch.randn(3, generator=gen) * torch.tensor([3.0, 4.0, 2.0])).tolist()
        if i % 5 == 0:
            c = 0.0
        if i % 7 == 0:
            a, b, c = 3.4445 + 0.1 * a, -4.7750 + 0.1 * b, 2.0315 + 0.1 * c
        steps = 1 + i % 12
        taken += ops._steps_in_range(a, b, c, steps)
        assert ops._steps_in_range(a, b, c, steps) == kernels.ortho_coefficients_ok(a, b, c, steps), (a, b, c, steps)
    assert 500 < taken < 3500
    for coef in OUT_OF_RANGE + [(3.4445, -4.7750, 2.0315), (1.5, -0.5, 0.0), (2.0, -1.5, 0.5)]:
        assert ops._steps_in_range(*coef, 5) == kernels.ortho_coefficients_ok(*coef, 5)


@pytest.mark.parametrize("eps", [float("inf"), 1e39, -1.0, 1e-31])
def test_eps_that_fp32_does_not_hold_is_refused(eps):
    import ctypes as c

    from distributeddeeplearning_amd.ops import kernels, native

    with pytest.raises(ValueError, match="eps"):
        ops.orthogonalize(torch.zeros(4, 4), eps=eps)
    with pytest.raises(ValueError, match="eps"):
        FusedMuon([("w", torch.nn.Parameter(torch.zeros(2, 3)))], eps=eps)
    if native.kernels_available():
        table, count = kernels.ortho_table([(64, 90, 9, 1, 64, 90, 9, 1, 10, 9, 1)])
        assert kernels.lib().ddl_orthogonalize(table, c.c_int(count), c.c_int(0), c.c_float(3.4445), c.c_float(-4.7750), c.c_float(2.0315), c.c_int(5),
                                               c.c_float(eps), c.c_void_p(256), c.c_longlong(1 << 40), c.c_void_p(0)) == -1


def test_any_number_of_steps_is_answered_at_once():
    """The library's checks are not as long as the number of steps that they refuse."""
    import time

    from distributeddeeplearning_amd.ops import kernels, native

    if not native.kernels_available():
        pytest.skip("kernel library not built")
    table, count = kernels.ortho_table([(64, 90, 9, 1, 64, 90, 9, 1, 10, 9, 1)])
    start = time.perf_counter()
    for steps in (2 ** 31 - 1, 10 ** 9, -1, -(2 ** 31)):
        kernels.ortho_workspace(table, count, (1.5, -0.5, 0.0), steps)
        assert not kernels.ortho_coefficients_ok(1.5, -0.5, 0.0, steps)
    assert time.perf_counter() - start < 1.0
