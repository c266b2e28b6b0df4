"""Orthogonalisation kernels and the Muon step against the formula in 64 bits, where they can go wrong: odd sizes, strides,
spectra, empty and infinite matrices, many matrices, captured graphs, other streams, the launch tape."""
import math

import pytest
import torch

from tests.test_orthogonalize import oracle, reference_step

pytestmark = pytest.mark.gpu
DEV, BF = "cuda", torch.bfloat16

# Result: one rounding to bf16 (half a step: 2^-8 of each value).  Within the five steps the products' operands are rounded to
# fp16 three times a step (half a step: 2^-11): 15 * 2^-11 = 7.3e-3 if every one of them were at its largest and of one sign.
TOL = 2 ** -8 + 15 * 2 ** -11


def off(out, g, **kw):
    """Relative 2-norm error."""
    e = oracle(g.cpu(), **kw)
    return float((out.double().cpu() - e).norm() / max(float(e.norm()), 1e-30))


def spectrum(kind, r, c, seed=0):
    gen = torch.Generator().manual_seed(seed)
    k = min(r, c)
    if kind == "gauss":
        return torch.randn(r, c, generator=gen)
    left = torch.linalg.qr(torch.randn(r, k, generator=gen, dtype=torch.float64))[0]
    right = torch.linalg.qr(torch.randn(c, k, generator=gen, dtype=torch.float64))[0]
    i = torch.arange(k, dtype=torch.float64)
    s = {"power": 1 / (i + 1), "exp": 10 ** (-6 * i / max(k - 1, 1)), "rank1": (i == 0).double(),
         "lowrank": torch.where(i < max(1, k // 16), 1.0, 1e-3)}[kind]
    return ((left * s) @ right.T).float()


SHAPES = [(1, 1), (1, 7), (7, 1), (3, 1000), (64, 64), (65, 63), (63, 130), (128, 128), (129, 257), (257, 129), (64, 147),
          (300, 1000), (1000, 300), (256, 2304), (512, 513), (640, 640)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, BF], ids=["fp32", "bf16"])
def test_sizes(shape, dtype):
    from distributeddeeplearning_amd.ops import functional as ops

    g = spectrum("gauss", *shape).to(DEV, dtype)
    keep = g.clone()
    out = ops.orthogonalize(g)
    assert out.shape == g.shape and out.dtype == BF and torch.equal(g, keep)
    assert off(out, g) < TOL


@pytest.mark.parametrize("kind", ["power", "exp", "rank1", "lowrank"])
@pytest.mark.parametrize("shape", [(96, 200), (256, 1024), (400, 256)], ids=str)
def test_spectra(kind, shape):
    from distributeddeeplearning_amd.ops import functional as ops

    g = spectrum(kind, *shape, seed=5).to(DEV)
    assert off(ops.orthogonalize(g), g) < TOL


@pytest.mark.parametrize("steps, coef", [(1, (3.4445, -4.7750, 2.0315)), (7, (3.4445, -4.7750, 2.0315)),
                                         (12, (2.0, -1.5, 0.5)), (20, (1.5, -0.5, 0.0))])
def test_steps_and_coefficients(steps, coef):
    from distributeddeeplearning_amd.ops import functional as ops

    g = spectrum("gauss", 70, 200, 2).to(DEV)
    out = ops.orthogonalize(g, steps=steps, coefficients=coef)
    assert off(out, g, steps=steps, coef=coef) < 2 ** -8 + 3 * steps * 2 ** -11


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e30])
def test_magnitudes(scale):
    """Squares of these leave fp32; below eps the matrix is divided by eps."""
    from distributeddeeplearning_amd.ops import functional as ops

    g = (spectrum("gauss", 40, 90, 3) * scale).to(DEV)
    out = ops.orthogonalize(g, eps=1e-20)
    assert off(out, g, eps=1e-20) < TOL


def test_strides_stacks_and_lists():
    from distributeddeeplearning_amd.ops import functional as ops

    base = spectrum("gauss", 200, 331, 4).to(DEV)
    views = [base.t(), base[3:100, 5:200], base[::2, 1::3], base[:, 7:8], base[10:11], base[:50, :50].expand(50, 50)]
    for v in views:
        assert off(ops.orthogonalize(v), v) < TOL
    stack = spectrum("gauss", 5 * 70, 33, 6).to(DEV).view(5, 70, 33)
    for s in (stack, stack.transpose(0, 1), stack.transpose(1, 2), stack[::2, 1:, :20], stack[:1].expand(4, 70, 33)):
        out = ops.orthogonalize(s)
        assert out.shape == s.shape
        for k in range(s.shape[0]):
            assert off(out[k], s[k]) < TOL
    # more matrices than one launch takes, ragged, some empty
    mats = [spectrum("gauss", 1 + 7 * (i % 13), 1 + 11 * (i % 17), i).to(DEV) for i in range(150)]
    mats[20], mats[140] = torch.empty(0, 5, device=DEV), torch.empty(5, 0, device=DEV)
    outs = ops.orthogonalize(mats)
    for m, o in zip(mats, outs):
        assert o.shape == m.shape and (m.numel() == 0 or off(o, m) < TOL)
    assert ops.orthogonalize([mats[20]])[0].shape == (0, 5)


def test_matrices_do_not_touch_each_other():
    from distributeddeeplearning_amd.ops import functional as ops

    clean = [spectrum("gauss", 65, 130, i).to(DEV) for i in range(4)]
    want = ops.orthogonalize(clean)
    bad = [m.clone() for m in clean]
    bad[1][3, 4] = float("nan")
    bad[2][64, 129] = float("inf")
    bad.insert(1, torch.zeros(65, 130, device=DEV))
    got = ops.orthogonalize(bad)
    assert torch.equal(got[0], want[0]) and torch.equal(got[4], want[3])
    assert not got[1].any() and got[2].isnan().all() and got[3].isnan().all()


def test_out_of_range_coefficients_are_refused():
    from distributeddeeplearning_amd.ops import functional as ops

    for coef in ((50.0, 0.0, 0.0), (3.0, 3.0, 3.0), (float("nan"), 0.0, 0.0), (1.0, -40.0, 0.0)):
        with pytest.raises(ValueError, match="range"):
            ops.orthogonalize(torch.zeros(4, 4, device=DEV), coefficients=coef)


def test_repeated_calls_are_equal_and_other_streams_work():
    from distributeddeeplearning_amd.ops import functional as ops

    g = [spectrum("gauss", 300, 700, 1).to(DEV), spectrum("power", 512, 64, 2).to(DEV)]
    a = ops.orthogonalize(g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = ops.orthogonalize(g)
    torch.cuda.current_stream().wait_stream(side)
    c = ops.orthogonalize(g)
    for x, y, z in zip(a, b, c):
        assert torch.equal(x, y) and torch.equal(x, z)


def test_two_captured_graphs():
    from distributeddeeplearning_amd.ops import functional as ops

    xs = [torch.zeros(130, 260, device=DEV), torch.zeros(3, 64, 70, device=DEV)]
    graphs, outs = [], []
    for x in xs:
        ops.orthogonalize(x)
    torch.cuda.synchronize()
    for x in xs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.orthogonalize(x))
        graphs.append(gr)
    for rep in range(4):
        for x in xs:
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(rep)))
        for gr in graphs if rep % 2 else graphs[::-1]:
            gr.replay()
        eager = [ops.orthogonalize(x) for x in xs]
        torch.cuda.synchronize()
        for o, e in zip(outs, eager):
            assert torch.equal(o, e)


# ---------------------------------------------------------------------------------------------------- the optimizer
def _params(shapes, dtype, seed=0, many=0):
    gen = torch.Generator().manual_seed(seed)
    out = []
    for i, s in enumerate(list(shapes) + [(6 + i % 5, 9 + i % 7) for i in range(many)]):
        t = (0.1 * torch.randn(s, generator=gen)).to(DEV)
        t = t.to(dtype) if len(s) > 1 else t
        if len(s) == 4:
            t = t.contiguous(memory_format=torch.channels_last)
        out.append(("p%d" % i, torch.nn.Parameter(t)))
    return out


MUON_SHAPES = [(64,), (64, 3, 7, 7), (130, 64, 3, 3), (200, 130, 1, 1), (200,), (10, 200), (257, 31), (1, 5), (5, 1)]


@pytest.mark.parametrize("dtype, grads", [(BF, "auto"), (BF, "fp32"), (torch.float32, "auto")], ids=["bf16", "bf16-fp32-grads", "fp32"])
@pytest.mark.parametrize("nesterov, wd, many", [(True, 0.0, 0), (False, 0.05, 0), (True, 0.05, 70)])
def test_muon_steps(dtype, grads, nesterov, wd, many):
    from distributeddeeplearning_amd.optim import FusedMuon
    from distributeddeeplearning_amd.utils.config import EngineConfig

    named = _params(MUON_SHAPES, dtype, many=many)
    opt = FusedMuon(named, lr=0.02, momentum=0.9, weight_decay=wd, nesterov=nesterov, vector_lr_scale=0.25,
                    engine_config=EngineConfig(comm_dtype=grads))
    ref = {n: p.detach().double().cpu() for n, p in named}
    vel = {n: torch.zeros_like(w) for n, w in ref.items()}
    change = {n: 0.0 for n in ref}
    for step in range(3):
        gen = torch.Generator().manual_seed(100 + step)
        for n, p in named:
            p.grad.copy_(1e-3 * torch.randn(p.shape, generator=gen))
            before = ref[n].clone()
            reference_step(ref[n], p.grad.double().cpu(), vel[n], 0.02, 0.9, wd, nesterov, p.dim() > 1, 0.25)
            change[n] += float((ref[n] - before).norm())
        opt.step()
    torch.cuda.synchronize()
    for dt, plan in opt.arena.plans.items():
        covered = torch.zeros(plan.numel, dtype=torch.bool)
        for seg in plan.segments:
            w = opt._weights(dt)[seg.offset:seg.offset + seg.numel]
            v = opt.momentum_buf[dt][seg.offset:seg.offset + seg.numel]
            covered[seg.offset:seg.offset + seg.numel] = True

            def flat(t):
                return (t.permute(0, 2, 3, 1) if t.dim() == 4 else t).reshape(-1)

            # the weights are fp32: off by the direction's error (16-bit products; no final rounding) times how far they went,
            # and three roundings a step
            err = float((w.double().cpu() - flat(ref[seg.name])).norm())
            assert err <= 15 * 2 ** -11 * change[seg.name] + 9 * 2 ** -24 * float(ref[seg.name].norm()) + 1e-12, seg.name
            torch.testing.assert_close(v.double().cpu(), flat(vel[seg.name]), rtol=1e-6, atol=1e-9)
            if dt in opt.master:
                assert torch.equal(opt.arena.params[dt][seg.offset:seg.offset + seg.numel], w.to(BF))
        assert not opt.momentum_buf[dt].cpu()[~covered].any() and not opt.arena.params[dt].cpu()[~covered].any()


def test_muon_frozen_lr_follows_the_schedule_bit_for_bit():
    from distributeddeeplearning_amd.optim import FusedMuon

    results = []
    for frozen in (False, True):
        named = _params(MUON_SHAPES, BF)
        opt = FusedMuon(named, lr=0.02, weight_decay=0.01)
        if frozen:
            opt.freeze_lr()
        for step, lr in enumerate((0.02, 0.013, 0.004)):
            opt.param_groups[0]["lr"] = lr
            opt.sync_lr()
            gen = torch.Generator().manual_seed(step)
            for _, p in named:
                p.grad.copy_(torch.randn(p.shape, generator=gen))
            opt.step()
        results.append([opt.master[BF].clone(), opt.arena.params[torch.float32].clone()])
    for a, b in zip(*results):
        assert torch.equal(a, b)


def _train(taped, graphed=False, steps=7):
    from distributeddeeplearning_amd.data.synthetic import DeviceSyntheticLoader
    from distributeddeeplearning_amd.models import resnet18
    from distributeddeeplearning_amd.ops import functional as ops, hip_ops
    from distributeddeeplearning_amd.optim import FusedMuon
    from distributeddeeplearning_amd.training.graph import GraphedTrainStep
    from distributeddeeplearning_amd.training.tape import TapedTrainStep

    hip_ops.reset_caches()
    torch.manual_seed(3)
    model = resnet18(num_classes=16).to_compute(torch.device(DEV), BF).train()
    opt = FusedMuon(model.named_parameters(), lr=0.01, momentum=0.9, weight_decay=1e-3)
    loader = DeviceSyntheticLoader(8, length=8 * 64, pool_size=32, height=64, width=64, n_classes=16, device=DEV, dtype=BF, seed=11)
    if graphed:
        step = GraphedTrainStep(model, opt, ops.softmax_cross_entropy, warmup=2)
    else:
        step = TapedTrainStep(model, opt, ops.softmax_cross_entropy, loader=loader, warmup=2, enabled=taped)
    for s in range(steps):
        if s == 4:
            opt.param_groups[0]["lr"] = 0.003
        if graphed:
            step(*loader.batch())
        else:
            step()
    torch.cuda.synchronize()
    return step, opt


def test_muon_step_on_the_launch_tape_is_the_eager_step():
    eager, a = _train(False)
    taped, b = _train(True)
    assert taped.taped and not eager.taped
    assert torch.equal(a.master[BF], b.master[BF]) and torch.equal(a.momentum_buf[BF], b.momentum_buf[BF])


def test_muon_step_in_a_captured_graph_is_the_eager_step():
    _, a = _train(False)
    graphed, b = _train(False, graphed=True)
    assert graphed.graphed
    assert torch.equal(a.master[BF], b.master[BF]) and torch.equal(a.momentum_buf[BF], b.momentum_buf[BF])


# ------------------------------------------------------------------------------------------ each of the kernels' forms
# A workgroup a matrix, the Gram matrix's steps (all up to 32 rows), tiles: sizes on both sides of their borders.
# Up to 32 rows the steps are fp64; the matrix that they make (entries up to 3.4445^5 = 485) is rounded to fp32 and multiplied with
# fp32 values in sums of 32 terms: 34 * 2^-24 * 485 = 2^-10 at most, and the rounding to bf16.
TOL_THIN = 2 ** -8 + 2 ** -10
THIN = [(1, 513), (1, 3157), (5, 100001), (16, 2304), (17, 2762), (2762, 17), (31, 1000), (32, 520), (700, 32), (32, 8193)]


@pytest.mark.parametrize("kind", ["gauss", "power", "exp", "rank1", "lowrank"])
@pytest.mark.parametrize("shape", THIN, ids=str)
def test_few_rows(shape, kind):
    from distributeddeeplearning_amd.ops import functional as ops

    for dtype in (torch.float32, BF):
        g = spectrum(kind, *shape, seed=7).to(DEV, dtype)
        assert off(ops.orthogonalize(g), g) < TOL_THIN


def test_few_rows_stacks_strides_and_lists():
    from distributeddeeplearning_amd.ops import functional as ops

    stack = spectrum("gauss", 21 * 9, 1400, 1).to(DEV).view(9, 21, 1400)
    for s in (stack, stack.transpose(1, 2), stack[::3, 2:, 1::2], stack[:1].expand(4, 21, 1400)):
        out = ops.orthogonalize(s)
        for k in range(s.shape[0]):
            assert off(out[k], s[k]) < TOL_THIN
    mats = [spectrum("gauss", 1 + i % 32, 513 + 37 * i, i).to(DEV) for i in range(80)]       # more than one call's groups
    for m, o in zip(mats, ops.orthogonalize([m.t() if i % 2 else m for i, m in enumerate(mats)])):
        assert off(o if o.shape == m.shape else o.t(), m) < TOL_THIN


@pytest.mark.parametrize("shape", [(32, 512), (33, 512), (64, 512), (64, 513), (65, 256), (128, 256), (128, 260), (129, 129), (200, 1111), (321, 4500)], ids=str)
@pytest.mark.parametrize("kind", ["gauss", "exp", "lowrank"])
def test_borders_between_the_forms(shape, kind):
    from distributeddeeplearning_amd.ops import functional as ops

    g = spectrum(kind, *shape, seed=8).to(DEV)
    assert off(ops.orthogonalize(g), g) < TOL
    assert off(ops.orthogonalize(g.t()), g.t()) < TOL


FORMS = [(40, 90), (20, 700), (200, 300)]


@pytest.mark.parametrize("shape", FORMS, ids=str)
@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e30])
def test_magnitudes_in_each_form(shape, scale):
    from distributeddeeplearning_amd.ops import functional as ops

    g = (spectrum("gauss", *shape, 3) * scale).to(DEV)
    assert off(ops.orthogonalize(g, eps=1e-20), g, eps=1e-20) < TOL


@pytest.mark.parametrize("shape", FORMS, ids=str)
def test_matrices_do_not_touch_each_other_in_each_form(shape):
    from distributeddeeplearning_amd.ops import functional as ops

    clean = [spectrum("gauss", *shape, i).to(DEV) for i in range(4)]
    want = ops.orthogonalize(clean)
    bad = [m.clone() for m in clean]
    bad[1][3, 4] = float("nan")
    bad[2][-1, -1] = float("inf")
    bad.insert(1, torch.zeros(shape, device=DEV))
    got = ops.orthogonalize(bad)
    assert torch.equal(got[0], want[0]) and torch.equal(got[4], want[3])
    assert not got[1].any() and got[2].isnan().all() and got[3].isnan().all()


@pytest.mark.parametrize("shape", FORMS, ids=str)
@pytest.mark.parametrize("steps, coef", [(1, (3.4445, -4.7750, 2.0315)), (7, (3.4445, -4.7750, 2.0315)), (10, (2.0, -1.5, 0.5)), (3, (1.5, -0.5, 0.0))])
def test_steps_and_coefficients_in_each_form(shape, steps, coef):
    from distributeddeeplearning_amd.ops import functional as ops

    g = spectrum("gauss", *shape, 2).to(DEV)
    assert off(ops.orthogonalize(g, steps=steps, coefficients=coef), g, steps=steps, coef=coef) < 2 ** -8 + 3 * steps * 2 ** -11


def on_the_card(g, steps=5):
    """The steps themselves in 64 bits, for sizes whose singular values take too long."""
    x = g.double()
    x = x / x.norm()
    a, b, c = 3.4445, -4.7750, 2.0315
    x = x.t().contiguous() if x.shape[0] > x.shape[1] else x
    for _ in range(steps):
        aa = torch.mm(x, x.t().contiguous())
        x = a * x + torch.mm(b * aa + c * torch.mm(aa, aa), x)
    return x if x.shape == g.shape else x.t()


# tiles of 128 in P X; of 128 in A and A^2 too; of 256 in all (odd sizes; tall)
@pytest.mark.parametrize("shapes", [[(2040, 2001)], [(2048, 4096), (4001, 2000), (1000, 4090)], [(4000, 8100)], [(8191, 4001)]], ids=str)
def test_larger_tiles(shapes):
    from distributeddeeplearning_amd.ops import functional as ops

    gen = torch.Generator(DEV).manual_seed(4)
    mats = [torch.randn(s, generator=gen, device=DEV) * torch.logspace(0, -4, s[1], device=DEV) for s in shapes]
    for m, o in zip(mats, ops.orthogonalize(mats)):
        want = on_the_card(m)
        assert float((o.double() - want).norm() / want.norm()) < TOL


@pytest.mark.parametrize("shapes", [[(8, 16), (64, 300), (300, 64), (100, 250), (127, 127), (1, 1)], [(16, 3, 7, 7), (16, 64, 3, 3), (700, 30), (5, 2000)],
                                    [(4000, 8100)]], ids=["small", "few-rows", "large"])
@pytest.mark.parametrize("dtype", [BF, torch.float32], ids=["bf16", "fp32"])
def test_muon_in_each_form(shapes, dtype):
    from distributeddeeplearning_amd.optim import FusedMuon

    large = max(max(s) for s in shapes) > 4000
    named = _params(shapes if large else shapes * 12, dtype)
    opt = FusedMuon(named, lr=0.02, momentum=0.9, weight_decay=0.05)
    ref = {n: p.detach().double().clone() for n, p in named}
    vel = {n: torch.zeros_like(w) for n, w in ref.items()}
    change = {n: 0.0 for n in ref}
    for step in range(2):
        gen = torch.Generator(DEV).manual_seed(step)
        for n, p in named:
            p.grad.copy_(1e-3 * torch.randn(p.shape, generator=gen, device=DEV))
            before, g = ref[n].clone(), p.grad.double()
            vel[n].mul_(0.9).add_(g)
            u = (g + 0.9 * vel[n]).flatten(1)
            o = (on_the_card(u) if large else oracle(u.cpu()).to(DEV)).reshape(g.shape)
            ref[n].mul_(1 - 0.02 * 0.05).sub_(o, alpha=0.02 * max(1.0, u.shape[0] / u.shape[1]) ** 0.5)
            change[n] += float((ref[n] - before).norm())
        opt.step()
    for seg in opt.arena.plans[dtype].segments:
        w = opt._weights(dtype)[seg.offset:seg.offset + seg.numel].double()
        r = ref[seg.name]
        r = (r.permute(0, 2, 3, 1) if r.dim() == 4 else r).reshape(-1)
        assert float((w - r).norm()) <= 15 * 2 ** -11 * change[seg.name] + 9 * 2 ** -24 * float(r.norm()) + 1e-12, seg.name


def test_captured_in_each_form():
    from distributeddeeplearning_amd.ops import functional as ops

    xs = [torch.randn(s, device=DEV) for s in FORMS + [(3, 31, 600), (1030, 2050)]]
    graphs, outs = [], []
    for x in xs:
        ops.orthogonalize(x)
    torch.cuda.synchronize()
    for x in xs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.orthogonalize(x))
        graphs.append(gr)
    side = torch.cuda.Stream()
    for rep in range(4):
        for x in xs:
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(rep)))
        for gr in graphs if rep % 2 else graphs[::-1]:
            gr.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = [ops.orthogonalize(x) for x in xs]
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        for o, e in zip(outs, eager):
            assert torch.equal(o, e)


def test_trained_with_muon_and_served_with_the_8_bit_head():
    """Both together, as a user has them: some steps, then answers from the head's codes of the trained weights."""
    from tests.test_int8_linear import check
    from distributeddeeplearning_amd.ops import functional as ops

    step, opt = _train(False)
    model = step.model.eval()
    x = torch.randn(5, 3, 64, 64, device=DEV).to(BF).contiguous(memory_format=torch.channels_last)
    seen = []
    with torch.no_grad():
        model.fc.register_forward_hook(lambda mod, args, out: seen.append(args[0]))
        model(x)
        w, b = model.fc.weight.detach().clone(), model.fc.bias.detach().clone()
        got = model.int8_head()(x)
    check(got, seen[0], *ops.quantize_int8(w), b)


# stacks of more than 2^31 values, in each form: the last matrix is the one that it is alone (another form's launch for the tiles
# of a large one: both within the tolerance)
@pytest.mark.parametrize("shape", [(300000, 64, 128), (70000, 32, 1024), (140000, 130, 120)], ids=str)
def test_offsets_beyond_32_bits(shape):
    from distributeddeeplearning_amd.ops import functional as ops

    x = torch.zeros(shape, dtype=BF, device=DEV)
    g = spectrum("gauss", *shape[1:]).to(DEV, BF)
    for k in (0, shape[0] // 2, shape[0] - 1):
        x[k] = g
    out = ops.orthogonalize(x)
    assert not out[1].any() and not out[shape[0] - 2].any()
    for k in (0, shape[0] // 2, shape[0] - 1):
        assert off(out[k], g) < TOL


# sums of X X^T that are cut into parts: one tile, several of them ragged, more groups than CUs, stacks; fp16 rounds as elsewhere
@pytest.mark.parametrize("shapes", [[(64, 6144 + 13)], [(33, 100001)], [(9001, 100), (300, 12345), (40, 7000), (70, 50)], [(3, 65, 9000), (2, 40, 64 * 191)],
                                    [(500, 6200), (20, 30000), (640, 700), (64, 64)]], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, BF], ids=["fp32", "bf16"])
def test_long_rows(shapes, dtype):
    from distributeddeeplearning_amd.ops import functional as ops

    gen = torch.Generator(DEV).manual_seed(9)
    mats = []
    for s in shapes:
        x = torch.randn(s, generator=gen, device=DEV) * torch.logspace(0, -3, s[-1], device=DEV)
        mats += [m.to(dtype) for m in (x if len(s) == 3 else x[None])]
    if len(shapes[0]) == 3:
        outs = [o for k in (0, 3) for o in ops.orthogonalize(torch.stack(mats[k:k + 3 - k // 3]))]
    else:
        outs = ops.orthogonalize(mats)
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(outs, ops.orthogonalize(mats)))
    for m, o in zip(mats, outs):
        want = on_the_card(m)
        assert float((o.double() - want).norm() / want.norm()) < TOL


def test_long_rows_in_graphs_and_in_the_optimizer():
    from distributeddeeplearning_amd.ops import functional as ops
    from distributeddeeplearning_amd.optim import FusedMuon

    xs = [torch.randn(130, 8000, device=DEV), torch.randn(2, 50, 20000, device=DEV)]
    graphs, outs = [], []
    for x in xs:
        ops.orthogonalize(x)
    torch.cuda.synchronize()
    for x in xs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.orthogonalize(x))
        graphs.append(gr)
    for rep in range(4):
        for x in xs:
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(rep)))
        for gr in graphs if rep % 2 else graphs[::-1]:
            gr.replay()
        eager = [ops.orthogonalize(x) for x in xs]
        torch.cuda.synchronize()
        for o, e in zip(outs, eager):
            assert torch.equal(o, e)
    # the step is the operator's: w - lr sqrt(max(1, r / c)) O, O in fp32 there (half a bf16 step, 2^-8, from the operator's)
    named = _params([(130, 8000), (20000, 50)], torch.float32)
    opt = FusedMuon(named, lr=1.0, momentum=0.0, nesterov=False)
    before = [p.detach().clone() for _, p in named]
    for _, p in named:
        p.grad.copy_(torch.randn(p.shape, generator=torch.Generator(DEV).manual_seed(5), device=DEV))
    wants = [w - max(1.0, w.shape[0] / w.shape[1]) ** 0.5 * ops.orthogonalize(p.grad).float() for w, (_, p) in zip(before, named)]
    opt.step()
    for (_, p), w, b in zip(named, wants, before):
        assert float((p.detach() - w).norm()) <= 2 ** -8 * float((w - b).norm()) + 2 ** -22 * float(b.norm())


# the largest sizes that a workgroup holds, the next ones, and those that the Gram matrix's form takes before
@pytest.mark.parametrize("shape", [(64, 576), (33, 577), (64, 768), (50, 767), (64, 769), (128, 257), (65, 384), (128, 384), (127, 383), (128, 385), (129, 384),
                                   (16, 256), (16, 257), (17, 512), (17, 513), (300, 64, 600), (260, 20, 300), (260, 16, 300), (3, 100, 380)], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, BF], ids=["fp32", "bf16"])
def test_borders_of_one_workgroup(shape, dtype):
    from distributeddeeplearning_amd.ops import functional as ops

    for kind in ("gauss", "exp"):
        g = spectrum(kind, *shape[-2:], seed=10).to(DEV, dtype)
        x = g if len(shape) == 2 else torch.stack([g * (k + 1) for k in range(shape[0])])
        for y in (x, x.transpose(-2, -1), x.transpose(-2, -1).contiguous()):
            out = ops.orthogonalize(y)
            for k in (0,) if len(shape) == 2 else (0, 1, shape[0] - 1):
                o, v = (out, y) if len(shape) == 2 else (out[k], y[k])
                assert off(o, v) < TOL


# one size for all: lists whose rows, columns and classes differ; more than one launch's groups
@pytest.mark.parametrize("shapes", [[(64, 147), (64, 64), (64, 576), (256, 64), (64, 256)], [(64, 147), (128, 64), (100, 300), (5, 5), (384, 1)],
                                    [(100, 100), (64, 700)], [(16, 256), (3, 2)], [(16, 300), (64, 64)], [(9 + i, 700 - 8 * i) for i in range(50)]], ids=str)
def test_lists_of_small_matrices(shapes):
    from distributeddeeplearning_amd.ops import functional as ops
    from distributeddeeplearning_amd.optim import FusedMuon

    mats = [spectrum("power", *s, seed=i).to(DEV) for i, s in enumerate(shapes)]
    outs = ops.orthogonalize(mats)
    for m, o in zip(mats, outs):
        assert off(o, m) < TOL
    named = _params(shapes, torch.float32)
    opt = FusedMuon(named, lr=1.0, momentum=0.0, nesterov=False)
    before = [p.detach().clone() for _, p in named]
    for (_, p), m in zip(named, mats):
        p.grad.copy_(m)
    opt.step()
    # the operator's result before its rounding to bf16: half a step, 2^-8, from it
    for (_, p), w, o in zip(named, before, outs):
        want = w - max(1.0, w.shape[0] / w.shape[1]) ** 0.5 * o.float()
        assert float((p.detach() - want).norm()) <= 2 ** -8 * float((want - w).norm()) + 2 ** -22 * float(w.norm())


@pytest.mark.parametrize("dtype", [torch.float32, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(40, 90), (20, 700), (200, 301), (300, 200), (3, 130, 201)], ids=str)
def test_arrays_that_start_anywhere(shape, dtype):
    from distributeddeeplearning_amd.ops import functional as ops

    n = math.prod(shape)
    x = torch.randn(n, generator=torch.Generator().manual_seed(3)).to(DEV, dtype)
    want = ops.orthogonalize(x.view(shape))
    store = torch.full((n + 16,), float("nan"), device=DEV, dtype=dtype)
    for at in (1, 4, 7):
        store.fill_(float("nan"))
        store[at:at + n] = x
        got = ops.orthogonalize(store[at:at + n].view(shape))
        for w, o, v in zip(want.view(-1, *shape[-2:]), got.view(-1, *shape[-2:]), x.view(-1, *shape[-2:])):
            assert off(o, v) < TOL and off(w, v) < TOL


def test_matrices_that_are_too_large_are_refused():
    from distributeddeeplearning_amd.ops import functional as ops
    from distributeddeeplearning_amd.ops.kernels import KernelError
    from distributeddeeplearning_amd.optim import FusedMuon

    g = torch.zeros(32705, 32705, dtype=BF, device=DEV)          # rounded up to 64: 32768^2 = 2^30
    with pytest.raises(KernelError, match="out of range"):
        ops.orthogonalize(g)
    with pytest.raises(KernelError, match="out of range"):
        FusedMuon([("w", torch.nn.Parameter(g))])


# What the steps' roundings may leave, before the result's own to bf16: each step rounds X_hi, offdiag(A) and offdiag(P) to fp16, at most
# 2^-11 of a value each, 2^-11 / sqrt(3) in the mean of many; a value's error enters by P - a (|b s^2 + c s^4| < 3 here) and is not
# amplified by the later steps, whatever the spectrum; 15 independent ones: sqrt(15) 3 2^-11 / sqrt(3).  Of few values: without the mean.
def direction_limit(shape):
    return math.sqrt(15) * 3 * 2 ** -11 / (math.sqrt(3) if min(shape) >= 16 else 1)


@pytest.mark.parametrize("shape, kind", [(s, k) for k in ["gauss", "power", "exp", "rank1", "lowrank"] for s in
                                         [(2, 8), (2, 64), (4, 64), (64, 3), (8, 256), (16, 256), (32, 512), (64, 64), (64, 768), (768, 64), (33, 1000), (128, 384),
                                          (1000, 40), (129, 300), (256, 1024), (520, 512)] + ([(2040, 2001)] if k in ("gauss", "rank1") else [])], ids=str)
def test_the_direction_of_any_spectrum(shape, kind):
    """The fp32 weights that a step from zero leaves: the direction itself, in each form."""
    from distributeddeeplearning_amd.ops import functional as ops
    from distributeddeeplearning_amd.optim import FusedMuon

    p = torch.nn.Parameter(torch.zeros(shape, device=DEV))
    opt = FusedMuon([("w", p)], lr=1.0, momentum=0.0, nesterov=False)
    g = spectrum(kind, *shape, seed=11).to(DEV)
    p.grad.copy_(g)
    opt.step()
    want = -max(1.0, shape[0] / shape[1]) ** 0.5 * (on_the_card(g) if max(shape) > 2000 else oracle(g.cpu()).to(DEV))
    err = float((p.detach().double() - want).norm() / want.norm())
    assert err < direction_limit(shape), err
    out = ops.orthogonalize(g.to(BF))                 # a bf16 input has a spectrum of its own
    want = on_the_card(g.to(BF)) if max(shape) > 2000 else oracle(g.to(BF).cpu()).to(DEV)
    assert float((out.double() - want).norm() / want.norm()) < direction_limit(shape) + 2 ** -8


@pytest.mark.parametrize("scale", [0.3, 1.7, 0.0])
def test_muon_frozen_lr_with_a_scale_for_vectors_is_bit_identical(scale):
    """As test_muon_frozen_lr_follows_the_schedule_bit_for_bit, with scales whose product with the learning rate has to be rounded."""
    from distributeddeeplearning_amd.optim import FusedMuon

    results = []
    for frozen in (False, True):
        named = _params(MUON_SHAPES, BF)
        opt = FusedMuon(named, lr=0.02, weight_decay=0.01, vector_lr_scale=scale)
        for step, lr in enumerate((0.02, 0.013, 0.0041, 0.0007)):
            opt.param_groups[0]["lr"] = lr
            opt.param_groups[0]["vector_lr_scale"] = scale if step < 3 else 0.9
            if frozen:
                opt.freeze_lr() if step == 1 else opt.sync_lr()
            gen = torch.Generator().manual_seed(step)
            for _, p in named:
                p.grad.copy_(torch.randn(p.shape, generator=gen))
            opt.step()
        results.append([opt.master[BF].clone(), opt.arena.params[torch.float32].clone()])
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_a_refused_optimizer_leaves_the_parameters_where_they_were():
    from distributeddeeplearning_amd.ops.kernels import KernelError
    from distributeddeeplearning_amd.optim import FusedMuon

    small = torch.nn.Parameter(torch.ones(4, 4, device=DEV))
    large = torch.nn.Parameter(torch.zeros(1, 1 << 24, dtype=BF, device=DEV))       # rounded up to 64 rows: 2^30
    at = small.data_ptr(), large.data_ptr()
    with pytest.raises(KernelError, match="out of range"):
        FusedMuon(p for p in [("a", small), ("b", large)])
    assert (small.data_ptr(), large.data_ptr()) == at and small.grad is None and large.grad is None


# more equal matrices than a launch takes: 2^20 of one tile a call, fewer of more tiles
@pytest.mark.parametrize("shape", [(4_300_000, 4, 4), (300_000, 2, 900), (60_000, 130, 960)], ids=str)
def test_stacks_of_more_matrices_than_a_launch_takes(shape):
    from distributeddeeplearning_amd.ops import functional as ops, kernels

    most = kernels.ortho_most_matrices(*shape[1:])
    assert most < shape[0]
    x = torch.zeros(shape, dtype=BF, device=DEV)
    g = spectrum("gauss", *shape[1:]).to(DEV, BF)
    at = [0, most - 1, most, 2 * most - 1, shape[0] - 1]
    at = [k for k in at if k < shape[0]]
    for k in at:
        x[k] = g
    out = ops.orthogonalize(x)
    assert out.shape == x.shape
    for k in at:
        assert off(out[k], g) < TOL
    assert int(out.flatten(1).any(1).sum()) == len(at)
    every = ops.orthogonalize(g.expand(shape))            # a stack of strides 0
    assert torch.equal(every[shape[0] - 1], out[0]) and torch.equal(every[most - 1], every[0])


def test_the_most_matrices_of_a_call_are_within_the_launches():
    from distributeddeeplearning_amd.ops import kernels

    for r, c in ((1, 1), (64, 64), (65, 1), (1, 1000), (33, 1 << 20), (1000, 1000), (128, 130000), (32000, 32000), (1, 1 << 23), (4000, 100000)):
        n = kernels.ortho_most_matrices(r, c)
        assert kernels.ortho_workspace_of(((r, c, n),)) >= 0 and kernels.ortho_workspace_of(((c, r, n),)) >= 0


def test_a_stride_that_is_never_taken_may_be_anything():
    from distributeddeeplearning_amd.ops import functional as ops

    x = torch.randn(700, generator=torch.Generator().manual_seed(1)).to(DEV)
    for size, strides in (((1, 700), (1 << 31, 1)), ((700, 1), (1, 1 << 40)), ((1, 1), (1 << 33, 1 << 33)), ((1, 1, 700), (1 << 50, 1 << 31, 1)),
                          ((7, 1, 100), (100, 1 << 31, 1)), ((1, 7, 100), (1 << 40, 100, 1))):
        v = x.as_strided(size, strides)
        assert torch.equal(ops.orthogonalize(v), ops.orthogonalize(v.clone(memory_format=torch.contiguous_format)))


# Up to 32 rows the direction is Q X_0 in fp32, a sum of up to 32 terms whose two factors are rounded: 34 * 2^-24 |Q| |X_0| with |Q| <= 3.4445^5 = 485
# and |X_0| = 1, against a result of 0.68 at least in its largest direction.  (Q's own error: 2^-53 * 485^2.)
FEW_LIMIT = 34 * 485 * 2 ** -24 / 0.68
FEW = [(2, 8), (8, 2), (2, 64), (3, 16), (4, 64), (5, 9), (16, 16), (16, 512), (16, 513), (17, 256), (17, 257), (32, 256), (32, 700), (700, 30), (31, 3000)]
BESIDE = {"alone": [], "small": [(64, 147), (100, 90)], "tiles": [(300, 200), (40, 900)]}


def directions(mats):
    """fp32 directions of one FusedMuon step from zero, all in one call."""
    from distributeddeeplearning_amd.optim import FusedMuon

    ps = [torch.nn.Parameter(torch.zeros(m.shape, device=DEV)) for m in mats]
    opt = FusedMuon([("w%d" % i, p) for i, p in enumerate(ps)], lr=1.0, momentum=0.0, nesterov=False)
    for p, m in zip(ps, mats):
        p.grad.copy_(m)
    opt.step()
    return [-p.detach() / max(1.0, p.shape[0] / p.shape[1]) ** 0.5 for p in ps]


@pytest.mark.parametrize("beside", sorted(BESIDE))
@pytest.mark.parametrize("kind", ["gauss", "rank1", "exp"])
def test_few_rows_keep_their_digits_in_any_call(kind, beside):
    from distributeddeeplearning_amd.ops import functional as ops

    small = [s for s in FEW if max(s) <= (512 if min(s) <= 16 else 256)]
    for shapes in ([[s] for s in FEW] if beside == "alone" else []) + [FEW, small]:
        mats = [spectrum(kind, *s, seed=i).to(DEV) for i, s in enumerate(shapes + BESIDE[beside])]
        for m, d, o in zip(mats, directions(mats), ops.orthogonalize(mats)):
            want = oracle(m.cpu()).to(DEV)
            limit = FEW_LIMIT if min(m.shape) <= 32 else direction_limit(m.shape)
            assert float((d.double() - want).norm() / want.norm()) < limit, tuple(m.shape)
            assert float((o.double() - want).norm() / want.norm()) < limit + 2 ** -8, tuple(m.shape)


@pytest.mark.parametrize("beside", [[], [(64, 147)], [(300, 200)], [(300, 200), (5, 40)]], ids=str)
def test_one_row_keeps_its_digits_in_any_call(beside):
    # beside larger ones: A is a sum of squares of values rounded to fp16, off by 2 * 2^-11 / sqrt(3) sqrt(3 / 300) = 5.6e-5 of it in the mean; a
    # step's factor a + b A + c A^2 by 0.71 of that (A near 1), five of them added up: 2e-4 of a result of 0.7
    shapes = [(1, 300), (2000, 1), (1, 1), (1, 5000)]
    mats = [spectrum("gauss", *s, seed=i).to(DEV) for i, s in enumerate(shapes + beside)]
    for m, d in list(zip(mats, directions(mats)))[:4]:
        want = oracle(m.cpu()).to(DEV)
        limit = 3e-4 * max(1.0, (300 / max(m.shape)) ** 0.5) if beside else FEW_LIMIT
        assert float((d.double() - want).norm() / want.norm()) < limit, tuple(m.shape)


def test_stacks_of_few_rows():
    """A matrix for each CU: one launch whatever the length; beside strides."""
    from distributeddeeplearning_amd.ops import functional as ops

    for dtype in (torch.float32, BF):
        x = spectrum("gauss", 300 * 20, 1100, 3).to(DEV, dtype).view(300, 20, 1100)
        for s in (x, x.transpose(1, 2), x[:, 3:, 1::2], x[:1].expand(260, 20, 1100)):
            out = ops.orthogonalize(s)
            for k in (0, 1, s.shape[0] - 1):
                want = oracle(s[k].cpu()).to(DEV)
                assert float((out[k].double() - want).norm() / want.norm()) < FEW_LIMIT + 2 ** -8


ONE_LAUNCH = [(20, 100), (5, 9), (1, 300), (16, 512), (300, 31, 40)]


@pytest.mark.parametrize("shape", ONE_LAUNCH, ids=str)
def test_few_rows_that_are_zero_tiny_huge_or_not_finite(shape):
    from distributeddeeplearning_amd.ops import functional as ops

    r, c = shape[-2:]
    clean = [spectrum("gauss", r, c, i).to(DEV) for i in range(4)]
    want = ops.orthogonalize(clean)
    bad = [m.clone() for m in clean]
    bad[1][0, c // 2] = float("nan")
    bad[2][-1, -1] = float("inf")
    bad.insert(1, torch.zeros(r, c, device=DEV))
    many = shape[0] // len(bad) if len(shape) == 3 else 1                # (a stack: its own form)
    got = ops.orthogonalize(torch.stack(bad * many)) if many > 1 else ops.orthogonalize(bad)
    for k in range(0, len(got), 5):
        assert torch.equal(got[k], want[0]) and torch.equal(got[k + 4], want[3])
        assert not got[k + 1].any() and got[k + 2].isnan().all() and got[k + 3].isnan().all()
    for scale in (1e-38, 1e-30, 1e-12, 1e30, 1e37):
        g = clean[0] * scale
        assert off(ops.orthogonalize(g, eps=1e-20), g, eps=1e-20) < FEW_LIMIT + 2 ** -8
    for steps, coef in ((1, (3.4445, -4.7750, 2.0315)), (10, (2.0, -1.5, 0.5)), (3, (1.5, -0.5, 0.0))):
        assert off(ops.orthogonalize(clean[0], steps=steps, coefficients=coef), clean[0], steps=steps, coef=coef) < FEW_LIMIT + 2 ** -8
