"""The dense layer on 8-bit integers: CPU path, refusals, the model's 8-bit head."""
import pytest
import torch

from distributeddeeplearning_amd.ops import functional as ops


def rows_oracle(x):
    """Codes and scales in the stated arithmetic (fp32, one rounding an operation), row by row."""
    x = x.detach().float().cpu()
    q, s = torch.zeros(x.shape, dtype=torch.int8), torch.zeros(x.shape[0])
    for i, row in enumerate(x):
        top = row.abs().max()
        if not torch.isfinite(row).all():
            s[i] = float("nan")
        elif top >= 1e-30:
            s[i] = top / 127.0
            q[i] = torch.round(row * (127.0 * top.reciprocal())).to(torch.int8)
    return q, s


def product_oracle(x, q, scale, bias):
    """64 bits, from the codes of the stated arithmetic; and the sum of magnitudes that its fp32 evaluation rounds."""
    xq, sx = rows_oracle(x.reshape(-1, x.shape[-1]))
    acc = xq.double() @ q.cpu().double().t()
    y = acc * sx.double()[:, None] * scale.cpu().double()[None]
    mag = y.abs()
    if bias is not None:
        y, mag = y + bias.cpu().double(), mag + bias.cpu().double().abs()
    return y, mag


def check(y, x, q, scale, bias):
    want, mag = product_oracle(x, q, scale, bias)
    got = y.detach().double().cpu().reshape(want.shape)
    assert torch.equal(got.isnan(), want.isnan())
    # fp32: the sum's conversion, two products of scales and the addition, half a step (2^-24) each; bf16: half a step more (2^-8)
    tol = 4 * 2 ** -24 * mag + 1e-37
    if y.dtype == torch.bfloat16:
        tol = tol + 2 ** -8 * (want.abs() + tol)
    over = want.abs() > torch.finfo(y.dtype).max * (1 + 2 ** -8)     # beyond the type: rounds to an infinity
    assert torch.equal(got[over], want[over].sign() * float("inf"))
    assert bool(((got - want).abs() <= tol)[~want.isnan() & ~over].all())


@pytest.mark.parametrize("shape", [(1, 1), (3, 64), (5, 65), (2, 1000)])
def test_quantize(shape):
    gen = torch.Generator().manual_seed(0)
    w = torch.randn(shape, generator=gen)
    q, s = ops.quantize_int8(w)
    qo, so = rows_oracle(w)
    assert torch.equal(q, qo) and torch.equal(s, so) and q.stride(0) % 64 == 0
    # half a code: scale / 2 (and the fp32 roundings of the quotient)
    assert bool(((q.float() * s[:, None] - w).abs() <= s[:, None] * (0.5 + 127 * 2 ** -22)).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bias", [True, False])
def test_cpu_product(dtype, bias):
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(2, 3, 70, generator=gen).to(dtype)
    x[0, 1], x[1, 0, 3], x[1, 1, 2] = 0.0, float("nan"), float("inf")
    q, s = ops.quantize_int8(torch.randn(9, 70, generator=gen))
    b = torch.randn(9, generator=gen) if bias else None
    y = ops.linear_int8(x, q, s, b)
    assert y.shape == (2, 3, 9) and y.dtype == dtype
    check(y, x, q, s, b)
    assert ops.linear_int8(x[:0], q, s, b).shape == (0, 3, 9)


def _args():
    return [torch.zeros(2, 8), torch.zeros(3, 8, dtype=torch.int8), torch.zeros(3), torch.zeros(3)]


@pytest.mark.parametrize("index, value, text", [
    (0, torch.zeros(2, 8, dtype=torch.float16), "fp32 or bf16"),
    (0, torch.zeros(2, 8, dtype=torch.int8), "fp32 or bf16"),
    (0, torch.tensor(1.0), "fp32 or bf16"),
    (0, torch.zeros(2, 7), "codes"),
    (0, torch.zeros(2, 8, requires_grad=True), "gradient"),
    (1, torch.zeros(3, 8), "codes"),
    (1, torch.zeros(8, dtype=torch.int8), "codes"),
    (2, torch.zeros(4), "scale"),
    (2, torch.zeros(3, dtype=torch.bfloat16), "scale"),
    (3, torch.zeros(3, 1), "bias"),
    (3, torch.zeros(3, requires_grad=True), "gradient"),
])
def test_refusals(index, value, text):
    args = _args()
    args[index] = value
    with pytest.raises(ValueError, match=text):
        ops.linear_int8(*args)


def test_refusals_of_sizes():
    with pytest.raises(ValueError, match="codes"):
        ops.linear_int8(torch.zeros(1, 133145), torch.zeros(1, 133145, dtype=torch.int8), torch.zeros(1))
    with pytest.raises(ValueError, match="codes"):
        ops.linear_int8(torch.zeros(1, 0), torch.zeros(1, 0, dtype=torch.int8), torch.zeros(1))
    for w in (torch.zeros(3), torch.zeros(3, 0), torch.zeros(3, 3, dtype=torch.int8)):
        with pytest.raises(ValueError, match="quantize_int8"):
            ops.quantize_int8(w)


def test_int8_head_of_a_model():
    from distributeddeeplearning_amd.models import resnet18

    torch.manual_seed(0)
    model = resnet18(num_classes=12).eval()
    x = torch.randn(2, 3, 32, 32)
    with torch.no_grad():
        want = model(x)
        w, b = model.fc.weight.detach().clone(), model.fc.bias.detach().clone()
        got = model.int8_head()(x)
        feats = ops.global_avgpool(model._trunk(ops.stem(x, model.conv1.weight, 2, 3, model.bn1.weight, model.bn1.bias, model.bn1.running_mean,
                                                         model.bn1.running_var, False)))
    check(got, feats, *ops.quantize_int8(w), b)
    # half a code of each weight and of each feature: |f| (s_w / 2) + |w| (s_f / 2) summed, and their product
    sw, sf = w.abs().amax(1) / 127, feats.abs().amax(1, keepdim=True) / 127
    tol = 0.51 * (feats.abs().sum(1, keepdim=True) * sw + sf * w.abs().sum(1) + w.shape[1] * sf * sw)
    assert bool(((got - want).abs() <= tol).all())
    assert "fc.codes" in model.state_dict() and "fc.weight" not in model.state_dict()
    other = resnet18(num_classes=12).int8_head()
    other.load_state_dict(model.state_dict())
    with torch.no_grad():
        assert torch.equal(other(x), got)


def test_int8_head_twice_is_the_same_head():
    from distributeddeeplearning_amd.models import resnet18

    model = resnet18(num_classes=12).int8_head()
    head = model.fc
    assert model.int8_head().fc is head


def test_arguments_that_the_kernels_refuse():
    """The library's own checks: before anything is launched, so they need no GPU."""
    import ctypes as c

    from distributeddeeplearning_amd.ops import kernels, native

    if not native.kernels_available():
        pytest.skip("kernel library not built")
    lib = kernels.lib()

    def rows(x=64, ldx=64, m=4, k=64, kp=64, q=64, scale=64):
        return lib.ddl_int8_rows(c.c_void_p(x), c.c_int(1), c.c_longlong(ldx), c.c_longlong(m), c.c_int(k), c.c_int(kp), c.c_void_p(q), c.c_void_p(scale),
                                 c.c_void_p(0))

    for kw in (dict(x=0), dict(q=0), dict(scale=0), dict(m=-1), dict(m=1 << 31), dict(k=0), dict(kp=48), dict(kp=72), dict(ldx=-1), dict(q=72)):
        assert rows(**kw) != 0, kw
    assert rows(m=0) == 0

    def product(x=64, ldx=64, q=64, ldq=64, q_bytes=640, s=64, bias=0, y=64, ldy=10, m=20, n=10, k=64, ws=256, nbytes=1 << 40):
        return lib.ddl_int8_linear(c.c_void_p(x), c.c_int(1), c.c_longlong(ldx), c.c_void_p(q), c.c_longlong(ldq), c.c_longlong(q_bytes), c.c_void_p(s),
                                   c.c_void_p(bias), c.c_void_p(y), c.c_longlong(ldy), c.c_longlong(m), c.c_int(n), c.c_int(k), c.c_void_p(ws),
                                   c.c_longlong(nbytes), c.c_void_p(0))

    for kw in (dict(x=0), dict(q=0), dict(s=0), dict(y=0), dict(m=-1), dict(m=1 << 31), dict(n=-1), dict(k=0), dict(k=133145, ldq=133152, q_bytes=1 << 40),
               dict(ldq=48), dict(ldq=72), dict(ldq=1 << 22, q_bytes=1 << 40), dict(q=72), dict(y=72), dict(ws=64), dict(ws=0), dict(nbytes=100),
               dict(q_bytes=639), dict(ldy=9), dict(ldx=-1), dict(m=1 << 30, n=1 << 30, ldy=1 << 30, q_bytes=1 << 50)):
        assert product(**kw) != 0, kw
    assert product(m=0) == 0 and product(n=0) == 0


def test_dual_tensors_are_refused():
    """Forward-mode differentiation: nothing is passed by silently."""
    from torch.autograd import forward_ad

    x, w, b = torch.randn(3, 8), torch.randn(5, 8), torch.randn(5)
    q, s = ops.quantize_int8(w)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual
        for args in ((dual(x, x), q, s, b), (x, q, dual(s, s), b), (x, q, s, dual(b, b))):
            with pytest.raises(ValueError, match="tangent"):
                ops.linear_int8(*args)
        assert torch.equal(ops.linear_int8(x, q, s, b), ops.linear_int8(forward_ad.unpack_dual(dual(x, x)).primal, q, s, b))
        codes, scale = ops.quantize_int8(dual(w, w))
        assert forward_ad.unpack_dual(scale).tangent is None and torch.equal(codes, q)
        for m in (dual(x, x), [w, dual(x, x)]):
            with pytest.raises(ValueError, match="tangent"):
                ops.orthogonalize(m)
    with pytest.raises(ValueError, match="tangent"):
        torch.func.jvp(lambda t: ops.linear_int8(t, q, s, b), (x,), (x,))
    with pytest.raises(ValueError, match="tangent"):
        torch.func.jvp(ops.orthogonalize, (x,), (x,))


@pytest.mark.parametrize("move", [lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.double().float(), lambda m: m.bfloat16().cpu()],
                         ids=["bf16", "half", "double-float", "bf16-cpu"])
@pytest.mark.parametrize("bias", [True, False])
def test_the_layer_keeps_its_scales_when_it_is_moved_to_another_type(move, bias):
    from distributeddeeplearning_amd.models import Int8Linear

    gen = torch.Generator().manual_seed(2)
    linear = torch.nn.Linear(70, 9, bias=bias)
    linear.weight.data = torch.randn(9, 70, generator=gen)
    layer, x = Int8Linear.from_linear(linear), torch.randn(4, 70, generator=gen)
    want = layer(x)
    moved = move(torch.nn.Sequential(layer))
    assert moved[0].scale.dtype == torch.float32 and torch.equal(moved(x), want)
    assert moved(x.to(torch.bfloat16)).dtype == torch.bfloat16


def test_int8_head_from_the_masters():
    """The codes of the fp32 weights that the optimizer holds, not of their bf16 copy."""
    from distributeddeeplearning_amd.models import Int8Linear, resnet18
    from distributeddeeplearning_amd.optim import FusedMuon

    torch.manual_seed(0)
    model = resnet18(num_classes=12).to_compute("cpu", torch.bfloat16)
    opt = FusedMuon(model.named_parameters(), lr=0.01)
    for _, p in model.named_parameters():
        p.grad.copy_(torch.randn(p.shape))
    opt.step()
    masters = opt.master_state_dict(model)
    q, s = ops.quantize_int8(masters["fc.weight"])
    rounded = ops.quantize_int8(model.fc.weight)
    assert not torch.equal(s, rounded[1])
    with pytest.raises(ValueError, match="fit"):
        Int8Linear.from_linear(model.fc, masters["fc.weight"][:3])
    head = model.int8_head(masters).fc
    assert torch.equal(head.codes[:, :q.shape[1]], q) and torch.equal(head.scale, s)
