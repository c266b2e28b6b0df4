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
