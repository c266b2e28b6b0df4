"""The 8-bit dense layer's kernels against exact integer sums: sizes around every tile border, strides, rows that are zero or
not finite, the longest exact sum, captured graphs."""
import pytest
import torch

from tests.test_int8_linear import check, rows_oracle

pytestmark = pytest.mark.gpu
DEV, BF = "cuda", torch.bfloat16


def make(m, n, k, dtype, seed=0, bias=True):
    from distributeddeeplearning_amd.ops import functional as ops

    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=gen).to(dtype).to(DEV)
    q, s = ops.quantize_int8(torch.randn(n, k, generator=gen).to(DEV))
    return x, q, s, torch.randn(n, generator=gen).to(DEV) if bias else None


@pytest.mark.parametrize("dtype", [torch.float32, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 1), (1, 15), (5, 64), (7, 65), (3, 129), (300, 2047), (2, 8192), (2, 20001)], ids=str)
def test_codes_are_the_stated_ones(shape, dtype):
    from distributeddeeplearning_amd.ops import functional as ops

    gen = torch.Generator().manual_seed(3)
    w = torch.randn(shape, generator=gen).to(dtype)
    w[0] *= 1e-20
    if shape[0] > 4:
        w[1], w[2, 0], w[3, -1], w[4] = 0.0, float("inf"), float("nan"), 1e-32
    q, s = ops.quantize_int8(w.to(DEV))
    qo, so = rows_oracle(w)
    assert torch.equal(q.cpu(), qo) and torch.equal(s.cpu().nan_to_num(-1.0), so.nan_to_num(-1.0))
    assert not q.as_strided((shape[0], q.stride(0) - shape[1]), q.stride(), shape[1]).any()   # the padding holds zeros
    t = w.t().to(DEV).t()                              # column-major
    assert torch.equal(ops.quantize_int8(t)[0].cpu(), qo)


@pytest.mark.parametrize("dtype", [torch.float32, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("m", [1, 2, 7, 16, 17, 33, 64, 65, 129, 300])
@pytest.mark.parametrize("n, k", [(1, 1), (17, 63), (1000, 64), (64, 65), (129, 200), (1001, 2048), (250, 2047)])
def test_sizes(m, n, k, dtype):
    from distributeddeeplearning_amd.ops import functional as ops

    x, q, s, b = make(m, n, k, dtype, m + n + k, bias=(m + n) % 2 == 0)
    check(ops.linear_int8(x, q, s, b), x, q, s, b)


@pytest.mark.parametrize("m, n, k", [(1, 21841, 2048), (13, 30000, 512), (2500, 700, 1100), (1, 40, 133144), (70, 40, 133144)])
def test_long_ones(m, n, k):
    from distributeddeeplearning_amd.ops import functional as ops

    x, q, s, b = make(m, n, k, BF, 1)
    if k == 133144:
        x.fill_(1.0), q.fill_(127)                       # the largest sum: 127^2 k = 2 147 479 576
    check(ops.linear_int8(x, q, s, b), x, q, s, b)


@pytest.mark.parametrize("m", [3, 70])
def test_rows_that_are_zero_or_not_finite(m):
    from distributeddeeplearning_amd.ops import functional as ops

    x, q, s, b = make(m, 130, 100, torch.float32, 2)
    x[0], x[1, 5], x[2, 99] = 0.0, float("inf"), float("nan")
    if m > 3:
        x[3], x[4], x[69, 0] = 1e-32, 3e38, float("-inf")
    y = ops.linear_int8(x, q, s, b)
    check(y, x, q, s, b)
    assert torch.equal(y[0], b) and y[1].isnan().all() and y[2].isnan().all()


@pytest.mark.parametrize("m", [5, 90])
def test_strides(m):
    from distributeddeeplearning_amd.ops import functional as ops

    x, q, s, b = make(m, 96, 320, torch.float32, 4)
    wide = torch.full((m, 1001), float("nan"), device=DEV)
    wide[:, 33:353] = x
    want = ops.linear_int8(x, q, s, b)
    for v in (wide[:, 33:353], x.t().contiguous().t()):
        assert torch.equal(ops.linear_int8(v, q, s, b), want)
    assert torch.equal(ops.linear_int8(x[:1].expand(m, 320), q, s, b), want[:1].expand(m, 96))
    assert torch.equal(ops.linear_int8(x.view(1, m, 1, 320), q, s, b).view(m, 96), want)
    # codes inside a wider array, with other values behind each row's end
    store = torch.full((96, 480), 77, dtype=torch.int8, device=DEV)
    store[:, 32:332] = q[:, :300]
    view = store[:, 32:332]
    check(ops.linear_int8(x[:, :300], view, s, b), x[:, :300], view, s, b)
    check(ops.linear_int8(x, q[::2], s[::2], b[::2]), x, q[::2], s[::2], b[::2])
    assert ops.linear_int8(x[:0], q, s, b).shape == (0, 96) and ops.linear_int8(x, q[:0], s[:0], b[:0]).shape == (m, 0)


def test_layouts_that_are_refused():
    from distributeddeeplearning_amd.ops import functional as ops
    from distributeddeeplearning_amd.ops.kernels import KernelError

    x, q, s, b = make(2, 8, 100, BF)
    for codes in (q.contiguous(), q.t().contiguous().t(), torch.zeros(8, 160, dtype=torch.int8, device=DEV)[:, 1:101]):
        with pytest.raises(KernelError, match="quantize_int8"):
            ops.linear_int8(x, codes, s, b)
    with pytest.raises(ValueError, match="one device"):
        ops.linear_int8(x, q.cpu(), s, b)


def test_captured_and_on_another_stream():
    from distributeddeeplearning_amd.ops import functional as ops

    cases = [make(m, 333, 500, BF, m) for m in (1, 40, 200)]
    for c in cases:
        ops.linear_int8(*c)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.linear_int8(*c))
        graphs.append(g)
    for rep in range(4):
        for c in cases:
            c[0].copy_(torch.randn(c[0].shape, generator=torch.Generator().manual_seed(rep)))
        for g in graphs if rep % 2 else graphs[::-1]:
            g.replay()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = [ops.linear_int8(*c) for c in cases]
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        for o, e in zip(outs, eager):
            assert torch.equal(o, e)


def test_int8_head_answers_on_the_gpu():
    from distributeddeeplearning_amd.models import resnet18

    torch.manual_seed(0)
    model = resnet18(num_classes=40).to_compute(torch.device(DEV), BF).eval()
    x = torch.randn(3, 3, 64, 64, device=DEV).to(BF).contiguous(memory_format=torch.channels_last)
    seen = []
    with torch.no_grad():
        model.fc.register_forward_hook(lambda mod, args, out: seen.append(args[0]))
        model(x)
        w, b = model.fc.weight, model.fc.bias
        got = model.int8_head()(x)
    from distributeddeeplearning_amd.ops import functional as ops

    check(got, seen[0], *ops.quantize_int8(w.detach()), b.detach())


# tiles of 128 (256 of them or more); the last sizes that a workgroup's LDS takes whole, and the next
@pytest.mark.parametrize("dtype", [torch.float32, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("m, n, k", [(2100, 2100, 200), (9000, 500, 130), (16, 300, 2432), (16, 300, 2560), (1, 200, 40832), (1, 200, 41000), (15, 77, 100),
                                     (1030, 1000, 128), (1024, 1024, 1), (600, 600, 129)])
def test_borders_between_the_forms(m, n, k, dtype):
    from distributeddeeplearning_amd.ops import functional as ops

    x, q, s, b = make(m, n, k, dtype, k, bias=n % 3 != 0)
    check(ops.linear_int8(x, q, s, b), x, q, s, b)


@pytest.mark.parametrize("dtype", [torch.float32, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("m", [1, 6, 16, 40])
def test_unaligned_rows(m, dtype):
    from distributeddeeplearning_amd.ops import functional as ops

    x, q, s, b = make(m, 50, 700, dtype, 9)
    wide = torch.full((2 * m, 1003), float("nan"), device=DEV, dtype=dtype)
    for at in (1, 3, 8):
        v = wide[::2, at:at + 700]
        v.copy_(x)
        check(ops.linear_int8(v, q, s, b), x, q, s, b)
        assert torch.equal(ops.quantize_int8(v)[0], ops.quantize_int8(x)[0])
    every = torch.full((m, 1400), float("nan"), device=DEV, dtype=dtype)
    every[:, ::2] = x
    check(ops.linear_int8(every[:, ::2], q, s, b), x, q, s, b)


def test_a_row_out_of_range_leaves_the_others():
    from distributeddeeplearning_amd.ops import functional as ops

    for m in (4, 16, 100, 2200):
        x, q, s, b = make(m, 2100, 260, BF, 5)
        want = ops.linear_int8(x, q, s, b)
        x[m // 2, 259] = float("inf")
        got = ops.linear_int8(x, q, s, b)
        assert got[m // 2].isnan().all()
        got[m // 2] = want[m // 2]
        assert torch.equal(got, want)


# codes of the input, its values, codes of the weights, results: each beyond 2^31 bytes or values
@pytest.mark.parametrize("m, n, k", [(270000, 24, 8200), (17000001, 8, 128), (9, 1100000, 2048), (40, 1100000, 2048), (47000, 47000, 64)])
def test_offsets_beyond_32_bits(m, n, k):
    from distributeddeeplearning_amd.ops import functional as ops

    gen = torch.Generator(DEV).manual_seed(6)
    x = torch.randn(m, k, generator=gen, device=DEV, dtype=BF)
    q, s = ops.quantize_int8(torch.randn(n, k, generator=gen, device=DEV, dtype=BF))
    b = torch.randn(n, generator=gen, device=DEV)
    y = ops.linear_int8(x, q, s, b)
    rows = sorted({0, m // 2, m - 1}) if m < 100 else [0, 1, m // 3, m // 2, m - 2, m - 1]
    cols = torch.tensor([0, 1, n // 2, n - 2, n - 1], device=DEV)
    check(y[rows][:, cols], x[rows], q[cols], s[cols], b[cols])


# rows of codes that end inside a stage of 128 bytes, one channel in the last tile, a stage that the second group of waves does not have
@pytest.mark.parametrize("k", [64, 192, 257, 272, 320, 513, 769])
@pytest.mark.parametrize("m, n", [(17, 1), (40, 65), (100, 129), (1100, 4097)])
def test_rows_that_end_inside_a_stage(m, n, k):
    from distributeddeeplearning_amd.ops import functional as ops

    x, q, s, b = make(m, n, k, BF, k, bias=k % 2 == 0)
    check(ops.linear_int8(x, q, s, b), x, q, s, b)
    # rows 16 bytes apart where they can be, and nothing behind the last one
    ld = (k + 15) // 16 * 16
    store = torch.zeros(n * ld, dtype=torch.int8, device=DEV)
    tight = store.view(n, ld)[:, :k]
    tight.copy_(q)
    check(ops.linear_int8(x, tight, s, b), x, tight, s, b)
