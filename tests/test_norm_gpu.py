"""The norms around a block on the device against the formula in float64. A result is rounded once, u of it; before that b has passed four
roundings of 2^-24 and the sum one, which h inherits times its factor, with three of its own and two of the root's: 2^-21 of the sizes
that are added covers them. Smallest steps of the types: 2^-24 (fp16), 2^-133 (bf16), halved."""
import pytest
import torch

from oracle.attention import U
from test_attention_gpu import BF, DEV, HF, NAN, randn

pytestmark = pytest.mark.gpu
EPS = 1e-5


def reference(x, y, gate, post, pre, scale, eps):
    d = lambda t: None if t is None else t.cpu().double()  # noqa: E731
    x, y, gate, post, pre = d(x), d(y), d(gate), d(post), d(pre)
    rms = lambda z: (z.square().mean(-1, keepdim=True) + eps).sqrt()  # noqa: E731
    s, size = x, x.abs()
    if y is not None:
        b = y if post is None else y / rms(y) * post
        b = scale * b if gate is None else scale * b * gate
        s, size = x + b, x.abs() + b.abs()
    factor = 1 / rms(s) * (1 if pre is None else pre)
    return s, s * factor, size, size * factor.abs()


def check(got, x, y, gate, post, pre, scale, eps, dtype):
    want = reference(x, y, gate, post, pre, scale, eps)
    step = 2.0 ** -25 if dtype == HF else 2.0 ** -134
    for out, ref, size in ((got[0], want[0], want[2]), (got[1], want[1], want[3])):
        if out is not None:
            err, tol = (out.cpu().double() - ref).abs(), U[dtype] * ref.abs() + 2.0 ** -21 * size + step
            assert (err <= tol).all(), (err - tol).max().item()


@pytest.mark.parametrize("M,D", [(1, 8), (1, 4096), (3, 512), (5, 520), (7, 2048), (2, 2056), (4, 4104), (9, 8192), (3, 8200), (2, 16384),
                                 (2, 16392), (1, 32768), (3000, 64), (2100, 1000), (1200, 8192)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_add_norm(capi, M, D, dtype):
    gen = torch.Generator().manual_seed(M + D)
    x, y, rows, per_row = (randn(gen, M, D, dtype=dtype, scale=2.0).to(DEV) for _ in range(4))
    post, pre, channel = (randn(gen, D, dtype=dtype).to(DEV) for _ in range(3))
    for gate, a, b, scale in ((None, None, None, 1.0), (channel, post, None, 0.5), (per_row, post, pre, -1.25), (None, None, pre, 1.0)):
        check(capi.add_norm(x, y, gate, a, b, scale, EPS), x, y, gate, a, b, scale, EPS, dtype)
        if M > 1000:
            break
    check(capi.add_norm(rows, pre=pre), rows, None, None, None, pre, 1.0, EPS, dtype)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_rows_in_wider_ones_in_place_and_one_result_alone(capi, dtype):
    gen = torch.Generator().manual_seed(1)
    M, D = 37, 264
    wide = [torch.full((M, D + 16), NAN, dtype=dtype, device=DEV) for _ in range(5)]
    x, y, gate, xo, h = (w[:, 8:8 + D] for w in wide)
    for t in (x, y, gate):
        t.copy_(randn(gen, M, D, dtype=dtype))
    post = randn(gen, D, dtype=dtype).to(DEV)
    want = capi.add_norm(x.contiguous(), y.contiguous(), gate.contiguous(), post, None, 0.5, EPS)
    capi.add_norm(x, y, gate, post, None, 0.5, EPS, xo, h)
    assert torch.equal(xo, want[0]) and torch.equal(h, want[1])
    assert all(torch.isnan(w[:, :8]).all() and torch.isnan(w[:, 8 + D:]).all() for w in wide)
    assert torch.equal(capi.add_norm(x, y, gate, post, None, 0.5, EPS, h=False)[0], want[0])
    assert torch.equal(capi.add_norm(x, y, gate, post, None, 0.5, EPS, x_out=False)[1], want[1])
    one = x[:1].expand(M, D)                                    # one row for all
    assert torch.equal(capi.lib().fsw_version() and capi.add_norm(x, y, x[0].contiguous(), post, None, 0.5, EPS)[1],
                       capi.add_norm(x, y, one.contiguous(), post, None, 0.5, EPS)[1])
    capi.add_norm(x, y, gate, post, None, 0.5, EPS, x, y)       # over the inputs
    assert torch.equal(x, want[0]) and torch.equal(y, want[1])


@pytest.mark.parametrize("D", [64, 1000, 8192])
def test_values_of_any_size(capi, D):
    """Squares that no float holds, at either end, and a row whose neighbours are not numbers."""
    gen = torch.Generator().manual_seed(D)
    for dtype, sizes in ((BF, (1e38, 1e20, 1.0, 1e-6, 1e-20, 1e-30)), (HF, (2e4, 1.0, 1e-3, 1e-6))):
        for size in sizes:
            x, y = (randn(gen, 3, D, dtype=torch.float32, scale=size / 4).to(dtype).to(DEV) for _ in range(2))
            post = torch.full((D,), size if size < 1e30 else 1.0).to(dtype).to(DEV)
            for eps in (EPS, 1e-37):
                check(capi.add_norm(x, y, None, post, None, 0.5, eps), x, y, None, post, None, 0.5, eps, dtype)
    x = randn(gen, 6, D).to(DEV)
    clean = capi.add_norm(x, x, None, x[0], x[1], 1.0, EPS)
    bad = x.clone()
    bad[2, 3], bad[4, D - 1] = NAN, float("inf")
    out = capi.add_norm(bad, x, None, x[0], x[1], 1.0, EPS)
    assert all(torch.equal(o[[0, 1, 3, 5]], c[[0, 1, 3, 5]]) for o, c in zip(out, clean))
    assert torch.isnan(out[1][2]).all() and torch.isnan(out[1][4, D - 1]) and out[0][4, D - 1] == float("inf")
    assert (out[1][4, :D - 1] == 0).all()                       # finite values over an infinite root


def test_rows_of_zeros(capi):
    z = torch.zeros(4, 128, dtype=BF, device=DEV)
    x, h = capi.add_norm(z, z, None, z[0], None, 1.0, EPS)
    assert not x.any() and not h.any()


@pytest.mark.parametrize("dtype,name", [(BF, "bf16"), (HF, "fp16")])
def test_torch_operators(capi, ext, dtype, name):
    gen = torch.Generator().manual_seed(3)
    x, y, gate = (randn(gen, 2, 5, 256, dtype=dtype).to(DEV) for _ in range(3))
    post, pre = (randn(gen, 256, dtype=dtype).to(DEV) for _ in range(2))
    flat = [t.view(10, 256) for t in (x, y, gate)]
    for add, norm in ((getattr(ext, "add_norm_" + name), getattr(ext, "rms_norm_" + name)),
                      (getattr(torch.ops.ASMLLM, "add_norm_" + name), getattr(torch.ops.ASMLLM, "rms_norm_" + name))):
        want = capi.add_norm(*flat, post, pre, 0.5, 1e-6)
        got = add(x, y, gate, post, pre, 0.5, 1e-6)
        assert got[0].shape == x.shape and all(torch.equal(a.view(10, 256), b) for a, b in zip(got, want))
        assert torch.equal(add(x, y)[1].view(10, 256), capi.add_norm(flat[0], flat[1])[1])
        assert torch.equal(add(x, y, post)[0].view(10, 256), capi.add_norm(flat[0], flat[1], post)[0])
        assert torch.equal(norm(x, pre).view(10, 256), capi.add_norm(flat[0], pre=pre)[1])
        one = x[0, 0]                                           # a single token, no batch dimension
        assert torch.equal(add(one, y[0, 0], gate[0, 0], post, pre)[1], add(x, y, gate, post, pre)[1][0, 0])
        strided = x.transpose(0, 1)                             # rows that have no common stride are copied
        assert torch.equal(add(strided, y.transpose(0, 1), gate.transpose(0, 1), post, pre)[1], add(x, y, gate, post, pre)[1].transpose(0, 1))
        assert add(x[:0], y[:0])[0].shape == (0, 5, 256) and norm(x[:0]).shape == (0, 5, 256)
        for bad in ((x, y[:1]), (x, y, gate[0]), (x, y, gate, post[:8]), (x.float(), y), (x, y.float())):
            with pytest.raises(RuntimeError):
                add(*bad)
        with pytest.raises(RuntimeError):
            add(x, y, None, None, None, float("nan"))
        with pytest.raises(RuntimeError):
            norm(x, pre, 0.0)
        with pytest.raises(RuntimeError):
            norm(x[..., :12].contiguous())
