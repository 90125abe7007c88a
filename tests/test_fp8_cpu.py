"""What the 8-bit operators refuse, without a GPU: formats, devices, types, and the C entry points' arguments."""

import pytest
import torch

import deconver_b200 as dcb
from deconver_b200 import _lib
from deconver_b200._build import build_library


@pytest.fixture(scope="module")
def lib():
    build_library()
    return _lib.load()


@pytest.mark.parametrize("kw", [{"checkpoint": "e5m2"}, {"products": "bf16"}, {"checkpoint": None}, {"products": True}])
def test_unknown_formats_are_refused(kw):
    with pytest.raises(ValueError, match="must be one of"):
        dcb.Linear(4, 8, **kw)
    with pytest.raises(ValueError, match="must be one of"):
        dcb.MLP(4, **kw)
    with pytest.raises(ValueError, match="must be one of"):
        dcb.channel_linear(torch.ones(1, 4, 3), torch.ones(8, 4, 1), **kw)
    if "checkpoint" in kw:
        with pytest.raises(ValueError, match="must be one of"):
            dcb.bias_gelu(torch.ones(1, 4, 3), None, **kw)


def test_cpu_tensors_are_refused_not_computed(lib):
    x, w = torch.ones(1, 4, 3), torch.ones(8, 4, 1)
    for kw in ({"checkpoint": "fp8"}, {"products": "fp8"}):
        with pytest.raises(RuntimeError, match="CUDA"):
            dcb.channel_linear(x, w, **kw)
        with pytest.raises(RuntimeError, match="CUDA"):
            dcb.MLP(4, **kw)(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        dcb.bias_gelu(x, None, checkpoint="fp8")
    with pytest.raises(RuntimeError, match="CUDA"):
        dcb.quantize(x)
    with pytest.raises(RuntimeError, match="do not hold"):
        dcb.Quantized(torch.zeros(1, 4, 16).to(torch.float8_e4m3fn), torch.ones(1, 4, 4).to(torch.float8_e8m0fnu), (1, 4, 3), torch.float32).dequantize()
    with pytest.raises(NotImplementedError, match="not supported"):
        dcb.Quantized(x, x, (1, 4, 3), torch.float32).dequantize(torch.float16)


def test_exact_formats_are_the_plain_layer():
    torch.manual_seed(0)
    x, m = torch.randn(2, 4, 3, 5), dcb.Linear(4, 8, checkpoint="exact", products="exact")
    assert torch.equal(m(x), dcb.channel_linear(x, m.linear.weight, m.linear.bias))
    assert m.extra_repr() == "" and "fp8" in repr(dcb.Linear(4, 8, products="fp8"))
    assert list(dcb.MLP(4, checkpoint="fp8").state_dict()) == list(dcb.MLP(4).state_dict())


def test_sizes_in_memory(lib):
    assert [lib.ndc_q8_pitch(n) for n in (-1, 0, 1, 16, 17, 2 ** 33 + 1)] == [0, 0, 16, 16, 32, 2 ** 33 + 16]
    assert [lib.ndc_q8_scales(n) for n in (-1, 0, 1, 128, 512, 513, 2 ** 33)] == [0, 0, 4, 4, 4, 8, 2 ** 26]
    assert lib.ndc_q8_product_workspace_bytes(0, 4, 4, 4, 0) == 0
    assert lib.ndc_q8_product_workspace_bytes(1, 64, 256, 128, 0) == 4 * 64 * 256
    assert lib.ndc_q8_product_workspace_bytes(16, 2048, 512, 262144, 1) >= 4 * 2048 * 512
    assert lib.ndc_q8_product_workspace_bytes(1, 8, 8, 2 ** 31 - 200, 0) == 4 * 8 * 8 * 65535       # the most slices of a launch
    assert lib.ndc_q8_wgrad_workspace_bytes(0, 4, 4, 4, 0) == 0 and lib.ndc_q8_wgrad_workspace_bytes(1, 96, 24, 64, 0) == 4 * 96 * 25


A = 4096       # an address that is aligned and never read


@pytest.mark.parametrize("status,call", [
    (1, lambda l: l.ndc_q8_hold(2, 8, 0, None, A, A, None)),
    (1, lambda l: l.ndc_q8_hold(0, 8, 0, A, A, A, None)),
    (1, lambda l: l.ndc_q8_hold(2, 8, 7, A, A, A, None)),
    (2, lambda l: l.ndc_q8_hold(2 ** 31, 8, 0, A, A, A, None)),
    (2, lambda l: l.ndc_q8_hold(2 ** 20, 2 ** 20, 0, A, A, A, None)),
    (5, lambda l: l.ndc_q8_hold(2, 8, 0, A, A + 8, A, None)),
    (5, lambda l: l.ndc_q8_hold(2, 8, 0, A, A, A + 2, None)),
    (1, lambda l: l.ndc_q8_hold_channels(2, 8, 0, 0, A, A, A, None, None, None)),
    (2, lambda l: l.ndc_q8_hold_channels(2, 8, 2 ** 24 + 1, 0, A, A, A, None, None, None)),
    (2, lambda l: l.ndc_q8_hold_channels(2 ** 20, 8, 2 ** 20, 0, A, A, A, None, None, None)),
    (1, lambda l: l.ndc_q8_hold_sum(2, 8, 4, 0, A, A, A, None, 0, A, 1 << 20, None)),
    (1, lambda l: l.ndc_q8_hold_sum(2, 8, 4, 0, A, A, A, A, 3, A, 1 << 20, None)),
    (2, lambda l: l.ndc_q8_hold_sum(2 ** 15, 2 ** 12, 4, 0, A, A, A, A, 0, A, 1 << 20, None)),
    (3, lambda l: l.ndc_q8_hold_sum(2, 8, 4, 0, A, A, A, A, 0, None, 0, None)),
    (5, lambda l: l.ndc_q8_hold_channels(2, 8, 4, 0, A, A + 4, A, None, None, None)),
    (1, lambda l: l.ndc_q8_hold_channels(2, 8, 4, 0, A, A, A, A, None, None)),
    (5, lambda l: l.ndc_q8_hold_channels(2, 8, 4, 1, A, A, A, A + 8, A, None)),
    (1, lambda l: l.ndc_q8_read(2, 8, 0, A, None, A, None)),
    (1, lambda l: l.ndc_q8_read(2, -8, 0, A, A, A, None)),
    (5, lambda l: l.ndc_q8_read(2, 8, 0, A + 1, A, A, None)),
    (1, lambda l: l.ndc_q8_bias_gelu_fwd(2, 8, 4, 0, A, None, A, A, None, None)),
    (1, lambda l: l.ndc_q8_bias_gelu_fwd(2, 8, 4, 0, A, None, None, A, A, None)),
    (1, lambda l: l.ndc_q8_bias_gelu_fwd(-2, -8, 4, 0, A, None, A, A, A, None)),
    (1, lambda l: l.ndc_q8_bias_gelu_bwd(2, 8, 4, 0, A, A, A, None, None, None, None, 0, None)),
    (2, lambda l: l.ndc_q8_bias_gelu_bwd(2 ** 15, 2 ** 12, 4, 0, A, A, A, None, A, None, None, 0, None)),
    (3, lambda l: l.ndc_q8_bias_gelu_bwd(2, 8, 4, 0, A, A, A, None, A, A, A, 64, None)),
    (1, lambda l: l.ndc_q8_product(1, 8, 8, 8, 0, A, A, A, A, None, 0, 8, None, None, 0, None)),
    (1, lambda l: l.ndc_q8_product(1, 8, 8, 0, 0, A, A, A, A, None, 0, 8, A, None, 0, None)),
    (1, lambda l: l.ndc_q8_product(1, 8, 8, 8, 0, A, A, A, A, None, 0, 3, A, None, 0, None)),
    (1, lambda l: l.ndc_q8_product(2, 8, 8, 8, 0, A, A, A, A, A, 0, 8, A, A, 1 << 20, None)),
    (1, lambda l: l.ndc_q8_product(2, 8, 8, 8, 0, A, A, A, A, None, 0, 4, A, A, 1 << 20, None)),
    (2, lambda l: l.ndc_q8_product(2, 2 ** 30, 8, 8, 0, A, A, A, A, None, 0, 2 ** 30, A, A, 1 << 40, None)),
    (2, lambda l: l.ndc_q8_product(1, 2 ** 30, 2 ** 23, 8, 0, A, A, A, A, None, 0, 2 ** 30, A, None, 0, None)),
    (3, lambda l: l.ndc_q8_product(2, 8, 8, 8, 0, A, A, A, A, None, 0, 8, A, None, 0, None)),
    (5, lambda l: l.ndc_q8_product(1, 8, 8, 8, 0, A, A, A + 8, A, None, 0, 8, A, None, 0, None)),
    (1, lambda l: l.ndc_q8_product(1, 8, 8, 8, 0, A, A, A, A, A, 5, 8, A, None, 0, None)),
    (1, lambda l: l.ndc_q8_project(2, 8, 8, 4, 0, A, A, A, None, 0, None, None)),
    (1, lambda l: l.ndc_q8_project(2, 8, 8, 0, 0, A, A, A, None, 0, A, None)),
    (1, lambda l: l.ndc_q8_project(2, 8, 8, 4, 0, A, A, A, A, 9, A, None)),
    (2, lambda l: l.ndc_q8_project(2, 513, 8, 4, 0, A, A, A, None, 0, A, None)),
    (2, lambda l: l.ndc_q8_project(2, 8, 8, 2 ** 24 + 1, 0, A, A, A, None, 0, A, None)),
    (2, lambda l: l.ndc_q8_project(1, 8, 2 ** 30 + 1, 4, 0, A, A + 8, A, None, 0, A, None)),
    (5, lambda l: l.ndc_q8_project(2, 8, 8, 4, 0, A, A + 8, A, None, 0, A, None)),
    (1, lambda l: l.ndc_q8_wgrad(2, 8, 8, 4, 0, A, A, A, None, None, 0, A, 1 << 20, None)),
    (1, lambda l: l.ndc_q8_wgrad(2, 8, 8, 4, 2, A, A, A, A, None, 0, A, 1 << 20, None)),
    (1, lambda l: l.ndc_q8_wgrad(2, 8, 8, 4, 0, A, A, A, A, A, 2, A, 1 << 20, None)),
    (2, lambda l: l.ndc_q8_wgrad(2, 8, 8, 2 ** 31, 0, A, A, A, A, None, 0, A, 1 << 20, None)),
    (3, lambda l: l.ndc_q8_wgrad(2, 8, 8, 4, 0, A, A, A, A, None, 0, A, 16, None)),
    (5, lambda l: l.ndc_q8_wgrad(2, 8, 8, 4, 0, A, A + 8, A, A, None, 0, A, 1 << 20, None)),
    (1, lambda l: l.ndc_q8_linear_fwd(2, 8, 8, 8, A, A, None, 0, A, A, None, None)),
    (1, lambda l: l.ndc_q8_linear_fwd(2, 8, 8, 8, A, A, A, 4, A, None, None, None)),
    (2, lambda l: l.ndc_q8_linear_fwd(2, 8, 8, 9, A, A, None, 0, A, None, None, None)),
    (2, lambda l: l.ndc_q8_linear_fwd(2, 512, 512, 8, A, A, None, 0, A, None, None, None)),
    (5, lambda l: l.ndc_q8_linear_fwd(2, 8, 8, 8, A + 2, A, None, 0, A, None, None, None)),
    (5, lambda l: l.ndc_q8_product(1, 8, 8, 8, 0, A, A, A, A + 1, None, 0, 8, A, None, 0, None)),
    (5, lambda l: l.ndc_q8_hold(2, 8, 0, A + 2, A, A, None)),
    (5, lambda l: l.ndc_q8_hold(2, 8, 1, A + 1, A, A, None)),
    (5, lambda l: l.ndc_q8_hold_sum(2, 8, 4, 1, A + 2, A, A, A + 2, 0, A, 1 << 20, None)),
    (5, lambda l: l.ndc_q8_hold_channels(2, 8, 4, 1, A + 1, A, A, None, None, None)),
    (5, lambda l: l.ndc_q8_read(2, 8, 0, A, A, A + 2, None)),
    (5, lambda l: l.ndc_q8_bias_gelu_fwd(2, 8, 4, 1, A, A + 2, A, A, A, None)),
    (5, lambda l: l.ndc_q8_bias_gelu_fwd(2, 8, 4, 0, A, A, A + 1, None, None, None)),
    (5, lambda l: l.ndc_q8_bias_gelu_bwd(2, 8, 4, 1, A, A, A, None, A + 1, None, None, 0, None)),
    (5, lambda l: l.ndc_q8_bias_gelu_bwd(2, 8, 4, 1, A, A, A, None, A, A + 2, A, 1 << 20, None)),
    (5, lambda l: l.ndc_q8_product(1, 8, 8, 8, 0, A, A, A, A, None, 0, 8, A + 2, None, 0, None)),
    (5, lambda l: l.ndc_q8_project(2, 8, 8, 4, 1, A + 1, A, A, None, 0, A, None)),
    (5, lambda l: l.ndc_q8_project(2, 8, 8, 4, 1, A, A, A, A + 2, 0, A, None)),
    (5, lambda l: l.ndc_q8_wgrad(2, 8, 8, 4, 0, A + 2, A, A, A, None, 0, A, 1 << 20, None)),
    (5, lambda l: l.ndc_q8_wgrad(2, 8, 8, 4, 1, A, A, A, A, A + 2, 0, A, 1 << 20, None)),
    (5, lambda l: l.ndc_q8_linear_fwd(2, 8, 8, 8, A, A, A + 2, 0, A, None, None, None)),
])
def test_entry_points_refuse_bad_arguments(lib, status, call):
    assert call(lib) == status, lib.ndc_q8_last_error()
    assert lib.ndc_q8_last_error().startswith(b"q8 ")


@pytest.mark.parametrize("status,call", [
    (1, lambda l: l.ndc_q8_linear_fwd_parts(2, 8, 8, 8, A, None, None, 0, A, A, A, None)),
    (1, lambda l: l.ndc_q8_linear_fwd_parts(2, 8, 8, 8, A, A, None, 0, A, None, A, None)),
    (1, lambda l: l.ndc_q8_linear_fwd_parts(2, 8, 8, 8, A, A, A, 4, A, None, None, None)),
    (2, lambda l: l.ndc_q8_linear_fwd_parts(2, 8, 8, 12, A, A, None, 0, A, None, None, None)),
    (2, lambda l: l.ndc_q8_linear_fwd_parts(2, 12, 8, 8, A, A, None, 0, A, None, None, None)),
    (2, lambda l: l.ndc_q8_linear_fwd_parts(2, 520, 8, 8, A, A, None, 0, A, None, None, None)),
    (2, lambda l: l.ndc_q8_linear_fwd_parts(2, 512, 2 ** 20 + 1, 8, A, A, None, 0, A, None, None, None)),
    (2, lambda l: l.ndc_q8_linear_fwd_parts(0, 8, 8, 8, A, A, None, 0, A, None, None, None)),
    (2, lambda l: l.ndc_q8_linear_fwd_parts(2 ** 20, 8, 8, 2 ** 25, A, A, None, 0, A, None, None, None)),
    (5, lambda l: l.ndc_q8_linear_fwd_parts(2, 512, 2048, 8, A, A + 8, None, 0, A, None, None, None)),
    (5, lambda l: l.ndc_q8_linear_fwd_parts(2, 512, 2048, 8, A, A, None, 0, A + 2, None, None, None)),
    (5, lambda l: l.ndc_q8_linear_fwd_parts(2, 512, 2048, 8, A, A, A + 2, 0, A, None, None, None)),
])
def test_the_forward_in_parts_refuses_bad_arguments(lib, status, call):
    assert call(lib) == status, lib.ndc_q8_last_error()
    assert lib.ndc_q8_last_error().startswith(b"q8 linear")


@pytest.mark.parametrize("status,call", [
    (1, lambda l: l.ndc_bias_round(2, 8, 8, A, None, A, 8, None)),
    (1, lambda l: l.ndc_bias_round(2, 8, 0, A, A, A, 8, None)),
    (1, lambda l: l.ndc_bias_round(2, 8, 8, A, A, A, 7, None)),
    (2, lambda l: l.ndc_bias_round(2 ** 20, 2 ** 10, 8, A, A, A, 8, None)),
    (5, lambda l: l.ndc_bias_round(2, 8, 8, A + 2, A, A, 8, None)),
    (5, lambda l: l.ndc_bias_round(2, 8, 8, A, A, A + 1, 8, None)),
])
def test_the_rounded_bias_refuses_bad_arguments(lib, status, call):
    assert call(lib) == status, lib.ndc_bias_last_error()
    assert lib.ndc_bias_last_error().startswith(b"bias")


@pytest.mark.parametrize("batch,co,ci,n", [(2, 2048, 512, 64 ** 3), (1, 1024, 1024, 64 ** 3), (1, 256, 256, 1 << 22), (1, 8, 8, 1 << 28), (16, 2048, 2048, 8192), (4, 4096, 4096, 1 << 18)])
def test_scratch_of_long_sums_is_bounded(lib, batch, co, ci, n):
    """float32 sums in slices of some hundred positions each: three results of scratch or 64 MiB, whatever the positions."""
    most = max(3 * 4 * co * (ci + 1), 64 << 20)
    for dtype in (0, 1):
        assert 0 < lib.ndc_q8_wgrad_workspace_bytes(batch, co, ci, n, dtype) <= most
        assert 0 < lib.ndc_q8_product_workspace_bytes(batch, ci, co, n, dtype) <= most


def test_scratch_of_what_is_refused(lib):
    for size in ((1, 2 ** 31 - 1, 8, 64), (1, 8, 2 ** 31 - 1, 64), (2, 8, 8, 2 ** 31), (1, 2 ** 20, 2 ** 20, 64), (2 ** 20, 8, 8, 2 ** 20)):
        assert lib.ndc_q8_wgrad_workspace_bytes(*size, 0) == 0
        assert lib.ndc_q8_wgrad(*size, 0, A, A, A, A, None, 0, A, 1 << 40, None) == 2
    for samples, m, n, k in ((1, 2 ** 31, 2 ** 31, 8), (1, 2 ** 62, 4, 8), (2, 2 ** 30, 8, 8), (1, 2 ** 30, 2 ** 23, 8), (1, 8, 8, 2 ** 31), (2 ** 20, 8, 8, 2 ** 20)):
        assert lib.ndc_q8_product_workspace_bytes(samples, m, n, k, 0) == 0
        assert lib.ndc_q8_product(samples, m, n, k, 0, A, A, A, A, None, 0, m, A, A, 1 << 40, None) == 2


def test_products_of_too_many_positions_are_refused(lib):
    """By the layer, before a kernel's own limit is met."""
    x, w = torch.zeros(1, 1, 1).expand(1, 1, 2 ** 24 + 1), torch.zeros(4, 1, 1)
    with pytest.raises(RuntimeError, match="up to 2.24 positions per sample"):
        _lib.load_ext().linear_q8(x, w, None, True)
    with pytest.raises(RuntimeError, match="up to 2.24 positions per sample"):
        _lib.load_ext().linear_q8(x.view(1, 1, -1, 1), w, None, True)


@pytest.mark.parametrize("with_bias", [True, False])
@pytest.mark.parametrize("shape,outputs", [((0, 4, 5), 8), ((2, 4, 0), 8), ((2, 0, 5), 8), ((2, 4, 3, 0, 2), 8), ((2, 4, 5), 0), ((0, 4, 0, 3), 0)], ids=str)
def test_the_exact_layer_of_no_elements(shape, outputs, with_bias):
    x, w, b = (torch.ones(s, requires_grad=True) for s in (shape, (outputs, shape[1], 1), (outputs,)))
    y = dcb.channel_linear(x, w, b if with_bias else None)
    assert y.shape == (shape[0], outputs, *shape[2:]) and (y == float(with_bias)).all()
    y.sum().backward()
    assert not x.grad.any() and not w.grad.any()
    assert not with_bias or torch.equal(b.grad, torch.full((outputs,), float(y[:, :1].numel())))


def test_an_mlp_that_keeps_its_hidden_tensor_says_so():
    import warnings

    class Same(torch.nn.Module):
        def forward(self, x):
            return x

    x = torch.randn(1, 4, 3)
    for checkpoint in ("exact", "fp8"):
        mlp = dcb.MLP(4, checkpoint=checkpoint)
        mlp.block[0], mlp.block[3] = Same(), Same()
        with warnings.catch_warnings(record=True) as told:
            warnings.simplefilter("always")
            assert torch.equal(mlp(x), torch.nn.functional.gelu(x))
        assert [str(w.message).count("keeps the hidden tensor exactly") for w in told] == [1] * (checkpoint == "fp8")
