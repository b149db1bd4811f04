"""A frozen BlockScaledLinear keeps its weight's codes; they are those of the weight as it is."""

import copy
import io

import pytest
import torch

import feather_ops as fo

pytestmark = pytest.mark.gpu


@pytest.fixture
def layer(cuda_device):
    torch.manual_seed(3)
    layer = torch.nn.Linear(300, 130, device="cuda", dtype=torch.bfloat16).requires_grad_(False)
    fo.to_block_scaled_linear(layer)
    return layer


def _x(rows=9, k=300):
    return torch.randn((rows, k), generator=torch.Generator("cuda").manual_seed(5), device="cuda").bfloat16()


def _is_current(layer, x=None):
    x = _x() if x is None else x
    return torch.equal(layer(x), fo.block_scaled_linear(x, layer.weight.detach().clone(), layer.bias))


def _double(layer):
    with torch.no_grad():
        layer.weight.mul_(2)


def _load(layer):
    layer.load_state_dict({name: value + 1 for name, value in layer.state_dict().items()})


def _assign(layer):
    layer.load_state_dict({name: value + 1 for name, value in layer.state_dict().items()}, assign=True)
    layer.requires_grad_(False)


def _replace(layer):
    layer.weight = torch.nn.Parameter(layer.weight + 1, requires_grad=False)


def _data(layer):
    layer.weight.data = layer.weight.data + 1


def _train(layer):
    layer.requires_grad_(True)
    optimizer = torch.optim.SGD(layer.parameters(), lr=1.0)
    layer(_x()).float().square().mean().backward()
    optimizer.step()
    layer.requires_grad_(False)
    layer.zero_grad()


@pytest.mark.parametrize("change", [_double, _load, _assign, _replace, _data, _train])
def test_codes_follow_the_weight(layer, change):
    before = layer(_x())
    assert _is_current(layer)
    change(layer)
    assert not torch.equal(layer(_x()), before) and _is_current(layer)
    codes, scale = fo.quantize_blocks(layer.weight, square=True)
    assert torch.equal(layer.weight_fp8.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(layer.weight_scale, scale)


@pytest.mark.parametrize("change", [_double, _train])
def test_input_gradient_is_that_of_the_forwards_weight(layer, change):
    change(layer)
    x = _x().requires_grad_()
    gy = torch.randn(9, 130, device="cuda").bfloat16()
    got, = torch.autograd.grad(layer(x), x, gy)
    want, = torch.autograd.grad(fo.block_scaled_linear(x, layer.weight.detach().clone(), layer.bias), x, gy)
    assert torch.equal(got, want)


def test_swapped_weight_for_one_call(layer):
    own = layer(_x())
    other = {"weight": layer.weight + 1, "bias": layer.bias}
    got = torch.func.functional_call(layer, other, (_x(),))
    assert torch.equal(got, fo.block_scaled_linear(_x(), other["weight"], layer.bias))
    assert torch.equal(layer(_x()), own)


def test_copies_and_files(layer):
    twin = copy.deepcopy(layer)
    _double(twin)
    assert _is_current(twin) and _is_current(layer) and not torch.equal(twin(_x()), layer(_x()))
    file = io.BytesIO()
    torch.save(layer.state_dict(), file)
    file.seek(0)
    twin.load_state_dict(torch.load(file, weights_only=True))
    assert torch.equal(twin(_x()), layer(_x()))


def test_codes_are_updated_in_place(layer):
    """A graph that was captured with the kept codes reads the new ones after an update, and no freed memory."""
    x = _x()
    layer(x)
    kept = layer.weight_fp8.data_ptr(), layer.weight_scale.data_ptr()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(x)
    for replay in range(3):
        _double(layer)
        if replay % 2:
            layer.quantize_weight_()
        want = layer(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        assert kept == (layer.weight_fp8.data_ptr(), layer.weight_scale.data_ptr())


def test_change_that_a_capture_meets(layer):
    """Codes that are out of date when a graph is captured: each replay quantizes the weight as it is then."""
    x = _x()
    layer(x)
    _double(layer)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(x)
    assert _is_current(layer)
    for _ in range(3):
        _double(layer)
        want = fo.block_scaled_linear(x, layer.weight, layer.bias)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_inference_mode(layer):
    with torch.inference_mode():
        _double(layer)
        assert _is_current(layer)
        layer.quantize_weight_()
        made = torch.nn.Linear(300, 130, device="cuda", dtype=torch.bfloat16).requires_grad_(False)
        fo.to_block_scaled_linear(made)
        assert _is_current(made)
    _double(layer)
    assert _is_current(layer) and _is_current(layer)


@pytest.mark.parametrize("swap", [False, True])
@pytest.mark.parametrize("move", [lambda m: m.half(), lambda m: m.to(torch.float32), lambda m: m.float().bfloat16(),
                                  lambda m: m.to("cuda"), lambda m: torch.nn.Sequential(m).float()[0].half(),
                                  lambda m: m.cpu().cuda(), lambda m: m.cpu().half().cuda()])
def test_in_another_type_or_on_another_device(layer, move, swap):
    """Codes stay fp8 and scales fp32, and are those of the weight in its new type."""
    before = torch.__future__.get_swap_module_params_on_conversion()
    torch.__future__.set_swap_module_params_on_conversion(swap)
    try:
        moved = move(layer)
    finally:
        torch.__future__.set_swap_module_params_on_conversion(before)
    assert moved is layer and layer.weight_fp8.dtype == torch.float8_e4m3fn and layer.weight_scale.dtype == torch.float32
    assert layer.weight_fp8.is_cuda and layer.weight_scale.is_cuda and not layer.weight.requires_grad
    assert _is_current(layer, _x().to(layer.weight.dtype))


def test_format_is_kept(layer):
    layer.quantize_weight_(torch.float8_e5m2)
    layer.cpu()
    assert {t.device.type for t in (layer.weight, layer.weight_fp8, layer.weight_scale)} == {"cpu"}
    layer.half().cuda()
    assert layer.weight_fp8.dtype == torch.float8_e5m2
    assert torch.equal(layer(_x().half()), fo.block_scaled_linear(_x().half(), layer.weight, layer.bias, torch.float8_e5m2))


def test_quantizing_again_keeps_the_layers_format(cuda_device):
    layer = torch.nn.Linear(300, 130, device="cuda", dtype=torch.bfloat16).requires_grad_(False)
    fo.to_block_scaled_linear(layer, torch.float8_e5m2)
    layer.weight.data.mul_(2)
    layer.quantize_weight_()
    assert layer.weight_fp8.dtype == torch.float8_e5m2
    assert torch.equal(layer(_x()), fo.block_scaled_linear(_x(), layer.weight, layer.bias, torch.float8_e5m2))
    layer.quantize_weight_(torch.float8_e4m3fn)
    assert layer.weight_fp8.dtype == torch.float8_e4m3fn and _is_current(layer)
