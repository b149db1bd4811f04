"""Int4Linear serves its weight as it is: codes follow every change that torch sees."""

import copy
import io

import pytest
import torch

import feather_ops as fo

pytestmark = pytest.mark.gpu
FORMATS = [(128, False), (32, True)]


@pytest.fixture(params=FORMATS, ids=str)
def layer(request, cuda_device):
    torch.manual_seed(3)
    layer = torch.nn.Linear(300, 130, device="cuda", dtype=torch.bfloat16)
    assert fo.to_int4_linear(layer, *request.param) == 1
    layer.format = request.param
    return layer


def _x(rows=9, k=300):
    return torch.randn((rows, k), generator=torch.Generator("cuda").manual_seed(5), device="cuda").bfloat16()


def _own(layer, x, dtype=None):
    weight = layer.weight.detach() if dtype is None else layer.weight.detach().to(dtype)
    group, zeros = layer.format
    return fo.int4_linear(x, *fo.quantize_int4(weight, group, zeros=zeros), layer.bias)


def _is_current(layer, x=None):
    x = _x() if x is None else x
    return torch.equal(layer(x), _own(layer, x))


def _double(layer):
    with torch.no_grad():
        layer.weight.mul_(2)


def _load(layer):
    layer.load_state_dict({name: value + 1 for name, value in layer.state_dict().items()})


def _assign(layer):
    layer.load_state_dict({name: value + 1 for name, value in layer.state_dict().items()}, assign=True)


def _replace(layer):
    layer.weight = torch.nn.Parameter(layer.weight + 1)


def _data(layer):
    layer.weight.data = layer.weight.data + 1


def _step(layer):
    layer.weight.grad = torch.ones_like(layer.weight)
    torch.optim.SGD([layer.weight], lr=1.0).step()


@pytest.mark.parametrize("change", [_double, _load, _assign, _replace, _data, _step])
def test_codes_follow_the_weight(layer, change):
    before = layer(_x())
    assert _is_current(layer)
    change(layer)
    assert not torch.equal(layer(_x()), before) and _is_current(layer)
    for got, want in zip(layer.quantized_weight(), fo.quantize_int4(layer.weight, layer.format[0], zeros=layer.format[1])):
        assert got is want is None or torch.equal(got, want)


@pytest.mark.parametrize("change", [_double, _load, _data])
def test_input_gradient_is_that_of_the_forwards_weight(layer, change):
    change(layer)
    x, gy = _x().requires_grad_(), torch.randn(9, 130, device="cuda").bfloat16()
    got, = torch.autograd.grad(layer(x), x, gy)
    want, = torch.autograd.grad(_own(layer, x), x, gy)
    assert torch.equal(got, want) and layer.weight.grad is None


def test_swapped_weight_for_one_call(layer):
    own = layer(_x())
    other = {"weight": layer.weight.detach() + 1, "bias": layer.bias}
    got = torch.func.functional_call(layer, other, (_x(),))
    group, zeros = layer.format
    assert torch.equal(got, fo.int4_linear(_x(), *fo.quantize_int4(other["weight"], group, zeros=zeros), layer.bias))
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
    with torch.no_grad():
        layer(x)
        kept = [None if t is None else t.data_ptr() for t in layer.quantized_weight()]
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
            assert kept == [None if t is None else t.data_ptr() for t in layer.quantized_weight()]


def test_change_that_a_capture_meets(layer):
    """Codes that are out of date when a graph is captured: each replay quantizes the weight as it is then."""
    x = _x()
    with torch.no_grad():
        layer(x)
        _double(layer)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer(x)
        assert _is_current(layer)
        for _ in range(3):
            _double(layer)
            want = _own(layer, x)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want)


def test_inference_mode(layer):
    with torch.inference_mode():
        _double(layer)
        assert _is_current(layer)
        layer.quantize_weight_()
        made = torch.nn.Linear(300, 130, device="cuda", dtype=torch.bfloat16)
        fo.to_int4_linear(made, *layer.format)
        made.format = layer.format
        assert _is_current(made)
    _double(layer)
    assert _is_current(layer) and _is_current(layer)


@pytest.mark.parametrize("swap", [False, True])
@pytest.mark.parametrize("move", [lambda m: m.half(), lambda m: m.float().bfloat16(), lambda m: m.to("cuda"),
                                  lambda m: torch.nn.Sequential(m).float()[0].half(), lambda m: m.cpu().cuda(),
                                  lambda m: m.cpu().half().cuda()])
def test_in_another_type_or_on_another_device(layer, move, swap):
    before = torch.__future__.get_swap_module_params_on_conversion()
    torch.__future__.set_swap_module_params_on_conversion(swap)
    try:
        moved = move(layer)
    finally:
        torch.__future__.set_swap_module_params_on_conversion(before)
    assert moved is layer and layer.weight_int4.dtype == torch.uint8 and layer.weight_scale.dtype == layer.weight.dtype
    assert _is_current(layer, _x().to(layer.weight.dtype))


def test_in_fp32(layer):
    """16-bit codes and scales of a weight in fp32."""
    want = layer(_x())
    layer.float()
    assert torch.equal(layer(_x()), want) and layer.weight_scale.dtype == torch.bfloat16
    _double(layer)
    assert torch.equal(layer(_x()), _own(layer, _x(), torch.bfloat16))


@pytest.mark.parametrize("change", [_double, _load])
def test_a_compiled_layer_sees_the_change(layer, change):
    x = _x().requires_grad_()
    compiled = torch.compile(layer, backend="aot_eager", fullgraph=True)
    assert torch.equal(compiled(x), layer(x))
    change(layer)
    y = compiled(x)   # before the layer itself is called
    want = _own(layer, x)
    gy = torch.randn_like(want)
    assert torch.equal(y, want)
    assert torch.equal(*(torch.autograd.grad(t, x, gy)[0] for t in (y, want)))
    assert _is_current(layer) and torch.equal(compiled(x), want)
    layer.bias.requires_grad_(False)
    assert layer.weight.requires_grad and not torch.compile(layer, backend="aot_eager")(x.detach()).requires_grad


def test_a_weight_that_was_let_go(layer):
    """To save its memory: the codes stay as they are."""
    want = layer(_x())
    kept = layer.weight.detach().clone()
    layer.weight.data = layer.weight.data.cpu()
    assert torch.equal(layer(_x()), want)
    layer.weight.data = torch.empty(0, dtype=torch.bfloat16, device="cuda")
    assert torch.equal(layer(_x()), want)
    layer.weight = None
    assert torch.equal(layer(_x()), want) and torch.equal(layer.to("cuda")(_x()), want)
    layer.weight = torch.nn.Parameter(kept * 2)
    assert _is_current(layer)


def test_format_is_kept(layer):
    layer.cpu()
    assert {t.device.type for t in (layer.weight, layer.weight_int4, layer.weight_scale)} == {"cpu"}
    layer.cuda()
    _double(layer)
    layer.quantize_weight_()
    assert _is_current(layer)
    layer.quantize_weight_(64, True)
    layer.format = (64, True)
    assert _is_current(layer)
