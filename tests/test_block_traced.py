"""Programs that make_fx traces from the block-scaled product, without a GPU: their own workspace, of which the arrival counters
are cleared in each run and no more."""

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

import feather_ops as fo
from feather_ops.block_scaled import _COUNTER_BYTES, _workspace_bytes

M, N, K = 512, 1024, 5120


@pytest.mark.parametrize("mode", ["fake", "symbolic"])
def test_only_the_counters_are_cleared(mode):
    f8, f32 = torch.float8_e4m3fn, torch.float32
    args = [torch.empty(shape, dtype=dtype) for shape, dtype in (((M, K), f8), ((M, 40), f32), ((N, K), f8), ((8, 40), f32))]
    graph = make_fx(lambda *a: fo.block_scaled_mm(*a), tracing_mode=mode)(*args).graph
    need = _workspace_bytes(M, N, K)
    assert need > 1 << 20
    nodes = [node for node in graph.nodes if node.op == "call_function"]
    made, part, cleared, product = nodes
    assert str(made.target) == "aten.empty.memory_format" and made.args[0] == [need]
    assert part.args[0] is made and part.args[-1] == _COUNTER_BYTES
    assert str(cleared.target) == "aten.zero_.default" and cleared.args == (part,)
    assert str(product.target) == "feather_ops.block_scaled_mm.default" and product.args[-1] is made
    again = torch.fx.GraphModule({}, graph)
    again.graph.eliminate_dead_code()
    assert len([node for node in again.graph.nodes if node.op == "call_function"]) == 4
