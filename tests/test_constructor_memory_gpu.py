"""What a graph constructor's captures reserve goes back when it is gone."""
import gc

import pytest
import torch

from intrasm_engine_amd.pytorch.cpp_extensions.cuda_graph_constructor import TorchCUDAGraphConstructor

pytestmark = pytest.mark.gpu


def test_pools_of_several_captures_are_given_back(dev):
    """Three recordings into one constructor, replayed, dropped: nothing stays reserved, however often."""
    a, b = torch.randn(256, 128, device=dev).half(), torch.randn(128, 192, device=dev).half()
    want = torch.ops.iex_ops.gemm_mfma(a, b, False)

    def once():
        constructor = TorchCUDAGraphConstructor()
        outs = []
        for _ in range(3):
            with constructor.get_primary_stream():
                constructor.capture_library_call_begin()
                try:
                    outs.append(torch.ops.iex_ops.gemm_mfma(a, b, False))
                finally:
                    constructor.capture_library_call_end()
        constructor.instantiate_graph_exec()
        constructor.execute_graph()
        constructor.synchronize()
        assert all(torch.equal(out, want) for out in outs)
        constructor.destroy_graph_exec()

    def reserved():
        gc.collect()
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        return torch.cuda.memory_reserved()

    once()
    before = reserved()
    for _ in range(8):
        once()
    assert reserved() <= before
