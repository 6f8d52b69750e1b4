"""Generation on the 4-bit cache where a step cannot be recorded."""
import pytest
import torch

from tests import test_gpu_packed_model as M
from tests.gpu_util import assert_no_kernel_error

pytestmark = pytest.mark.gpu


def test_steps_that_cannot_be_recorded_run_one_by_one(cuda, monkeypatch):
    model = M.runner(cuda, heads=4, kv_heads=2, H=64)
    ids = M.prompts(cuda, [20, 3])
    want = model.generate_packed(ids, 8, use_graph=False)
    tried = []

    class NoGraph:
        def __init__(self, *a, **kw):
            tried.append(1)

        def __enter__(self):
            raise RuntimeError("recording is not supported")

        def __exit__(self, *a):
            return False

    monkeypatch.setattr(torch.cuda, "graph", NoGraph)
    with pytest.warns(UserWarning, match="decoding eagerly"):
        got = model.generate_packed(ids, 8)
    assert len(tried) == 1 and all(torch.equal(a, b) for a, b in zip(got, want))
    assert_no_kernel_error()
