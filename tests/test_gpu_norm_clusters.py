"""Norms and joins of widths that clusters share, at the batch sizes where a cluster begins to hold several rows, against FP64."""
import pytest
import torch

import test_gpu_norm as base

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("n", [5120, 9216, 12288])
@pytest.mark.parametrize("T,pad,dt,kind", [(34, 0, HF, "layer"), (75, 1, BF, "rms"), (100, 0, BF, "layer"), (148, 0, BF, "rms"), (223, 8, HF, "layer")])
def test_norm(cuda, n, T, pad, dt, kind):
    base.test_forward_and_backward(cuda, T, n, pad, dt, kind)


@pytest.mark.parametrize("n", [5120, 9216, 12288])
@pytest.mark.parametrize("T,pad,dt,post,gate,pre", [(34, 0, BF, "layer", "vector", "layer"), (75, 0, BF, "rms", "vector", "rms"), (100, 1, HF, "layer", "matrix", "none"),
                                                    (148, 0, HF, "none", "matrix", "layer"), (223, 8, BF, "rms", "none", "rms")])
def test_join(cuda, n, T, pad, dt, post, gate, pre):
    base.test_join_and_its_gradients(cuda, post, gate, pre, T, n, pad, dt, None)
