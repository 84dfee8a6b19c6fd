"""What the expert layer refuses, without a GPU: nothing may be queued for such a call, since the exchange is collective and writes where it is told to."""
from types import SimpleNamespace

import pytest
import torch

from hcomm_b200.parallel.ep import ExpertParallelMlp


def layer():
    made = ExpertParallelMlp.__new__(ExpertParallelMlp)
    made.router = torch.zeros(8, 512, dtype=torch.bfloat16)
    made.moe = SimpleNamespace(hidden=512, max_tokens=16)
    return made


BF16 = torch.bfloat16
X = torch.zeros(4, 512, dtype=BF16)


@pytest.mark.parametrize("x", [X.float(), X[0], torch.zeros(4, 256, dtype=BF16), torch.zeros(4, 1024, dtype=BF16)[:, ::2], torch.zeros(4, 1024, dtype=BF16)[:, :512], X.to("meta"),
                               torch.zeros(17, 512, dtype=BF16)])
def test_tokens(x):
    with pytest.raises(ValueError):
        layer()(x)


@pytest.mark.parametrize("x", [X, X[:0]])
@pytest.mark.parametrize("out", [torch.zeros(4, 512), torch.zeros(4, 256, dtype=BF16), torch.zeros(2048, dtype=BF16),
                                 torch.zeros(512, 4, dtype=BF16).t(), torch.zeros(4, 1024, dtype=BF16)[:, :512], X.to("meta")])
def test_results(x, out):
    with pytest.raises(ValueError, match="out"):
        layer()(x, out)


def test_a_result_of_too_few_rows():
    with pytest.raises(ValueError, match="out"):
        layer()(X, torch.zeros(3, 512, dtype=BF16))
