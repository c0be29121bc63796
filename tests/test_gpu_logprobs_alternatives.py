"""GPU test of the log probabilities' two outputs of alternatives, which go together."""
import pytest

import fyodor_b200 as F

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

from .test_gpu_logprobs import i32, outputs, some  # noqa: E402


def test_alternatives_go_together():
    """Probabilities without tokens, or of another width, were not written, or not where they were looked for."""
    x, t = some(4, 900, 6)
    ws = F.logprobs_workspace(4, 900, 5)
    good = dict(logits=x, tokens=i32(t), workspace=ws) | outputs(4, 3)
    for bad in (dict(top_tokens=None), dict(top_logprobs=None), dict(top_tokens=torch.zeros((4, 0), dtype=torch.int32, device="cuda")),
                dict(top_logprobs=torch.zeros((4, 5), device="cuda")), dict(top_logprobs=torch.zeros((4, 3), device="cuda").cpu()),
                dict(top_logprobs=torch.zeros((4, 3), device="cuda").half())):
        with pytest.raises(ValueError):
            F.logprobs(**(good | bad))
    empty = dict(top_tokens=torch.zeros((4, 0), dtype=torch.int32, device="cuda"), top_logprobs=torch.zeros((4, 0), device="cuda"))
    for fine in (dict(top_tokens=None, top_logprobs=None), empty, empty | dict(top_logprobs=None),
                 dict(top_tokens=None, top_logprobs=empty["top_logprobs"]),
                 dict(top_logprobs=torch.zeros((6, 3), device="cuda"))):  # room for more rows
        F.logprobs(**(good | fine))
