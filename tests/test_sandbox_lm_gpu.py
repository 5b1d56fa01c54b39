"""GPU sandbox test of the language-model operators: a user's script imports
hipmx and hiplm next to torch and runs on the kernels."""

import asyncio

import pytest

pytestmark = pytest.mark.gpu

SCRIPT = """
import torch
import hipmx, hiplm, hiptorch

torch.manual_seed(0)
head = hipmx.quantize(torch.randn(5000, 512, device="cuda"))
x = torch.randn(40, 512, device="cuda", dtype=torch.bfloat16)
with torch.no_grad():
    logits = torch.nn.functional.linear(x, head)
said = hiplm.token_logprobs(logits, logits.argmax(-1), top=8)
assert torch.equal(said.top_tokens[:, 0], logits.argmax(-1))
student = torch.zeros(40, 5000, device="cuda", requires_grad=True)
loss = hiplm.topk_distill_loss(student, said.top_logprobs, said.top_tokens)
loss.backward()
# a student that knows nothing: p = 1 / 5000 everywhere
q = torch.softmax(said.top_logprobs, -1)
want = torch.full((40, 5000), 1 / 5000, device="cuda")
want.scatter_add_(1, said.top_tokens, -q)
torch.testing.assert_close(student.grad, want / 40, rtol=1e-5, atol=1e-8)
assert hipmx.STATS["linear"] == 1, hipmx.STATS
assert hiplm.STATS["topk_distill_loss"] == 1, hiplm.STATS
print("lm-ok", hiptorch._hiplm.__name__)
"""


def test_operators_in_a_sandbox(gpu_executor):
    r = asyncio.run(gpu_executor.execute(
        SCRIPT, env={"APP_HIP_TORCH": "require"}))
    assert r.exit_code == 0, r.stderr
    assert r.stdout.strip() == "lm-ok _hiplm"
