"""Every decode-attention kernel gets its own shared-memory limit, whichever kernel ran before it in the process."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

SCRIPT = """
import sys
sys.path[:0] = [{pkg!r}]
import torch
from llama import fused

def step(heads, d, seq, batch):
    gen = torch.Generator(device="cuda").manual_seed(heads + d)
    q = torch.randn(batch, heads * d, generator=gen, device="cuda").half()
    k, v = (torch.randn(batch, seq, 1, d, generator=gen, device="cuda").half() for _ in range(2))
    out, pos = torch.empty_like(q), torch.tensor([seq - 1], device="cuda")
    fused.decode_attention(q, k, v, pos, out, heads, 1)
    p = torch.softmax(torch.einsum("bhd,bsd->bhs", q.view(batch, heads, d).double(), k[:, :, 0].double()) / d ** 0.5, -1)
    want = torch.einsum("bhs,bsd->bhd", p, v[:, :, 0].double()).reshape(batch, -1)
    err = float((out.double() - want).abs().max())
    assert err <= 2e-3 * float(v.abs().max()), (heads, d, err)

# enough sequences that each has one CTA; the first needs the most shared memory, the others less, of other kernels
for heads, d, seq in ((8, 128, 150), (4, 128, 150), (2, 128, 150), (1, 128, 150), (8, 64, 300), (4, 64, 300)):
    step(heads, d, seq, 400)
print("ok")
"""


def test_kernels_of_one_signature_raise_their_own_limit(cuda_device):
    import build

    build.build()
    r = subprocess.run([sys.executable, "-c", SCRIPT.format(pkg=build.PKG_DIR)], capture_output=True, text=True,
                       timeout=300, env=dict(os.environ))
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stderr[-2000:]
