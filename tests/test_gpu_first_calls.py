"""Calls that are the first of their kernel in a process, at sizes whose shared memory is just under a kernel's default:
48 KB for what the launch asks for and what the kernel holds itself, together.  Past it a kernel needs an opt-in,
which stays for the process, so a larger call before would hide a missing one: each group of calls runs in a process
of its own."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]
SCRIPT = """
import sys
import torch
import mednext_accel_b200 as mx
from mednext_accel_b200 import _native as nat

def norm(rows, c, dtype, train):
    x = torch.randn((rows, c), device="cuda").to(dtype).requires_grad_(train)
    w = torch.ones(c, device="cuda", requires_grad=train)
    y = mx.layer_norm(x, w)
    torch.testing.assert_close(y, torch.nn.functional.layer_norm(x.float(), (c,), w, None, 1e-6).to(dtype),
                               rtol=2**-7, atol=2**-7)
    if train:
        dy = torch.randn_like(y)
        dx, dw = torch.autograd.grad(y, (x, w), dy)
        assert dx.isfinite().all() and dw.isfinite().all()

def product(tokens, k, dtype):
    x = torch.randn((tokens, k), device="cuda").to(dtype)
    q, s = mx.quantize_int8(torch.randn((24, k), device="cuda"))
    want = x.double() @ (q.double() * s.double()[:, None]).t()
    y = mx.int8_linear(x, q, s)
    assert (y.double() - want).norm() <= 0.02 * want.norm()

bf16, f16, f32 = torch.bfloat16, torch.float16, torch.float32
for call in sys.argv[1].split(";"):
    eval(call)
torch.cuda.synchronize()
assert nat.device_error() == 0
"""

# Rows of 5121 to 6144 columns, the weight grads' sums at 6144, blocks of odd rows just under a power of two, and a few
# tokens' 8-bit rows; the calls of a line reach different kernels.
GROUPS = [
    "norm(40, 6144, bf16, False);norm(40, 5122, f16, False);norm(40, 6000, f32, True)",
    "norm(40, 6144, bf16, True);norm(60001, 63, f16, True)",
    "norm(16001, 255, bf16, True);norm(16001, 511, f16, True)",
    "norm(30001, 127, bf16, False);norm(8001, 1023, f16, False)",
    "norm(4001, 2045, bf16, False);product(8, 6144, bf16);product(3, 16384, f16);product(6, 8192, f32)",
    "product(1, 49152, bf16);product(4, 12288, f32);product(2, 24570, f16)",
]


@pytest.mark.parametrize("calls", GROUPS)
def test_first_calls_near_the_default_shared_memory(calls):
    run = subprocess.run([sys.executable, "-c", SCRIPT, calls], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]
