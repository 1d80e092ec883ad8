"""Row lengths of the relation weights at which a kernel's shared memory, the part that the launch asks for and the
part that it holds anyway, first passes the 48 KB that need no permission.

The permission lasts as long as the process: each case is the first of its kernel in a process of its own.
"""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# dtype, n, mask, history: rows that one block keeps in registers (256 and 512 threads), and the two-pass form
SIZES = [("float32", 6860, True, True), ("float32", 8010, False, True), ("float32", 9800, True, False),
         ("float32", 12253, False, False), ("float32", 12284, False, False), ("bfloat16", 9400, True, True),
         ("bfloat16", 11750, False, True), ("bfloat16", 16350, True, False), ("float16", 9380, True, True),
         ("float16", 16330, True, False), ("float32", 23010, False, True), ("bfloat16", 23100, False, True)]

SCRIPT = """
import math, sys
import torch
from flashlog_b200 import attention
bad = []
for dt, n, masked, used in {sizes!r}:
    g = torch.Generator().manual_seed(n)
    rows = 400  # more than the few rows that a cluster of blocks takes
    z = (torch.randn(rows, n, generator=g) * 1.5).to(getattr(torch, dt)).cuda()
    mask = (torch.rand(5, n, generator=g) < 0.4).cuda() if masked else None
    states = torch.randint(0, 5, (rows,), generator=g).cuda() if masked else None
    history = torch.randint(-1, n, (rows, 7), generator=g).cuda() if used else None
    try:
        w = attention.relation_weights(z, mask=mask, states=states, history=history, presence=0.5)
    except Exception as e:
        bad.append((dt, n, masked, used, str(e)))
        continue
    u = z.double()
    if used:
        seen = torch.zeros(rows, n + 1, dtype=torch.bool, device=z.device)
        seen.scatter_(1, torch.where(history < 0, n, history), True)
        u = u - 0.5 * seen[:, :n]
    if masked:
        u = u.masked_fill(~mask[states], -math.inf)
    # each weight: an exponent's argument off by a few roundings of values of at most 20, and a sum of positive terms
    if not bool(((w - torch.softmax(u, 1)).abs() <= 2.0 ** -16 * torch.softmax(u, 1) + 1e-38).all()):
        bad.append((dt, n, masked, used, "wrong"))
print(bad)
sys.exit(1 if bad else 0)
"""


def test_first_calls_around_48_kilobytes():
    p = subprocess.run([sys.executable, "-c", SCRIPT.format(sizes=SIZES)], cwd=ROOT, capture_output=True, text=True,
                       timeout=300)
    assert p.returncode == 0, p.stdout[-3000:] + p.stderr[-2000:]
