"""Evictions whose keys and places fill the shared memory that a kernel gets without asking, in a process that has asked for none."""

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

CALLS = """
import torch
from calibquant_b200 import ops
for t_fp, keep in {tokens}:
    k = torch.randn(1, 1, t_fp, 128, device="cuda").half()
    w = torch.rand(1, 1, t_fp, device="cuda")
    k2, v2, w2, kept = ops.evict_tokens(k, -k, w, keep)
    want = torch.sort(torch.sort(w, descending=True, stable=True).indices[..., :keep]).values
    assert torch.equal(kept, want) and torch.equal(k2[0, 0], k[0, 0][want[0, 0]]) and torch.equal(v2, -k2)
for bits in (1, 2, 4):
    for groups, keep in {groups}:
        word = lambda *s: torch.randint(-2 ** 31, 2 ** 31 - 1, s, dtype=torch.int32, device="cuda")
        num = lambda *s: torch.randn(*s, device="cuda").half()
        kp = word(1, 1, 128, groups * bits), num(1, 1, 128, groups), num(1, 1, 128, groups)
        vp = word(1, 1, 32 * groups, 4 * bits), num(1, 1, 32 * groups, 4), num(1, 1, 32 * groups, 4)
        w = torch.randint(0, 1 << 20, (1, 1, 32 * groups), device="cuda").float()      # exact sums
        k2, v2, w2, kept = ops.evict_groups(kp, vp, w, keep, bits=bits)
        want = torch.sort(torch.sort(w.unflatten(-1, (-1, 32)).sum(-1), descending=True, stable=True).indices[..., :keep]).values
        assert torch.equal(kept, want) and torch.equal(k2[1], kp[1][..., want[0, 0]]) and torch.equal(v2[1].view(-1, 128), vp[1].view(-1, 128)[want[0, 0]])
"""


@pytest.mark.parametrize("tokens,groups", [([(6144, 6144)], []), ([(8000, 4000)], []), ([], [(4096, 4096)]), ([], [(4100, 3800)]),
                                           ([(11700, 100), (5000, 5000)], [(4000, 3700), (3000, 2000)])], ids=str)
def test_keys_and_places_of_48_kilobytes(tokens, groups):
    """4 bytes a token and a kept one, 8 bytes a group and 4 a kept one: 47 to 48 KB together, and a little less."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", CALLS.format(tokens=tokens, groups=groups)], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
