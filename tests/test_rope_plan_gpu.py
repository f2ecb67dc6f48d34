"""A rotary plan is on the device when its creation returns, whatever the streams do."""
import pytest
import torch

import block_ref as R
from crispembed_b200 import binding

pytestmark = pytest.mark.gpu


def test_plan_is_made_apart_from_the_default_stream(cuda):
    """Its upload is no part of the default stream, which side streams do not wait for: with work
    queued there, creation returns before that work has ended."""
    binding.Rope(64).close()
    torch.cuda.synchronize()
    done = torch.cuda.Event()
    torch.cuda._sleep(1_000_000_000)  # about half a second
    done.record()
    rope = binding.Rope(64)
    early = not done.query()
    torch.cuda.synchronize()
    assert early
    rope.close()


def test_plans_used_at_once_on_other_streams(cuda):
    x = torch.randn(40, 3, 64, device=cuda)
    pos = torch.arange(40, dtype=torch.int32)
    dpos = pos.to(cuda)
    torch.cuda.synchronize()
    outs = []
    for i in range(30):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            rope = binding.Rope(64, theta=1000.0 + 500 * i)
            outs.append((rope, rope(x, positions=dpos)))
    torch.cuda.synchronize()
    for i, (rope, out) in enumerate(outs):
        R.check(out, *R.rope(x, pos, 64, False, *R.frequencies(64, theta=1000.0 + 500 * i)))
