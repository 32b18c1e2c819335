"""The bindings of the paged serving steps: streams, scratch, devices and outputs (no reference counterpart)."""
import numpy as np
import pytest

import kvdecode as kvd
from test_blocks import DEV, _same_plan, plan_inputs, plan_oracle


@pytest.mark.gpu
@pytest.mark.parametrize("as_handle", [False, True])
def test_plan_on_a_side_stream_without_a_workspace(as_handle):
    """The workspace is zeroed on the stream that the plan runs on: work that waits on the current stream, and what
    the workspace's memory held before, change nothing. 20,000 slots are many CTAs, which count themselves in it."""
    import torch

    args = plan_inputs(3, 64, 16, 600, 4000, 2, 8, 7000)
    lens, new, table, free = (torch.from_numpy(a).to(DEV) for a in args[:4])
    count = torch.tensor([args[4]], dtype=torch.int32, device=DEV)
    slots = torch.full((20000,), 77, dtype=torch.int64, device=DEV)
    starts = torch.empty(65, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    stale = [torch.full((16,), 255, dtype=torch.uint8, device=DEV) for _ in range(64)]
    torch.cuda.synchronize()
    del stale
    torch.cuda._sleep(40_000_000)  # tens of milliseconds
    kvd.paged_plan(lens, new, table, free, count, 16, slots, starts,
                   stream=side.cuda_stream if as_handle else side)
    side.synchronize()
    torch.cuda.synchronize()
    got = (*(t.cpu().numpy() for t in (table, free)), int(count), *(t.cpu().numpy() for t in (lens, starts, slots)),
           kvd.device_status())
    _same_plan(got, plan_oracle(*args, 16, 20000))
