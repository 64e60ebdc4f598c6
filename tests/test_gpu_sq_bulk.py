"""Large writes of scalar-quantised rows with slots that repeat and slots outside
the store: of the rows that name a slot the last stays, whole.  Up to 16384
rows one cluster decides, from there on two launches do; above some 2.4 million
rows a thread of those takes several rounds of rows."""
import pytest
import torch

import insitu_b200 as ib

pytestmark = pytest.mark.gpu


def reference(x):
    """(codes, scales) of fp32 rows at 8 bits: the fp32 quotient max / 127, then the quotient in 64 bits to the nearest"""
    top = x.abs().amax(1)
    scale = (top.double() / 127).float()         # of two fp32 numbers: rounding the 64-bit quotient gives the fp32 one
    q = torch.round(x.double() / torch.where(scale > 0, scale, 1.0).double()[:, None])
    return q.clamp_(-127, 127).to(torch.int8), scale


@pytest.mark.parametrize("n,capacity", [(16383, 5000), (16384, 16384), (16385, 16385), (16385, 3), (40000, 1000003),
                                        (1200001, 700000), (2500001, 2000003)])
@pytest.mark.parametrize("hot", [0.0, 0.3])
def test_last_of_repeated_slots_stays(cuda_ok, n, capacity, hot):
    d = 17
    g = torch.Generator(device="cuda").manual_seed(n + capacity)
    x = torch.randn(n, d, generator=g, device="cuda")
    # a twentieth of the slots outside, on both sides; `hot` of the rows meet in a few slots
    slots = torch.randint(-(capacity // 40) - 1, capacity + capacity // 40 + 1, (n,), generator=g, device="cuda")
    few = torch.randint(0, min(capacity, 5), (n,), generator=g, device="cuda") * (capacity // 5) % capacity
    slots = torch.where(torch.rand(n, generator=g, device="cuda") < hot, few, slots)
    slots[n // 2] = 1 << 40
    codes = torch.full((capacity, 32), 99, dtype=torch.int8, device="cuda")
    scales = torch.full((capacity, 1), -5.0, device="cuda")
    store = ib.SQRows.from_arrays(codes, scales, d)

    inside = (slots >= 0) & (slots < capacity)
    last = torch.full((capacity + 1,), -1, device="cuda")
    last.scatter_reduce_(0, torch.where(inside, slots, capacity), torch.arange(n, device="cuda"), "amax")
    last = last[:-1]
    q, s = reference(x)
    want_codes, want_scales = codes.clone(), scales.clone()
    named = last >= 0
    want_codes[named, :d] = q[last[named]]
    want_scales[named, 0] = s[last[named]]
    for _ in range(3):                                   # what an earlier write left in the table does not count
        store.write(x, slots)
        assert torch.equal(codes, want_codes) and torch.equal(scales, want_scales)
        codes.fill_(99)
        scales.fill_(-5.0)
