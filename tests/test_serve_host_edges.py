"""Refusals of the serving decoder's operators, without a GPU: tensors that share
memory from another offset than their own."""
import numpy as np
import pytest

from test_decode_host import ARG, T, refused
from test_serve_host import plan_args

I32, I64 = np.int32, np.int64


@pytest.mark.parametrize("over", [  # (starts lie at 3000 to 3003, counts at 4000 to 4003 in 64 bits)
    dict(lengths=T((4,), I32, None, 2997)),
    dict(lengths=T((4,), I32, None, 3003)),
    dict(granted=T((4,), I32, None, 8007)),
    dict(granted=T((4,), I32, None, 7997)),
    dict(granted=T((4,), I32, None, 2997), starts=T((4,), I32, (-1,), 3003)),
    dict(granted=T((4,), I32, None, 3003), starts=T((4,), I32, (-1,), 3003)),
    dict(lengths=T((4,), I32, None, 3027), starts=T((4,), I32, (10,), 3000)),
    dict(lengths=T((4,), I32, None, 3010), starts=T((4,), I32, (10,), 3000)),
    dict(lengths=T((4,), I32, None, 2998), starts=T((1,), I32, None, 3001)),
    dict(lengths=T((4,), I32, None, 1000), granted=T((4,), I32, None, 1003)),
    dict(lengths=T((4,), I32, None, 5000), free=T((30,), I32, None, 4971)),
    dict(granted=T((4,), I32, None, 5000), used=T((1,), I32, None, 5003))])
def test_plan_pages_refuses_outputs_that_lie_in_what_it_reads(over):
    refused("kk_plan_pages", plan_args(**over), ARG, "lengths and granted must not")
