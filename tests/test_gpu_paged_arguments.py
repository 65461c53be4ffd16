"""The paged operators' answers to unusual arguments."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from tensor_fusion_amd.ops import paged

from paged_oracle import Batch, check

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
KEPT = pytest.mark.parametrize("quantized", [False, True],
                               ids=["wide", "e4m3"])


def test_results_under_a_mode_that_fakes_tensors():
    """Real arguments, but what would be allocated for the result has no
    memory: refused, and nothing is launched."""

    b = Batch([(1, 40), (2, 30)], 4, 2, 64, 16, BF16, False, seed=1)
    q, starts = b.q.cuda(), b.q_starts.cuda()
    lens, table = b.kv_lens.cuda(), b.table.cuda()
    slots = torch.arange(4, device="cuda")
    with FakeTensorMode():
        with pytest.raises(ValueError, match="plain tensor"):
            paged.paged_attention(q, b.cache, starts, lens, table)
        with pytest.raises(ValueError, match="plain tensor"):
            paged.kv_read(b.cache, slots)
    check(paged.paged_attention(q, b.cache, starts, lens, table), *b.want())
