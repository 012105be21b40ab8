"""paged_prefix_attention of a batch with an entry of cu_new out of its bounds: the call is
flagged, and the rows of the group's other sequences are what they are without it - nothing of
them comes from what the workspace held before."""
import pytest
import torch

import heteromm_b200 as hmm
from test_prefix_attention_gpu import groups_of, ints, shared, with_join
from test_serve_attention_gpu import check, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("offsets,good", [
    ([0, 1, 2, 99, 99], [0, 1]),       # the group's end lies behind the batch
    ([0, 1, 2, -3, 4], [0, 1]),        # and before it
    ([-1, 1, 2, 3, 4], [1, 2, 3]),     # its begin
    ([0, 1, 2, 3, -9], [0, 1, 2]),
    ([0, -5, 2, 3, 4], [2, 3]),
    ([0, 1, 2, 1 << 30, 4], [0, 1]),
    ([0, 1, 2, 1, 4], [0]),            # one that descends (rows 1 to 3 are two sequences')
])
@pytest.mark.parametrize("members", [3, 4])
def test_the_others_of_a_group(cuda, offsets, good, members):
    new, kv = [1, 1, 1, 1], [200, 170, 161, 300]
    groups = [(0, members, 128)]
    q, k, v, table, cu, kv_len, (cg, pl) = shared(cuda, 90, groups, new, kv, 8, 2, 128, 16, torch.bfloat16)
    ref = with_join(reference(q, k, v, table, new, kv))
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    for fill in (float("nan"), 1e30, 0.0):
        torch.full((32 << 20,), fill, device=cuda)       # what a workspace may find
        out, lse = hmm.paged_prefix_attention(q, k, v, table, ints(offsets, cuda), kv_len, cg, pl, return_lse=True,
                                              status=status.zero_())
        assert status.item() == 16
        check(out[good], lse[good], tuple(x[good] for x in ref))


def test_rows_behind_the_groups_end(cuda):
    """cu_new descends within a group: its first sequence's last rows lie behind the group's."""
    new, kv = [5, 1, 1], [200, 170, 161]
    groups = [(0, 3, 128)]
    q, k, v, table, cu, kv_len, (cg, pl) = shared(cuda, 91, groups, new, kv, 8, 2, 64, 16, torch.bfloat16)
    ref = with_join(reference(q, k, v, table, new, kv))
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    for fill in (float("nan"), 1e30):
        torch.full((32 << 20,), fill, device=cuda)
        out = torch.full_like(q, 9.0)
        hmm.paged_prefix_attention(q, k, v, table, ints([0, 5, 2, 3], cuda), kv_len, cg, pl, out=out, status=status.zero_())
        assert status.item() == 16
        check(out[:2], None, tuple(x[:2] for x in ref))
        check(out[3:5], None, tuple(x[3:5] for x in ref))
