"""The last sizes that embed_lookup (models/train_ops.py) takes and the first that it refuses: a
wave a row and 4 waves a block, a grid holds 2^32 - 1 threads.  Without a GPU."""
import pytest
import torch

from smsgate_amd import ops
from smsgate_amd.models import train_ops

LAST = (1 << 26) - 4  # 2^24 - 1 blocks of 256 threads


def _call(n, V):
    train_ops.embed_lookup(torch.empty(n, dtype=torch.int32, device="meta"), torch.empty(V, 1, device="meta"))


@pytest.mark.parametrize("n,V", [(LAST, 5), (5, LAST), (LAST, LAST)])
def test_last_sizes_pass_the_checks(n, V):
    with pytest.raises(ValueError, match="same GPU"):  # the check behind the sizes'
        _call(n, V)
    assert (max(n, V) + 3) // 4 * 256 < 1 << 32


@pytest.mark.parametrize("n,V", [(LAST + 1, 5), (5, LAST + 1), (LAST + 3, 5), (5, LAST + 3)])
def test_first_sizes_beyond_are_refused(n, V):
    with pytest.raises(ValueError, match=r"2\^26"):
        _call(n, V)
    assert (max(n, V) + 3) // 4 * 256 >= 1 << 32


@pytest.mark.parametrize("n,V", [(LAST + 1, 5), (5, LAST + 1)])
def test_entries_refuse_them_before_any_launch(n, V):
    if not ops.have_kernels():
        pytest.skip("no kernel library")
    lib = ops.load_library()
    assert lib.sg_embed_fwd(None, None, 0, None, None, n, V, 1, 1.0, 0, 0, None) == 1
    assert lib.sg_embed_grad(None, None, 0, None, None, n, V, 1, 1.0, 0, 0, None, 0, None) == 1
