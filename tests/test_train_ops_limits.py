"""Layouts and sizes of the training operators (models/train_ops.py) at their limits, checked
before any launch: these run without a GPU."""
import pytest
import torch

from smsgate_amd.models import train_ops


def test_rows_of_one_position_are_moved_to_16_bytes():
    """One head and one position: contiguous by torch's rules whatever its strides and start."""
    base = torch.arange(3 * 65, dtype=torch.float32).bfloat16()
    for t in (base[:65].view(1, 1, 1, 65)[..., 1:], base[1:65].view(1, 1, 1, 64), base[65:130].view(1, 1, 1, 65)[..., :64]):
        r = train_ops._rows16(t)
        assert r.data_ptr() % 16 == 0 and r.stride(3) == 1 and torch.equal(r, t)


def test_rows_that_fit_are_not_copied():
    t = torch.zeros(2, 10, 3, 64, dtype=torch.bfloat16).transpose(1, 2)
    assert train_ops._rows16(t).data_ptr() == t.data_ptr()


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_sizes_beyond_a_launch_are_refused():
    """A grid holds 2^32 threads."""
    with pytest.raises(ValueError, match=r"2\^26"):
        train_ops.embed_lookup(_meta(1 << 26, dtype=torch.int32), _meta(100, 8))
    with pytest.raises(ValueError, match=r"2\^26"):
        train_ops.embed_lookup(_meta(5, dtype=torch.int32), _meta(1 << 26, 8))
    q = _meta(1, 1 << 10, 1 << 21, 64)
    with pytest.raises(ValueError, match=r"2\^24 tiles"):
        train_ops.tiled_attention(q, q, q)
    with pytest.raises(ValueError, match=r"2\^24 tiles"):
        train_ops.lm_loss(_meta(1 << 20, 8), _meta(1 << 21, 8), _meta(1 << 20, dtype=torch.long))
    with pytest.raises(ValueError, match=r"2\^34"):
        train_ops.lm_loss(_meta(1 << 20, 1 << 14), _meta(8, 1 << 14), _meta(1 << 20, dtype=torch.long))


@pytest.mark.parametrize("scale", [1e39, 1e-46])
def test_scales_that_32_bits_do_not_hold_are_refused(scale):
    q = _meta(1, 2, 4, 64)
    with pytest.raises(ValueError, match="scale"):
        train_ops.tiled_attention(q, q, q, scale)
