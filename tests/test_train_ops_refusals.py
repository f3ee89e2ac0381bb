"""Arguments that the training operators (models/train_ops.py) refuse, checked before any
launch: these run without a GPU."""
import pytest
import torch

from smsgate_amd.models import train_ops


def _ids(*shape, dtype=torch.long):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("ids,table,add,err", [
    (_ids(3), torch.zeros(4), None, TypeError),                                     # table not 2-D
    (_ids(3), torch.zeros(4, 8, dtype=torch.float64), None, TypeError),             # a type without a kernel
    (_ids(3, dtype=torch.int16), torch.zeros(4, 8), None, TypeError),
    (torch.zeros(3), torch.zeros(4, 8), None, TypeError),                           # ids are whole numbers
    (_ids(3), torch.zeros(4, 8), _ids(4), ValueError),                              # add_ids of another shape
    (_ids(3), torch.zeros(4, 8), _ids(3, dtype=torch.int32), ValueError),           # or type
    (_ids(3), torch.zeros(0, 8), None, ValueError),                                 # an empty table
    (_ids(3), torch.zeros(4, 8), None, ValueError),                                 # not on a GPU
])
def test_embed_lookup_refuses(ids, table, add, err):
    with pytest.raises(err, match="embed_lookup"):
        train_ops.embed_lookup(ids, table, add)
