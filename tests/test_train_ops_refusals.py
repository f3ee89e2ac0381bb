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
    (_ids(3), torch.empty(1, 1 << 21, device="meta"), None, ValueError),             # rows too wide
    (_ids(3), torch.zeros(4, 8), None, ValueError),                                 # not on a GPU
])
def test_embed_lookup_refuses(ids, table, add, err):
    with pytest.raises(err, match="embed_lookup"):
        train_ops.embed_lookup(ids, table, add)


def _qkv(B=2, T=5, nh=4, nkv=2, D=64, dtype=torch.bfloat16):
    return torch.zeros(B, nh, T, D, dtype=dtype), torch.zeros(B, nkv, T, D, dtype=dtype), \
        torch.zeros(B, nkv, T, D, dtype=dtype)


@pytest.mark.parametrize("change,kw,err", [
    (dict(dtype=torch.float32), {}, TypeError),
    (dict(D=80), {}, ValueError),
    (dict(nh=3), {}, ValueError),                                            # heads that do not divide
    (dict(T=0), {}, ValueError),
    (dict(B=0), {}, ValueError),
    ({}, dict(scale=0.0), ValueError),
    ({}, dict(scale=-1.0), ValueError),
    ({}, dict(scale=float("nan")), ValueError),
    ({}, dict(scale=float("inf")), ValueError),
    ({}, dict(lengths=torch.zeros(2, dtype=torch.int64)), ValueError),
    ({}, dict(lengths=torch.zeros(3, dtype=torch.int32)), ValueError),
    ({}, {}, ValueError),                                                    # not on a GPU
])
def test_tiled_attention_refuses(change, kw, err):
    with pytest.raises(err, match="tiled_attention"):
        train_ops.tiled_attention(*_qkv(**change), **kw)


def test_tiled_attention_refuses_mismatched_operands():
    q, k, v = _qkv()
    for bad in ((q, k[:1], v[:1]), (q, k[:, :, :4], v[:, :, :4]), (q, k, v[:, :1]), (q[0], k, v), (q, k[0], v[0])):
        with pytest.raises(ValueError, match="tiled_attention"):
            train_ops.tiled_attention(*bad)
    with pytest.raises(TypeError, match="tiled_attention"):
        train_ops.tiled_attention(q, k.half(), v)


@pytest.mark.parametrize("h,table,labels,kw,err", [
    (torch.zeros(3, 16), torch.zeros(4, 16), _ids(3), {}, TypeError),                       # fp32
    (torch.zeros(3, 16).half(), torch.zeros(4, 16).bfloat16(), _ids(3), {}, TypeError),     # two types
    (torch.zeros(3, 16).half(), torch.zeros(4, 16).half(), torch.zeros(3), {}, TypeError),  # labels are whole numbers
    (torch.zeros(3, 16).half(), torch.zeros(4, 16).half(), _ids(4), {}, ValueError),
    (torch.zeros(3, 16).half(), torch.zeros(4, 24).half(), _ids(3), {}, ValueError),
    (torch.zeros(3, 12).half(), torch.zeros(4, 12).half(), _ids(3), {}, ValueError),        # rows of no whole 16 bytes
    (torch.zeros(0, 16).half(), torch.zeros(4, 16).half(), _ids(0), {}, ValueError),
    (torch.zeros(3, 16).half(), torch.zeros(0, 16).half(), _ids(3), {}, ValueError),
    (torch.zeros(3, 16).half(), torch.zeros(4, 16).half(), _ids(3), dict(reduction="max"), ValueError),
    (torch.zeros(3, 16).half(), torch.zeros(4, 16).half(), _ids(3), dict(ignore_index=1 << 40), ValueError),
    (torch.zeros(3, 16).half(), torch.zeros(4, 16).half(), _ids(3), {}, ValueError),        # not on a GPU
])
def test_lm_loss_refuses(h, table, labels, kw, err):
    with pytest.raises(err, match="lm_loss"):
        train_ops.lm_loss(h, table, labels, **kw)


def test_hip_ops_is_a_training_option_that_needs_a_gpu():
    from smsgate_amd.cli import build_parser, train_config
    from smsgate_amd.models.train import FLAGSHIP_RECIPE, TrainConfig, train_extractor

    assert not FLAGSHIP_RECIPE.hip_ops
    args = ["train-extractor", "--out", "x.safetensors"]
    assert not train_config(build_parser().parse_args(args)).hip_ops
    assert train_config(build_parser().parse_args(args + ["--hip-ops"])).hip_ops
    with pytest.raises(ValueError, match="hip_ops"):
        train_extractor(TrainConfig(model="tiny", steps=1, n_examples=2, hip_ops=True), device="cpu")
    with pytest.raises(ValueError, match="hip_ops"):
        train_extractor(TrainConfig(model="tiny", steps=1, n_examples=2, hip_ops=True, fused=False), device="cuda")
