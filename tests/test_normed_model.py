"""GCN_FC(norm="layer"), the AdamW choices and 8-bit evaluation: construction and refusals on the CPU."""
import pytest
import torch


def test_default_model_is_unchanged():
    from lpgnn import GCN_FC

    torch.manual_seed(0)
    a = GCN_FC(8, 8, hids=32, depth=4)
    torch.manual_seed(0)
    b = GCN_FC(8, 8, hids=32, depth=4, norm="layer")
    assert not any(k.startswith("norms") for k in a.state_dict())
    for k, v in a.state_dict().items():
        assert torch.equal(v, b.state_dict()[k])  # the norms draw no random numbers
    extra = set(b.state_dict()) - set(a.state_dict())
    assert extra == {f"norms.{i}.{s}.{p}" for i in range(3) for s in ("left", "right") for p in ("weight", "bias")}


def test_arch_string_and_refusals():
    from lpgnn import GCN_FC, build_model

    m = build_model("GCN_FC(8,8,hids=16,depth=3,norm='layer')")
    assert len(m.norms) == 2 and m.norms[0]["left"].dim == 16
    assert build_model("GCN_FC(8,8,hids=16,depth=3,norm=None)").norms is None
    with pytest.raises(ValueError, match="norm"):
        GCN_FC(8, 8, norm="batch")


def test_make_optimizer_choices():
    from lpgnn import GCN_FC, optim
    from lpgnn.train import make_optimizer

    m = GCN_FC(8, 8, hids=16)
    o, s = make_optimizer(m, "adamw", 1e-3, 8, max_grad_norm=2.0)
    assert isinstance(o, optim.AdamW) and o.state_bits == 32 and o.max_grad_norm == 2.0
    assert o.param_groups[0]["weight_decay"] == 1e-2 and s.step_size == 2
    assert make_optimizer(m, "adamw8")[0].state_bits == 8
    assert type(make_optimizer(m, "adam")[0]) is torch.optim.Adam
    assert type(make_optimizer(m, "sgd")[0]) is torch.optim.SGD
    with pytest.raises(ValueError, match="max_grad_norm"):
        make_optimizer(m, "adam", max_grad_norm=1.0)


def test_cli_flags():
    from lpgnn import run

    a = run.parse_args(["train", "--opt", "adamw8", "--max_grad_norm", "0.5", "--int8", "1"])
    assert a.opt == "adamw8" and a.max_grad_norm == 0.5 and a.int8 == 1
    b = run.parse_args([])
    assert b.max_grad_norm == 0 and b.int8 == 0


@pytest.mark.parametrize("name", ["lin_rel.weight", "lin_rel.bias", "lin_root.weight"])
def test_int8_layer_refuses_weights_that_want_a_gradient(name):
    """Also where its inputs want none (the layers before it frozen): the weights would silently get no gradient."""
    from lpgnn.arch import GraphConvTwoDirection
    from lpgnn.conv import two_direction_i8

    layer = GraphConvTwoDirection(4, 4, 4)
    for side in ("left2right", "right2left"):
        layer.requires_grad_(False)
        layer.get_parameter(f"{side}.{name}").requires_grad_(True)
        codes = [(None, None, None, [], d) for d in (layer.left2right, layer.right2left)]
        with pytest.raises(RuntimeError, match="no gradient"):
            two_direction_i8(torch.ones(2, 4), torch.ones(3, 4), None, codes, True)


@pytest.mark.parametrize("depth", [0, 1, 2, 5])
def test_a_norm_behind_every_layer(depth):
    """conv1 is there whatever the depth (arch.py:170-174), and so is its norm."""
    from lpgnn import GCN_FC

    m = GCN_FC(8, 8, hids=16, depth=depth, norm="layer")
    assert len(m.norms) == 1 + len(m.layers) == max(depth - 1, 1)
