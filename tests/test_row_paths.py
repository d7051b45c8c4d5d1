"""CPU: the options that bring the row operators into the framework's own paths -- their defaults leave everything as it was."""
import pytest
import torch

from tests.test_host_logic import _cfg


def test_head_norm_option():
    from simhand_amd.host import unsupervised

    torch.manual_seed(5)
    a = unsupervised.SimCLR(_cfg("18"), None, "train")
    assert isinstance(a.projection_head[1], torch.nn.BatchNorm1d) and a.act8 is False and a.encoder.engine.act8 is False
    torch.manual_seed(5)
    b = unsupervised.SimCLR(_cfg("18", projection_head_norm="batch"), None, "train")
    assert list(a.state_dict()) == list(b.state_dict()) and all(torch.equal(u, v) for u, v in zip(a.state_dict().values(), b.state_dict().values()))
    torch.manual_seed(5)
    c = unsupervised.SimCLR(_cfg("18", projection_head_norm="layer", act8=True), None, "train")
    assert isinstance(c.projection_head[1], torch.nn.LayerNorm) and c.act8 is True and c.encoder.engine.act8 is True
    assert all(torch.equal(u, v) for u, v in zip(a.encoder.parameters(), c.encoder.parameters()))
    with pytest.raises(RuntimeError):  # a batch-norm head's checkpoint does not load into a layer-norm head unnoticed
        c.load_state_dict(a.state_dict())
    with pytest.raises(ValueError):
        unsupervised.SimCLR(_cfg("18", projection_head_norm="group"), None, "train")


def test_the_option_outlives_a_new_compute_dtype():
    from simhand_amd.host import unsupervised

    m = unsupervised.SimCLR(_cfg("18", act8=True), None, "train")
    m.set_compute_dtype(torch.bfloat16)
    assert m.encoder.engine.act8 is True
    m.encoder.set_act8(False)
    assert m.encoder.engine.act8 is False


def test_command_line_flags():
    from simhand_amd.host import experiments_utils as eu

    a = eu.get_general_args(argv=[])
    assert a.projection_head_norm is None and a.act8 is False
    a = eu.get_general_args(argv=["--projection_head_norm", "layer", "--act8"])
    assert a.projection_head_norm == "layer" and a.act8 is True
    with pytest.raises(SystemExit):
        eu.get_general_args(argv=["--projection_head_norm", "group"])
    assert not hasattr(eu.get_general_args(argv=[], with_build_flags=False), "act8")
