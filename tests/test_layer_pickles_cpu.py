"""CPU: layers pickled whole by earlier versions, and subclasses with a `norm` of their own, run as they did."""

import copy
import pickle

import pytest
import torch

from flashfusedmoe_b200 import MoELayer, nn


class OwnNorm(MoELayer):
    """Normalises behind the layer, under the name that pre_norm uses."""

    def __init__(self, *args, **options):
        super().__init__(*args, **options)
        self.norm = torch.nn.LayerNorm(32)
        self.pre_norm = torch.nn.Identity()

    def forward(self, x):
        y, losses = super().forward(x)
        return self.norm(y), losses


class NormMethod(MoELayer):
    def norm(self, x):
        return x * 2.0

    def forward(self, x):
        y, losses = super().forward(x)
        return self.norm(y), losses


@pytest.fixture
def seen(monkeypatch):
    """What the layer hands to fused_moe(), and hands back."""
    rows = []
    monkeypatch.setattr(nn, "fused_moe", lambda x, *a, **o: (rows.append(x), (x + 1.0, {}))[1])
    monkeypatch.setattr(nn.LayerNorm, "forward", lambda self, x: x * 10.0)
    return rows


def test_layers_pickled_by_earlier_versions(seen):
    x = torch.randn(5, 32)
    # of a version without the option, of one that had None in its place, and of that one with a norm
    for pre_norm, attributes in ((False, {}), (False, {"norm": None}), (True, {})):
        old = MoELayer(32, 64, 4, pre_norm=pre_norm)
        for name in ("_pre_norm", "norm"):
            old.__dict__.pop(name, None)
        old.__dict__.update(attributes)
        out, _ = pickle.loads(pickle.dumps(old))(x)
        assert torch.equal(seen.pop(), x * 10.0 if pre_norm else x) and torch.equal(out, x * (10.0 if pre_norm else 1.0) + 1.0)
    for pre_norm in (False, True):
        layer = copy.deepcopy(MoELayer(32, 64, 4, pre_norm=pre_norm))
        layer(x)
        assert torch.equal(seen.pop(), x * 10.0 if pre_norm else x)


def test_a_norm_of_a_subclass_is_its_own(seen):
    x = torch.randn(5, 32)
    layer = OwnNorm(32, 64, 4)
    out, _ = layer(x)
    assert torch.equal(seen.pop(), x) and torch.equal(out, layer.norm(x + 1.0))
    assert any(name == "norm.weight" for name, _ in layer.named_parameters())
    out, _ = NormMethod(32, 64, 4)(x)
    assert torch.equal(seen.pop(), x) and torch.equal(out, 2.0 * (x + 1.0))
    out, _ = pickle.loads(pickle.dumps(layer))(x)
    assert torch.equal(seen.pop(), x) and torch.equal(out, layer.norm(x + 1.0))
