"""CPU: the depth options of GraphSAGE (norm, residual, input_dropout) where no kernel runs: checkpoints, configs, models of
other classes."""
import pytest
import torch

from graphsage_amd import GraphSAGE, create_model
from graphsage_amd.encoder import model_from_checkpoint


def test_a_model_from_a_checkpoint_drops_nothing_in_any_mode():
    cfg = {"model": {"hidden_dim": 16, "output_dim": 8, "num_layers": 3, "dropout": 0.5, "norm": "layer", "residual": True,
                     "input_dropout": 0.25}}
    saved = {"config": cfg, "model_state_dict": create_model(cfg).state_dict()}
    m = model_from_checkpoint(saved)
    assert (m.norm, m.residual) == ("layer", True)
    assert m.dropout_rate == 0.0 and m.input_dropout == 0.0


class _WithItsOwn(GraphSAGE):
    """What a class made from GraphSAGE could hold before the options existed."""

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        self.norm = torch.nn.LayerNorm(self.out_channels)
        self.input_dropout = torch.nn.Dropout(0.5)
        self.residual = torch.nn.Linear(self.in_channels, self.out_channels)


def test_names_of_the_options_in_classes_made_from_the_model():
    from graphsage_amd.graphsage import feature_dropout, layer_normed
    m = _WithItsOwn(7, 16, 16, 2)
    m.reset_parameters()
    assert not layer_normed(m) and feature_dropout(m) == 0.0
    assert layer_normed(GraphSAGE(norm="layer")) and feature_dropout(GraphSAGE(input_dropout=0.25)) == 0.25
    other = torch.nn.Module()                   # a model that is no GraphSAGE
    other.norm, other.input_dropout = "layer", 0.5
    assert not layer_normed(other) and feature_dropout(other) == 0.0 and not layer_normed(torch.nn.Module())


def test_options_that_a_config_leaves_empty_are_the_defaults():
    m = create_model({"model": {"norm": None, "residual": None, "input_dropout": None}})
    assert (m.norm, m.residual, m.input_dropout) == (None, False, 0.0)
