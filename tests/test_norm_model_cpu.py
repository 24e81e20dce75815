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
