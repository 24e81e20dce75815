"""GPU: a training step's autograd graph ends with the step: nothing that it holds outlives it until the garbage collector
runs, and a step can be captured after eager ones (a graph of the same parameters still alive would end the process)."""
import gc

import pytest
import torch

from graphsage_amd import GraphSAGE, SkipGramLoss, TrainStep
from graphsage_amd.synth import cooccurrence_batch, memory_features, powerlaw_graph

pytestmark = pytest.mark.gpu

MODELS = [dict(dropout=0.0), dict(dropout=0.3), dict(dropout=0.3, norm="layer"), dict(dropout=0.3, input_dropout=0.2)]


def _stepper(kw, n, layers=2):
    ei, x = powerlaw_graph(n, 8, seed=1), memory_features(n, seed=1)
    b = [t.cuda() for t in cooccurrence_batch(ei, n, 128, 5, seed=2)]
    torch.manual_seed(0)
    return TrainStep(GraphSAGE(7, 64, 64, layers, **kw).cuda(), x.cuda(), ei.cuda(), seed=3), b


@pytest.mark.parametrize("kw", MODELS)
def test_a_step_leaves_no_memory_behind(kw):
    st, b = _stepper(kw, 20_000)
    st.step(*b)
    torch.cuda.synchronize()
    gc.collect()
    gc.disable()
    try:
        before = torch.cuda.memory_allocated()
        for _ in range(3):
            st.step(*b)
        torch.cuda.synchronize()
        # (an activation table is 5 MB)
        assert torch.cuda.memory_allocated() - before < 1 << 20
    finally:
        gc.enable()


@pytest.mark.parametrize("kw", MODELS[1:])
def test_a_step_is_captured_after_eager_ones(kw):
    st, b = _stepper(kw, 500, 3)
    gc.disable()
    try:
        for _ in range(2):
            st.step(*b)
        st.capture_step(b[0].numel(), b[2].size(1), preserve_state=True)
    finally:
        gc.enable()
    losses = []
    for _ in range(3):
        losses.append(float(st.step_captured(*b)[0]))
        st.step(*b)                              # (eager steps between the replays)
        torch.cuda.synchronize()
    assert all(l == l and 0 < l < 100 for l in losses)
