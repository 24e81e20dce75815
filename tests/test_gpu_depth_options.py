"""GPU: GraphSAGE's depth options beside models that do not have them: classes made from it that keep modules of their own
under the options' names run as they did before the options existed."""
import pytest
import torch
import torch.nn.functional as F

from graphsage_amd import GraphSAGE, SkipGramLoss, TrainStep
from graphsage_amd.synth import cooccurrence_batch, memory_features, powerlaw_graph

pytestmark = pytest.mark.gpu


class _Own(GraphSAGE):
    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        self.norm = torch.nn.LayerNorm(self.out_channels)
        self.input_dropout = torch.nn.Dropout(0.5)

    def forward(self, x, edge_index, keep_masks=None):
        return self.norm(super().forward(x, edge_index, keep_masks))


def _pair(dropout):
    torch.manual_seed(3)
    own, plain = _Own(7, 64, 64, 2, dropout).cuda(), GraphSAGE(7, 64, 64, 2, dropout).cuda()
    plain.load_state_dict({k: v for k, v in own.state_dict().items() if not k.startswith("norm.")})
    ei, x = powerlaw_graph(300, 8, seed=1), memory_features(300, seed=1)
    return own, plain, x.cuda(), ei.cuda(), [t.cuda() for t in cooccurrence_batch(ei, 300, 128, 5, seed=2)]


@pytest.mark.parametrize("training", [True, False])
def test_a_class_with_modules_under_the_options_names(training):
    own, plain, x, ei, _ = _pair(0.3)
    own.train(training), plain.train(training)
    own.set_dropout_stream(5, 6), plain.set_dropout_stream(5, 6)
    assert torch.equal(own(x, ei), F.layer_norm(plain(x, ei), (64,), own.norm.weight, own.norm.bias))


def test_its_steps_eager_captured_and_receptive():
    own, _, x, ei, (t, c, neg) = _pair(0.3)
    st = TrainStep(own, x, ei, loss_fn=SkipGramLoss(deterministic=True))
    assert bool(torch.isfinite(st.step(t, c, neg)).all())
    st.capture_step(t.numel(), neg.size(1), preserve_state=True)
    losses = [float(st.step_captured(t, c, neg)[0]) for _ in range(3)]
    assert all(l == l for l in losses)
    own, plain, x, ei, (t, c, neg) = _pair(0.0)
    a = TrainStep(own, x, ei, receptive_field=True, seed=1).step(t, c, neg)      # (its convolutions alone: no norm of the class)
    b = TrainStep(plain, x, ei, receptive_field=True, seed=1).step(t, c, neg)
    assert abs(float(a[0]) - float(b[0])) <= 1e-6 * abs(float(b[0]))
