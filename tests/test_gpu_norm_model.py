"""GPU: GraphSAGE with norm="layer", residual and input_dropout: the operators run together as a model's layers, against
the same model in float64 on the CPU (masks from the host mirror of the kernels' hash), in training steps, captured
steps, evaluation and checkpoints."""
import pytest
import torch
import torch.nn.functional as F

from graphsage_amd import GraphSAGE, SkipGramLoss, StructuralEncoder, TrainStep, create_model, rng
from graphsage_amd.encoder import model_from_checkpoint
from graphsage_amd.graphsage import INPUT_SLOT, mix_seed
from oracle import sage_oracle as O

pytestmark = pytest.mark.gpu


def _plain(model, x, ei, base, step, training):
    """The model in float64 -> (embeddings, for each hidden layer the smallest |pre-activation|, the largest and `amp` in
    front of it, amp behind the last).  amp: how much larger the norms have made an error so far, 2 A / sigma a layer (A the
    row's largest |z|), multiplied up."""
    amp, margins = 1.0, []

    def drop(t, p, slot):
        if not training or p == 0.0:
            return t
        keep = torch.from_numpy(rng.dropout_keep_mask(mix_seed(base, step, slot), t.size(0), t.size(1), p)).bool()
        return torch.where(keep, t / (1.0 - p), torch.zeros((), dtype=t.dtype))
    h = drop(x, model.input_dropout, INPUT_SLOT)
    for i, conv in enumerate(model.convs[:-1]):
        pre = conv(h, ei)
        margins.append((float(pre.detach().abs().min()), float(pre.detach().abs().max()), amp))
        z = drop(F.relu(pre), model.dropout_rate, i)
        if model.residual and i > 0:
            z = h + z
        mean = z.mean(1, keepdim=True)
        rstd = 1.0 / ((z - mean).square().mean(1, keepdim=True) + 1e-5).sqrt()
        amp *= float((2.0 * z.abs().max(1, keepdim=True).values * rstd).detach().max())
        h = (z - mean) * rstd * model.norms[i].weight + model.norms[i].bias
    h = model.convs[-1](h, ei)
    return (F.normalize(h, p=2, dim=1) if model.normalize_output else h), margins, amp


class _Ref(torch.nn.Module):
    def __init__(self, m):
        super().__init__()
        self.convs = torch.nn.ModuleList([O.OracleSAGEConv(c.in_channels, c.out_channels) for c in m.convs])
        self.norms = torch.nn.ModuleList([torch.nn.LayerNorm(m.hidden_channels) for _ in m.convs[:-1]])
        self.load_state_dict(m.state_dict())
        self.double()
        self.residual, self.dropout_rate, self.input_dropout = m.residual, m.dropout_rate, m.input_dropout
        self.normalize_output = m.normalize_output


def _case(cfg, training, n=24, edges=90):
    """The first seed at which no pre-activation lies within the error bound of ReLU's kink (float64, on the CPU)."""
    for seed in range(200):
        torch.manual_seed(seed)
        m = GraphSAGE(**cfg)
        with torch.no_grad():
            for norm in m.norms:
                norm.weight.normal_(1.0, 0.1)
                norm.bias.normal_(0.0, 0.1)
        m.train(training)
        ref = _Ref(m)
        x, ei = torch.randn(n, cfg["in_channels"]), torch.randint(0, n, (2, edges))
        emb, margins, amp = _plain(ref, x.double(), ei, 11, seed, training)
        if all(lo > 1e-5 * before * hi for lo, hi, before in margins):
            return m, ref, x, ei, seed, emb, amp
    raise AssertionError("no seed keeps clear of the kinks")


CFGS = [dict(in_channels=7, hidden_channels=64, out_channels=64, num_layers=2, dropout=0.3, norm="layer"),
        dict(in_channels=7, hidden_channels=64, out_channels=64, num_layers=3, dropout=0.3, norm="layer", residual=True,
             input_dropout=0.2),
        dict(in_channels=5, hidden_channels=48, out_channels=20, num_layers=3, dropout=0.0, norm="layer", residual=True,
             normalize_output=False),
        dict(in_channels=7, hidden_channels=32, out_channels=32, num_layers=3, dropout=0.5, norm="layer")]


@pytest.mark.parametrize("training", [True, False])
@pytest.mark.parametrize("cfg", CFGS)
def test_forward_and_gradients_against_float64(cfg, training):
    """The bar of the plain model, 1e-5 of the largest value, times what the norms make of an error (forward once,
    backward once more)."""
    m, ref, x, ei, seed, want, amp = _case(cfg, training)
    m = m.cuda()
    m.set_dropout_stream(11, seed)
    emb = m(x.cuda(), ei.cuda())
    assert float((emb.detach().cpu().double() - want.detach()).abs().max()) <= 1e-5 * amp * float(want.detach().abs().max())
    gen = torch.Generator().manual_seed(1)
    g = torch.randn(want.shape, generator=gen)
    emb.backward(g.cuda())
    want.backward(g.double())
    for (name, p), (_, q) in zip(m.named_parameters(), ref.named_parameters()):
        err = float((p.grad.cpu().double() - q.grad).abs().max())
        assert err <= 1e-5 * amp * amp * float(q.grad.abs().max()), f"{name}: {err:.3e} of {float(q.grad.abs().max()):.3e}"


def test_large_graph_takes_the_same_layers():
    """200 k nodes: past the sizes where the plain model switches kernels; evaluation under no_grad equals the same
    forward with autograd, a training step's gradients are finite and repeat bit for bit."""
    from graphsage_amd.synth import memory_features, powerlaw_graph
    n = 200_000
    ei, x = powerlaw_graph(n, 8, seed=3).cuda(), memory_features(n, seed=3).cuda()
    torch.manual_seed(0)
    m = GraphSAGE(7, 128, 128, 3, 0.3, norm="layer", residual=True, input_dropout=0.1).cuda()
    m.eval()
    with torch.no_grad():
        a = m(x, ei)
    assert torch.equal(a, m(x, ei).detach())
    grads = []
    for _ in range(2):
        m.train()
        m.zero_grad()
        m.set_dropout_stream(5, 9)
        emb = m(x, ei)
        emb.backward(torch.linspace(-1, 1, emb.numel(), device="cuda").view_as(emb))
        grads.append([p.grad.clone() for p in m.parameters()])
    for a, b in zip(*grads):
        assert bool(torch.isfinite(a).all()) and float(a.abs().max()) > 0 and torch.equal(a, b)


def _stepper(dropout, seed=3, lr=1e-3, **kw):
    from graphsage_amd.synth import cooccurrence_batch, memory_features, powerlaw_graph
    n, b, k = 400, 256, 5
    ei, x = powerlaw_graph(n, 8, seed=1), memory_features(n, seed=1)
    t, c, neg = cooccurrence_batch(ei, n, b, k, seed=2)
    torch.manual_seed(0)
    m = GraphSAGE(7, 64, 64, 3, dropout, norm="layer", residual=True, **kw).cuda()
    # (the loss backward's default on so small a table sums by float atomics: its order, and the last bits, vary)
    st = TrainStep(m, x.cuda(), ei.cuda(), learning_rate=lr, seed=seed, loss_fn=SkipGramLoss(deterministic=True))
    return st, t.cuda(), c.cuda(), neg.cuda()


def test_training_steps_move_the_norms_and_repeat():
    runs = []
    for _ in range(2):
        st, t, c, neg = _stepper(0.3, input_dropout=0.1)
        before = st.model.norms[0].weight.detach().clone()
        losses = [float(st.step(t, c, neg)[0]) for _ in range(4)]
        assert all(l == l and abs(l) < 100 for l in losses)
        assert not torch.equal(before, st.model.norms[0].weight.detach())
        runs.append((losses, st.flat.flat.clone()))
    assert runs[0][0] == runs[1][0] and torch.equal(runs[0][1], runs[1][1])


def test_captured_step_without_dropout_equals_the_eager_step():
    eager, t, c, neg = _stepper(0.0)
    captured, _, _, _ = _stepper(0.0)
    captured.capture_step(t.numel(), neg.size(1), preserve_state=True)
    for _ in range(4):
        a = eager.step(t, c, neg).clone()
        b = captured.step_captured(t, c, neg).clone()
        torch.cuda.synchronize()
        assert torch.equal(a, b) and torch.equal(eager.flat.flat, captured.flat.flat)


def test_captured_step_draws_new_masks():
    """Learning rate 0: the parameters stay, so the losses of two replays of one batch differ by the masks alone."""
    st, t, c, neg = _stepper(0.3, lr=0.0, input_dropout=0.2)
    st.capture_step(t.numel(), neg.size(1), preserve_state=True)
    start = st.flat.flat.clone()
    losses = []
    for _ in range(4):
        losses.append(float(st.step_captured(t, c, neg)[0]))
        torch.cuda.synchronize()
    assert torch.equal(start, st.flat.flat)
    assert len(set(losses)) == 4 and all(l == l for l in losses)


def test_checkpoint_encoder_and_config(tmp_path):
    cfg = {"features": {"dimensions": 7}, "model": {"hidden_dim": 64, "output_dim": 64, "num_layers": 3, "dropout": 0.3,
                                                    "norm": "layer", "residual": True, "input_dropout": 0.1}}
    torch.manual_seed(1)
    m = create_model(cfg, torch.device("cuda"))
    assert m.norm == "layer" and m.residual and m.input_dropout == 0.1
    x, ei = torch.randn(50, 7).cuda(), torch.randint(0, 50, (2, 200)).cuda()
    m.eval()
    with torch.no_grad():
        want = m(x, ei)
    path = tmp_path / "m.pt"
    torch.save({"config": cfg, "model_state_dict": m.state_dict()}, path)
    enc = StructuralEncoder(str(path))
    assert enc.model.norm == "layer" and torch.equal(enc.encode_tensors(x, ei), want)
    again = model_from_checkpoint({"config": cfg, "model_state_dict": m.state_dict()})
    assert list(again.state_dict()) == list(m.state_dict())
    m.train()
    with pytest.raises(ValueError, match="keep_masks"):
        m(x, ei, keep_masks=[torch.ones(50, 64, dtype=torch.uint8, device="cuda")] * 2)
    with pytest.raises(ValueError, match="dropout_seeds"):
        m(x, ei, dropout_seeds=torch.zeros(2, dtype=torch.int64, device="cuda"))
    st = TrainStep(GraphSAGE(7, 64, 64, 2, 0.3, norm="layer").cuda(), x, ei, receptive_field=True)
    with pytest.raises(ValueError, match="receptive-field"):
        st.step(*(torch.zeros(4, dtype=torch.int64, device="cuda"),) * 2, torch.zeros(4, 5, dtype=torch.int64, device="cuda"))


def test_input_dropout_on_the_plain_model():
    """norm=None: the features' mask alone; evaluation is untouched and the cached aggregate is not taken from it."""
    torch.manual_seed(0)
    x, ei = torch.randn(300, 7).cuda(), torch.randint(0, 300, (2, 2000)).cuda()
    m = GraphSAGE(7, 64, 64, 2, 0.0, cache_input_aggregation=True, input_dropout=0.4).cuda()
    plain = GraphSAGE(7, 64, 64, 2, 0.0).cuda()
    plain.load_state_dict(m.state_dict())
    m.eval(), plain.eval()
    want = plain(x, ei).detach()
    assert torch.equal(m(x, ei).detach(), want)
    m.train(), plain.train()
    m.set_dropout_stream(2, 3)
    mask = torch.from_numpy(rng.dropout_keep_mask(mix_seed(2, 3, INPUT_SLOT), 300, 7, 0.4)).bool().cuda()
    dropped = torch.where(mask, x * torch.full((), 1.0 / (1.0 - 0.4), device="cuda"), torch.zeros((), device="cuda"))
    assert torch.equal(m(x, ei).detach(), plain(dropped, ei).detach())
    m.eval()
    assert torch.equal(m(x, ei).detach(), want)
