"""The operators together, as the temporal encoder runs them (temporal_model='ssm'): features, gradients of every parameter,
streaming on kept states, checkpoints, training in a window; against oracle/ref_ssm.py in 64 bits.

Tolerance: every bf16 rounding is off by at most 2^-8.  A layer rounds the norm, the projection, the convolution, the scan's
output and the block's output (5), and its five weight operands (in_proj, out_proj and what the kernels keep in fp32 do not
count twice): 7 a layer with the two weights, 3 around the stack.  Two layers forward: 17; their errors are independent, so
sqrt(17) * 2^-8 = 1.6e-2 of the features.  The backward pass rounds as often again: sqrt(34) * 2^-8 = 2.3e-2; the gates and
norms in between pass errors on at up to twice their size: 4.6e-2 for a gradient.
A head's A, D and dt_bias have ONE gradient each, a sum over samples, tokens, channels (and states) whose terms have both
signs: independent errors of 4.6e-2 of the terms make an error of 4.6e-2 * sqrt(sum of the terms' squares) of the sum, however
much of the sum itself cancels, so these are held against the root of the terms' squares (the oracle spreads them out)."""
import pytest
import torch

from oracle import ref_ssm as ref

pytestmark = pytest.mark.gpu

CFG = dict(backbone="patch16", embed_dim=128, num_heads=2, num_layers=1, dropout=0.0, temporal_hidden=64, temporal_layers=2, temporal_dropout=0.0,
           temporal_model="ssm", classifier_dropout=0.0, sequence_length=4, mode="sequence")


def _model(dev, seed=0, **kw):
    from vit_amd.sequence import CNNViTSequence
    torch.manual_seed(seed)
    m = CNNViTSequence(11, dict(CFG, **kw))
    with torch.no_grad():
        for n, p in m.named_parameters():
            if n.startswith(("temporal_encoder", "classifier")) and not n.rsplit(".", 1)[1].startswith(("A_log", "dt_bias")):
                p.add_(torch.randn_like(p) * 0.05)
    return m.to(dev)


def _ref(m):
    r = m.temporal_encoder.rnn
    return {n: p.detach().double().cpu().requires_grad_() for n, p in r.named_parameters()}, r


def _off(got, want):
    return float((got.detach().double().cpu() - want.detach()).norm() / want.detach().norm())


@pytest.mark.parametrize("B,T", [(1, 1), (3, 5), (2, 70)])
def test_features_and_gradients(dev, B, T):
    m = _model(dev).train()
    enc = m.temporal_encoder
    p, r = _ref(m)
    x = torch.randn(B, T, 128)
    x64 = x.double().requires_grad_()
    want = ref.ssm_stack(p, x64, 2, r.inner, r.states)[:, -1]
    cot = torch.randn(B, 64)
    gw = torch.autograd.grad(want, list(p.values()) + [x64], cot.double(), allow_unused=True)
    xd = x.to(dev).requires_grad_()
    got = enc(xd)
    assert got.shape == (B, 64) and _off(got, want) <= 1.6e-2
    gg = torch.autograd.grad(got, [q for _, q in r.named_parameters()] + [xd], cot.to(dev))
    spread = {}
    ref.ssm_stack({k: v.detach() for k, v in p.items()}, x.double(), 2, r.inner, r.states, spread=spread)[:, -1].backward(cot.double())
    for name, a, b in zip(list(p) + ["x"], gg, gw):
        if name in spread:
            terms = spread[name].grad
            heads = terms.shape[2]
            terms = terms.transpose(0, 2).reshape(heads, -1)
            assert torch.allclose(terms.sum(1), b, rtol=1e-9, atol=1e-12)
            assert float(((a.double().cpu() - b).abs() - 4.6e-2 * terms.norm(dim=1)).max()) <= 1e-9, (name, a, b, terms.norm(dim=1))
            continue
        if b is None or float(b.norm()) < 1e-9:     # one token: nothing passes through a decay
            assert float(a.double().norm()) <= 1e-4, name
            continue
        assert _off(a, b) <= 4.6e-2, (name, _off(a, b))


def test_lengths_pick_each_samples_last_frame(dev):
    m = _model(dev).eval()
    x = torch.randn(3, 9, 128, device=dev)
    lens = torch.tensor([9, 1, 4], dtype=torch.int32, device=dev)
    with torch.no_grad():
        got, _ = m.temporal_encoder.ssm_features(x, lens)
        for b, n in enumerate(lens.tolist()):
            want = m.temporal_encoder(x[b:b + 1, :n])
            assert _off(got[b:b + 1], want.double().cpu()) <= 1.6e-2


def test_streaming_frame_by_frame_is_the_window(dev):
    from vit_amd.sequence import StreamingClassifier
    m = _model(dev).eval()
    f = torch.randn(2, 12, 128, device=dev)
    cache = None
    with torch.no_grad():
        for t in range(12):
            logits, cache = m.forward_temporal_step(f[:, t], cache)
            want = m.forward_temporal_only(f[:, :t + 1])
            # both sides round; their errors are independent: sqrt(2) of one side's
            assert _off(logits, want.double().cpu()) <= 1.42 * 1.6e-2, t
    frames = [torch.randn(3, 224, 224) for _ in range(6)]
    sc = StreamingClassifier(model=m, classes=[str(i) for i in range(11)], config=CFG, smoothing_window=1, carry_state=True)
    first = [sc.update(x) for x in frames]
    assert [p is None for p in first] == [True] * 3 + [False] * 3
    sc.reset()
    again = [sc.update(x) for x in frames]
    assert [p.all_probs for p in again[3:]] == [p.all_probs for p in first[3:]]
    window = StreamingClassifier(model=m, classes=[str(i) for i in range(11)], config=CFG, smoothing_window=1)
    fourth = [window.update(x) for x in frames][3]          # its first window is the whole past
    assert abs(dict(fourth.all_probs)["0"] - dict(first[3].all_probs)["0"]) <= 3e-2


def test_prompt_cache_goes_on_frame_by_frame(dev):
    m = _model(dev).eval()
    f = torch.randn(2, 10, 128, device=dev)
    cache = []
    with torch.no_grad():
        m.temporal_encoder.ssm_features(f[:, :7], cache=cache)
        for t in range(7, 10):
            logits, cache = m.forward_temporal_step(f[:, t], cache)
        want = m.forward_temporal_only(f)
    assert _off(logits, want.double().cpu()) <= 1.42 * 1.6e-2


def test_training_step_runs_and_fills_every_gradient(dev):
    m = _model(dev, temporal_dropout=0.3, classifier_dropout=0.4).train()
    x = torch.randn(2, 4, 3, 224, 224, device=dev)
    loss = torch.nn.functional.cross_entropy(m(x), torch.tensor([1, 7], device=dev))
    loss.backward()
    for n, p in m.named_parameters():
        if n.startswith(("temporal_encoder", "classifier")):
            assert p.grad is not None and torch.isfinite(p.grad).all(), n
            assert float(p.grad.abs().sum()) > 0 or n.endswith("bias"), n


def test_checkpoint_round_trip(dev, tmp_path):
    from vit_amd.sequence import StreamingClassifier
    m = _model(dev).eval()
    path = str(tmp_path / "ssm.pt")
    torch.save({"model": {k: v.cpu() for k, v in m.state_dict().items()}, "classes": [str(i) for i in range(11)], "model_config": CFG}, path)
    sc = StreamingClassifier(path, carry_state=True)
    f = torch.randn(1, 128, device=dev)
    assert torch.equal(sc.model.forward_temporal_step(f)[0], m.forward_temporal_step(f)[0])


def test_a_frame_out_of_a_window_of_bf16_features(dev):
    """Features that already are bf16 come as a slice of a longer window: rows apart in memory."""
    m = _model(dev).eval()
    f = torch.randn(3, 4, 128, device=dev).bfloat16()
    with torch.no_grad():
        a, b = m.forward_temporal_step(f[:, 1])[0], m.forward_temporal_step(f[:, 1].contiguous())[0]
        assert torch.equal(a, b)
        x = torch.randn(4, 3, 128, device=dev).bfloat16().transpose(0, 1)
        assert torch.equal(m.forward_temporal_only(x), m.forward_temporal_only(x.contiguous()))
