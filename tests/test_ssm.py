"""CPU: the state-space operators' oracle against differences and against torch's own convolution, and every refusal of
vit_amd.ssm / vit_amd.ops / the C entry points that is decided on the host."""
import ctypes

import pytest
import torch

from oracle import ref_ssm as ref
from tests.ssm_cases import scan_inputs


def test_conv_oracle_is_torchs_convolution():
    g = torch.Generator().manual_seed(0)
    x, w, b = torch.randn(2, 9, 5, generator=g).double(), torch.randn(5, 4, generator=g).double(), torch.randn(5, generator=g).double()
    y, after = ref.causal_conv(x, w, b)
    want = torch.nn.functional.conv1d(torch.nn.functional.pad(x.transpose(1, 2), (3, 0)), w[:, None], b, groups=5).transpose(1, 2)
    assert torch.allclose(y, want, atol=1e-12) and torch.equal(after, x[:, -3:])
    lens = torch.tensor([2, 9], dtype=torch.int32)
    y, after = ref.causal_conv(x, w, b, lengths=lens)
    assert torch.equal(y[0, 2:], torch.zeros(7, 5).double()) and torch.equal(after[0], torch.cat([torch.zeros(1, 5).double(), x[0, :2]]))


def test_oracle_gradients_against_differences():
    s = scan_inputs(1, torch.float32, 2, 5, 4, 3, 2, 3, state=True)
    s = {k: v.double().requires_grad_() for k, v in s.items()}
    lens = torch.tensor([5, 3], dtype=torch.int32)

    def f(x, dt, A, Bm, Cm, D, z, dt_bias, state):
        return ref.selective_scan(x, dt, A, Bm, Cm, D=D, z=z, dt_bias=dt_bias, state=state, lengths=lens)

    torch.autograd.gradcheck(f, [s[k] for k in ("x", "dt", "A", "Bm", "Cm", "D", "z", "dt_bias", "state")])
    g = torch.Generator().manual_seed(2)
    r = lambda *sh: torch.randn(*sh, generator=g).double().requires_grad_()  # noqa: E731
    torch.autograd.gradcheck(lambda *a: ref.sandwich_norm(*a[:6], gate=a[6], scale=0.5, kind="layer"), [r(2, 3, 6), r(2, 3, 6), r(6), r(6), r(6), r(6), r(2, 6)])
    torch.autograd.gradcheck(lambda x, w, b, st: ref.causal_conv(x, w, b, silu=True, state=st, lengths=lens), [r(2, 5, 3), r(3, 4), r(3), r(2, 3, 3)])


def test_oracle_split_sequence_is_the_whole():
    s = scan_inputs(3, torch.float32, 2, 7, 2, 3, 1, 4)
    s = {k: v if v is None else v.double() for k, v in s.items()}
    cut = lambda a, b: dict(s, **{k: s[k][:, a:b] for k in ("x", "dt", "Bm", "Cm", "z")})  # noqa: E731
    y, end = ref.selective_scan(**s)
    y0, mid = ref.selective_scan(**cut(0, 4))
    y1, end1 = ref.selective_scan(**dict(cut(4, 7), state=mid))
    assert torch.allclose(torch.cat([y0, y1], 1), y, atol=1e-12) and torch.allclose(end, end1, atol=1e-12)


def _scan(**kw):
    s = scan_inputs(4, torch.float32, 2, 5, 4, 8, 2, 16)
    s.update(kw)
    from vit_amd import ssm
    x, dt, A, Bm, Cm = (s.pop(k) for k in ("x", "dt", "A", "Bm", "Cm"))
    return ssm.selective_scan(x, dt, A, Bm, Cm, **s)


@pytest.mark.parametrize("bad", [
    dict(x=torch.zeros(2, 5, 32)), dict(x=torch.zeros(2, 5, 4, 8, dtype=torch.float16)), dict(x=torch.zeros(2, 5, 3, 8)),
    dict(dt=torch.zeros(2, 5, 3)), dict(dt=torch.zeros(2, 5, 4, dtype=torch.bfloat16)), dict(z=torch.zeros(2, 5, 4, 4)),
    dict(Bm=torch.zeros(2, 5, 3, 16), Cm=torch.zeros(2, 5, 3, 16)), dict(Cm=torch.zeros(2, 5, 2, 8)), dict(Bm=torch.zeros(2, 4, 2, 16)),
    dict(Bm=torch.zeros(2, 5, 2, 129), Cm=torch.zeros(2, 5, 2, 129)), dict(A=torch.zeros(3)), dict(A=torch.zeros(4, dtype=torch.bfloat16)),
    dict(D=torch.zeros(4, 8)), dict(dt_bias=torch.zeros(4).double()), dict(state=torch.zeros(2, 4, 8, 15)),
    dict(state=torch.zeros(2, 4, 8, 16, dtype=torch.bfloat16)), dict(lengths=torch.tensor([1, 2])), dict(lengths=torch.tensor([1], dtype=torch.int32)),
])
def test_scan_refuses(bad):
    with pytest.raises(ValueError):
        _scan(**bad)


def test_scan_has_no_cpu_path():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        _scan()
    from vit_amd import ssm
    s = scan_inputs(4, torch.float32, 2, None, 4, 8, 2, 16, state=True)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ssm.selective_scan_step(*(s[k] for k in ("x", "dt", "A", "Bm", "Cm", "state")))
    with pytest.raises(ValueError):      # the state of another batch
        ssm.selective_scan_step(*(s[k] for k in ("x", "dt", "A", "Bm", "Cm")), torch.zeros(1, 4, 8, 16))


@pytest.mark.parametrize("x,w,kw", [
    (torch.zeros(2, 5), torch.zeros(5, 4), {}), (torch.zeros(2, 3, 5), torch.zeros(4, 4), {}), (torch.zeros(2, 3, 5), torch.zeros(5, 1), {}),
    (torch.zeros(2, 3, 5), torch.zeros(5, 7), {}), (torch.zeros(2, 3, 5).half(), torch.zeros(5, 4), {}), (torch.zeros(2, 3, 5), torch.zeros(5, 4).bfloat16(), {}),
    (torch.zeros(2, 3, 5), torch.zeros(5, 4), dict(bias=torch.zeros(4))), (torch.zeros(2, 3, 5), torch.zeros(5, 4), dict(state=torch.zeros(2, 4, 5))),
    (torch.zeros(2, 3, 5), torch.zeros(5, 4), dict(lengths=torch.zeros(3, dtype=torch.int32))), (torch.zeros(2, 3, 5), torch.zeros(5, 4), dict(activation="relu")),
    (torch.zeros(2, 3, 5).bfloat16(), torch.zeros(5, 4), dict(state=torch.zeros(2, 3, 5))),
])
def test_conv_refuses(x, w, kw):
    from vit_amd import ssm
    with pytest.raises(ValueError):
        ssm.causal_conv(x, w, **kw)


def test_conv_has_no_cpu_path():
    from vit_amd import ssm
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ssm.causal_conv(torch.zeros(2, 3, 5), torch.zeros(5, 4))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ssm.causal_conv_step(torch.zeros(2, 5), torch.zeros(5, 4), None, torch.zeros(2, 3, 5))


@pytest.mark.parametrize("kw", [
    dict(residual=torch.zeros(2, 3, 7)), dict(y=torch.zeros(2, 3, 8).half()), dict(post_weight=torch.zeros(7)), dict(pre_weight=torch.zeros(8).double()),
    dict(gate=torch.zeros(3, 8)), dict(gate=torch.zeros(2, 3)), dict(gate=torch.zeros(8, dtype=torch.bfloat16)), dict(kind="batch"),
    dict(kind="rms"), dict(residual=torch.zeros(1, 4097), y=torch.zeros(1, 4097)),
])
def test_sandwich_refuses(kw):
    from vit_amd import ssm
    a = dict(residual=torch.zeros(2, 3, 8), y=torch.zeros(2, 3, 8), post_weight=torch.ones(8), post_bias=torch.zeros(8), pre_weight=torch.ones(8),
             pre_bias=torch.zeros(8))
    a.update(kw)
    with pytest.raises(ValueError):
        ssm.sandwich_norm(**a)


def test_sandwich_has_no_cpu_path():
    from vit_amd import ssm
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ssm.sandwich_norm(torch.zeros(3, 8), torch.zeros(3, 8), torch.ones(8), None, torch.ones(8), None)


def test_c_entries_refuse_without_a_launch():
    """Sizes, null pointers, small or unaligned workspaces: an error code and a text, decided before anything is enqueued."""
    from vit_amd import _lib
    lib = _lib.load()
    n = ctypes.c_int64(0)
    plan = lambda *a: lib.rvit_ssm_scan_plan(ctypes.byref(n), None, None, *a)  # noqa: E731
    assert plan(1, 64, 8, 64, 1, 64) == 0
    for bad in ((0, 64, 8, 64, 1, 64), (1, -1, 8, 64, 1, 64), (1, 64, 8, 64, 3, 64), (1, 64, 8, 64, 1, 129), (1, 64, 8, 64, 1, 0), (1 << 20, 64, 32, 64, 1, 64)):
        assert plan(*bad) == -1, bad
    assert lib.rvit_ssm_conv_bwd_workspace(ctypes.byref(n), 1, 8, 8, 7) == -1
    assert lib.rvit_sandwich_norm_bwd_workspace(ctypes.byref(n), 10, 3, 8, 2) == -1      # rows are not whole samples
    scan = [64, 1, 1, 64, 1, 1, 64, 64, 1, 1, 64, 1, 1, None, None, 0, 0, None, None, None, 64, None, None, None]
    assert lib.rvit_ssm_scan_fwd(*scan, None, 0, 1, 1, 4096, 1, 64, 1, 64, None) == -1   # cut into segments: needs a workspace
    assert b"workspace" in lib.rvit_last_error()
    assert lib.rvit_ssm_scan_fwd(*scan, 8, 1 << 40, 1, 1, 4096, 1, 64, 1, 64, None) == -1
    assert lib.rvit_ssm_scan_fwd(None, *scan[1:], None, 0, 1, 1, 64, 1, 64, 1, 64, None) == -1
    assert lib.rvit_ssm_scan_fwd(*scan, None, 0, 2, 1, 64, 1, 64, 1, 64, None) == -1     # dtype
    assert lib.rvit_ssm_conv_fwd(64, 1, 1, 64, None, 128, None, 64, 128, 1, 1, 8, 8, 4, 0, None) == -1   # the kept inputs in place
    assert lib.rvit_sandwich_norm_fwd(64, 1, 64, 1, 64, 4, 1, 1.0, 64, None, 64, None, 1e-5, 0, 64, 64, None, 4, 2, 8, None) == -1


def test_temporal_encoder_refusals():
    from vit_amd.sequence import CNNViTSequence, TemporalEncoder
    with pytest.raises(ValueError, match="causal"):
        TemporalEncoder(128, 64, model_type="ssm")                                     # bidirectional by default
    with pytest.raises(NotImplementedError):
        TemporalEncoder(128, 40, bidirectional=False, model_type="ssm")
    with pytest.raises(NotImplementedError):
        TemporalEncoder(130, 64, bidirectional=False, model_type="ssm")
    enc = TemporalEncoder(128, 64, 2, bidirectional=False, model_type="ssm")
    assert enc.output_dim == 64
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        enc(torch.zeros(1, 4, 128))
    cfg = dict(backbone="patch16", embed_dim=128, num_heads=2, num_layers=1, dropout=0.0, temporal_hidden=64, temporal_layers=1)
    with pytest.raises(ValueError, match="keeps no state"):
        CNNViTSequence(11, cfg).forward_temporal_step(torch.zeros(1, 128))
    m = CNNViTSequence(11, dict(cfg, temporal_model="ssm"))
    assert not m.temporal_encoder.bidirectional and m.classifier["0"].weight.shape == (32, 64)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        m.forward_temporal_step(torch.zeros(1, 128))
