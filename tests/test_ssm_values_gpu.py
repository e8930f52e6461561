"""State-space operators on the GPU, value by value, against oracle/ref_ssm.py and the formulas in 64 bits: results that are rounded
once, decays and gates at the ends of their range, masks, empty batches, backward passes of one chunk, row counts around the
segments."""
import pytest
import torch

from oracle import ref_ssm as ref
from tests.ssm_cases import DTYPES, close, leaves64, randn, scan_inputs, to

pytestmark = pytest.mark.gpu


def _call(ssm, s, **kw):
    return ssm.selective_scan(s["x"], s["dt"], s["A"], s["Bm"], s["Cm"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"], state=s["state"], **kw)


def _within(name, got, want, bound):
    """Every value within its own bound."""
    off = (got.detach().double().cpu() - want).abs()
    worst = float((off / bound).max())
    assert worst <= 1.0, (name, worst, int((off > bound).sum()), off.numel())


@pytest.mark.parametrize("shape", [(1, 8, 2, 64, 1, 64), (2, 64, 3, 24, 1, 16), (2, 130, 4, 64, 2, 128), (1, 600, 2, 40, 1, 33)])
def test_gate_gradient_is_rounded_once(dev, shape):
    """dz = dy v silu'(z) of bf16 calls: half a step of the value, 2^-8, and what v itself is off by.  v is held in 32 bits: its
    operands of two parts leave 2^-17 of the terms' size, and at most 192 terms a chunk are added with 2^-24 each (2^-16.4),
    so 2^-15 of the sum of the terms' sizes (|x|, |B|, |C|, |D| in the place of x, B, C, D).  silu'(z) = s + z s (1 - s): 2^-21 of
    its two parts' sizes."""
    from vit_amd import ssm
    B, T, H, P, G, N = shape
    s = scan_inputs(sum(shape), torch.bfloat16, B, T, H, P, G, N, state=T == 130)
    dy = randn(torch.Generator().manual_seed(2), B, T, H, P, dtype=torch.bfloat16)
    d = {k: v if v is None else v.double() for k, v in s.items()}
    bare = dict(d, z=None)
    v, _ = ref.selective_scan(**bare)
    size, _ = ref.selective_scan(**{k: t.abs() if t is not None and k in ("x", "Bm", "Cm", "D", "state") else t for k, t in bare.items()})
    sg = torch.sigmoid(d["z"])
    parts = sg + d["z"].abs() * sg * (1 - sg)
    want = dy.double() * v * (sg + d["z"] * sg * (1 - sg))
    bound = 2.0 ** -8 * want.abs() + (1 + 2.0 ** -8) * dy.double().abs() * parts * (2.0 ** -15 * size + 2.0 ** -21 * v.abs())
    leaf = to(s, dev)
    leaf["z"].requires_grad_()
    (dz,) = torch.autograd.grad(_call(ssm, leaf), [leaf["z"]], dy.to(dev))
    _within("dz", dz, want, bound + 1e-30)


def test_function_transforms_are_refused(dev):
    """torch.func's wrappers hold no memory a kernel could read: an error, never a result without its derivative."""
    from vit_amd import ssm
    x, w = torch.randn(2, 5, 8, device=dev), torch.randn(8, 4, device=dev)
    f = lambda v: ssm.causal_conv(v, w)  # noqa: E731
    for call in (lambda: torch.func.jvp(f, (x,), (x,)), lambda: torch.func.grad(lambda v: f(v).sum())(x), lambda: torch.func.vmap(f)(x[None])):
        with pytest.raises(RuntimeError):
            call()
    with torch.autograd.forward_ad.dual_level():       # a tangent that arrives with the gradient
        y = ssm.causal_conv(x.clone().requires_grad_(), w)
        dy = torch.autograd.forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.backward(y, dy)
