"""Inputs and tolerances of the state-space operator tests (shared by the CPU and the GPU files).

Tolerances, relative in the 2-norm over a tensor, from the arithmetic alone:
  * an output stored in bf16 is off by at most half a step, finfo.eps / 2 = 2^-8 of each value.  Computed operands of bf16
    products keep 2^-17 of their size; a sum whose terms cancel to 1/32 of their size makes that 2^-12, and a chain of four
    such products 2^-10: 2^-8 + 2^-10.
  * fp32 outputs: each of about 250 roundings on the way (64 tokens, 128 states, the joins) is off by 2^-25 in the mean and
    they are independent, so 16 * 2^-25 of the terms' size; cancellation to 1/32 makes that 2^-16 = 1.6e-5; 2e-5."""
import torch

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
TOL = {torch.bfloat16: 2.0 ** -8 + 2.0 ** -10, torch.float32: 2e-5}


def close(name, got, want):
    assert got.shape == want.shape, (name, got.shape, want.shape)
    got, tol = got.detach().double().cpu(), TOL[got.dtype]
    want = want.detach().double()
    assert torch.isfinite(got).all(), name
    err, size = float((got - want).norm()), float(want.norm())
    assert err <= tol * size + 1e-30, (name, err / max(size, 1e-300), tol)


def randn(g, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype)


def scan_inputs(seed, dtype, B, T, H, P, G, N, *, state=False, slices=True):
    """CPU tensors; x, Bm, Cm slices of one wider tensor and z, dt of another, as the layer has them."""
    g = torch.Generator().manual_seed(seed)
    lead = (B,) if T is None else (B, T)
    inner = randn(g, *lead, H * P + 2 * G * N, dtype=dtype)
    outer = randn(g, *lead, H * P + H, dtype=dtype)
    s = dict(x=inner[..., :H * P].unflatten(-1, (H, P)), Bm=inner[..., H * P:H * P + G * N].unflatten(-1, (G, N)),
             Cm=inner[..., H * P + G * N:].unflatten(-1, (G, N)), z=outer[..., :H * P].unflatten(-1, (H, P)), dt=outer[..., H * P:],
             A=-torch.exp(torch.rand(H, generator=g) * 2.8), D=randn(g, H, shift=1.0, scale=0.2),
             dt_bias=randn(g, H, shift=-3.0), state=randn(g, B, H, P, N) if state else None)
    if not slices:
        s = {k: v if v is None else v.contiguous() for k, v in s.items()}
    return s


def to(s, dev):
    """The same strides on the device: slices of one tensor stay slices of one tensor's copy."""
    out = {}
    for k, v in s.items():
        if v is None or not torch.is_tensor(v):
            out[k] = v
            continue
        base = torch.empty(v.untyped_storage().nbytes() // v.element_size(), dtype=v.dtype).set_(v.untyped_storage()).to(dev)
        out[k] = base.as_strided(v.shape, v.stride(), v.storage_offset())
    return out


def leaves64(s):
    return {k: v.detach().double().requires_grad_() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in s.items()}
