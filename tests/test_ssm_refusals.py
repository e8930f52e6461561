"""CPU: refusals of the state-space operators that are decided on the host before any launch: derivatives they do not have,
traces, sizes, strides and pointers no kernel can take."""
import ctypes

import pytest
import torch

from tests.ssm_cases import scan_inputs


def _calls(wrap=lambda v: v, batch=2):
    """Every entry point on CPU tensors, `wrap` around its main input: without a refusal before it, each ends at "no CPU fallback"."""
    from vit_amd import ssm
    s = scan_inputs(4, torch.float32, batch, 5, 4, 8, 2, 16, state=True)
    t = {k: v[:, 0] if k in ("x", "dt", "Bm", "Cm") else v for k, v in s.items()}
    x, w, e = torch.ones(batch, 5, 8), torch.ones(8, 4), torch.ones(8)
    return {
        "causal_conv": lambda: ssm.causal_conv(wrap(x), w),
        "causal_conv_step": lambda: ssm.causal_conv_step(wrap(x[:, 0]), w, None, torch.zeros(batch, 3, 8)),
        "selective_scan": lambda: ssm.selective_scan(wrap(s["x"]), s["dt"], s["A"], s["Bm"], s["Cm"]),
        "selective_scan_step": lambda: ssm.selective_scan_step(wrap(t["x"]), t["dt"], t["A"], t["Bm"], t["Cm"], s["state"]),
        "sandwich_norm": lambda: ssm.sandwich_norm(wrap(x), x, e, None, e, None),
    }


NAMES = ("causal_conv", "causal_conv_step", "selective_scan", "selective_scan_step", "sandwich_norm")


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(name):
    """A dual tensor does not require grad; without a refusal its tangent would be lost, which reads as zero."""
    from torch.autograd import forward_ad
    with forward_ad.dual_level(), torch.no_grad():
        with pytest.raises(RuntimeError, match="forward-mode"):
            _calls(lambda v: forward_ad.make_dual(v, torch.ones_like(v)))[name]()
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        _calls()[name]()


@pytest.mark.parametrize("name", NAMES)
def test_traces_are_refused(name):
    """torch.jit.trace records torch operations: of these calls it would keep an uninitialised result and no kernel."""
    def run(v):
        return _calls(lambda x: x * v)[name]()

    with pytest.raises(RuntimeError, match="torch.jit.trace"):
        torch.jit.trace(run, torch.ones(()))


@pytest.mark.parametrize("which", ["x", "w", "b", "state"])
def test_a_convolution_step_drops_no_gradient(which):
    """In grad mode an input that requires grad is an error, not a result without its gradient; nothing is written into a leaf."""
    from vit_amd import ssm
    t = dict(x=torch.ones(2, 8), w=torch.ones(8, 4), b=torch.ones(8), state=torch.zeros(2, 3, 8))
    t[which].requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        ssm.causal_conv_step(t["x"], t["w"], t["b"], t["state"])
    with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU fallback"):
        ssm.causal_conv_step(t["x"], t["w"], t["b"], t["state"])


@pytest.mark.parametrize("which", ["x", "dt", "A", "Bm", "Cm", "state", "D", "z", "dt_bias"])
def test_a_scan_step_drops_no_gradient(which):
    from vit_amd import ssm
    s = scan_inputs(4, torch.float32, 2, None, 4, 8, 2, 16, state=True, slices=False)
    s[which].requires_grad_()

    def call():
        return ssm.selective_scan_step(*(s[k] for k in ("x", "dt", "A", "Bm", "Cm", "state")), D=s["D"], z=s["z"], dt_bias=s["dt_bias"])

    with pytest.raises(RuntimeError, match="no gradient"):
        call()
    with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU fallback"):
        call()


SCAN = [64, 1, 1, 64, 1, 1, 64, 64, 1, 1, 64, 1, 1, None, None, 0, 0, None, None, None, 64, None, None, None]


def _scan_fwd(lib, *, args=SCAN, ws=(None, 0), dtype=1, sizes=(1, 64, 1, 64, 1, 64)):
    return lib.rvit_ssm_scan_fwd(*args, *ws, dtype, *sizes, None)


def test_no_tokens_still_need_their_decay():
    """A scan of no tokens reads A on its way to the state it returns: null is refused before a launch."""
    from vit_amd import _lib
    lib = _lib.load()
    args = list(SCAN)
    args[6] = None
    assert _scan_fwd(lib, args=args, sizes=(1, 0, 1, 64, 1, 64)) == -1 and b"null" in lib.rvit_last_error()


@pytest.mark.parametrize("at", [1, 2, 4, 5, 8, 9, 11, 12, 15, 16])
def test_negative_strides_are_refused(at):
    """The wide paths take token strides as 32-bit unsigned offsets: a negative one would read 4 GiB further on."""
    from vit_amd import _lib
    lib = _lib.load()
    args = list(SCAN)
    args[at] = -64
    assert _scan_fwd(lib, args=args) == -1 and b"stride" in lib.rvit_last_error()
    bwd = args[:19] + [64, 64, 64, 1, 1, None, 64, 64, 64, 64, 64, None, None, None, None, 64, 1 << 40]
    assert lib.rvit_ssm_scan_bwd(*bwd, 1, 1, 64, 1, 64, 1, 64, None) == -1 and b"stride" in lib.rvit_last_error()


def test_negative_strides_of_the_gradient_and_of_a_convolution():
    from vit_amd import _lib
    lib = _lib.load()
    for syb, syt in ((-1, 64), (64, -1)):
        bwd = SCAN[:19] + [64, 64, 64, syb, syt, None, 64, 64, 64, 64, 64, None, None, None, None, 64, 1 << 40]
        assert lib.rvit_ssm_scan_bwd(*bwd, 1, 1, 64, 1, 64, 1, 64, None) == -1 and b"stride" in lib.rvit_last_error()
        assert lib.rvit_ssm_conv_fwd(64, syb, syt, 64, None, None, None, 64, None, 1, 1, 8, 8, 4, 0, None) == -1 and b"stride" in lib.rvit_last_error()
        assert lib.rvit_ssm_conv_bwd(64, 64, 8, 64, None, None, None, 64, syb, syt, None, 64, 64, None, None, 64, 1 << 40, 1, 1, 8, 8, 4, 0, None) == -1
        assert b"stride" in lib.rvit_last_error()
    for i in (1, 3, 6, 8, 11):
        step = [64, 1, 64, 1, 64, 64, 1, 64, 1, None, 64, 1, None, 64, 64]
        step[i] = -1
        assert lib.rvit_ssm_scan_step(*step, 1, 1, 1, 64, 1, 64, None) == -1 and b"stride" in lib.rvit_last_error(), i
    assert lib.rvit_ssm_conv_step(64, -1, 64, None, 64, 64, 1, 1, 8, 4, 0, None) == -1 and b"stride" in lib.rvit_last_error()


def test_sizes_no_launch_can_take_are_refused():
    """A launch has fewer than 2^32 threads: what would need more is refused by size (no kernel, no launch error), for a training
    call before its forward pass."""
    from vit_amd import _lib
    lib = _lib.load()
    n = ctypes.c_int64(0)
    text = lambda: lib.rvit_last_error()  # noqa: E731
    # scan, backward: 512 threads for each (sample, chunk, group)
    assert lib.rvit_ssm_scan_plan(ctypes.byref(n), None, None, 1 << 22, 128, 1, 64, 1, 16) == 0
    assert lib.rvit_ssm_scan_plan(None, None, ctypes.byref(n), 1 << 22, 128, 1, 64, 1, 16) == -1 and b"backward" in text()
    assert lib.rvit_ssm_scan_plan(None, None, ctypes.byref(n), (1 << 22) - 1, 128, 1, 64, 1, 16) == 0
    assert lib.rvit_ssm_scan_plan(None, None, ctypes.byref(n), 1, 64, (1 << 24) - 1, 1, 1, 1) == -1
    # a sample's heads of more channels than an index over a chunk of them holds
    assert lib.rvit_ssm_scan_plan(ctypes.byref(n), None, None, 1, 64, 1, 1 << 24, 1, 16) == -1 and b"channels" in text()
    # convolution: backward 256 threads for each (sample, 8 strips, 32 accesses), its sums, forward
    assert lib.rvit_ssm_conv_bwd_workspace(ctypes.byref(n), 1 << 24, 1, 4, 4) == -1 and b"ssm_conv" in text()
    assert lib.rvit_ssm_conv_bwd_workspace(ctypes.byref(n), (1 << 24) - 1, 1, 4, 4) == 0
    assert lib.rvit_ssm_conv_bwd_workspace(ctypes.byref(n), 1, 1, 1 << 28, 4) == -1 and b"ssm_conv" in text()
    bwd = lambda B, C: lib.rvit_ssm_conv_bwd(64, C, C, 64, None, None, None, 64, C, C, None, 64, 64, None, None, 64, 1 << 50, 1, B, 1, C, 4, 0, None)  # noqa: E731
    assert bwd(1 << 24, 4) == -1 and b"ssm_conv" in text()
    assert bwd((1 << 24) - 1, 33) == -1 and b"ssm_conv" in text()       # two blocks of one-channel accesses
    assert lib.rvit_ssm_conv_fwd(64, 1, 1, 64, None, None, None, 64, None, 1, 1 << 12, (1 << 28) - 1, 17, 4, 0, None) == -1 and b"ssm_conv" in text()
    # norms: 64 threads a row, 256 where a row takes a workgroup; backward 256 a part, and a sample with its own gate is one at least
    fwd = lambda rows, E: lib.rvit_sandwich_norm_fwd(64, 1, 64, 1, None, 0, 1, 1.0, 64, None, 64, None, 1e-5, 0, 64, 64, None, rows, 1, E, None)  # noqa: E731
    assert fwd(1 << 26, 8) == -1 and b"sandwich" in text()
    assert fwd(1 << 24, 2048) == -1 and b"sandwich" in text()
    assert fwd(1 << 24, 257) == -1 and b"sandwich" in text()
    assert lib.rvit_sandwich_norm_bwd_workspace(ctypes.byref(n), 1 << 25, 2, 8, 2) == -1 and b"sandwich" in text()
    assert lib.rvit_sandwich_norm_bwd_workspace(ctypes.byref(n), (1 << 25) - 2, 2, 8, 2) == 0
    assert lib.rvit_sandwich_norm_bwd_workspace(ctypes.byref(n), 1 << 30, 2, 8, 1) == 0


@pytest.mark.parametrize("name", NAMES)
def test_an_empty_batch_is_no_error_of_shape(name):
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        _calls(batch=0)[name]()


def test_a_learned_scale_is_refused():
    """A tensor would be read as a number, its gradient lost: a learned scale belongs into the gate."""
    from vit_amd import ssm
    x, e = torch.ones(2, 8), torch.ones(8)
    for scale in (torch.ones((), requires_grad=True), torch.nn.Parameter(torch.ones(1)), torch.ones(())):
        with pytest.raises(ValueError, match="scale"):
            ssm.sandwich_norm(x, x, e, None, e, None, scale=scale)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ssm.sandwich_norm(x, x, e, None, e, None, scale=2)


def test_odd_widths_no_backward_launch_can_take_are_refused_beforehand():
    """Channels that are no multiple of four are taken one an access: their backward pass has four times the workgroups, and the
    forward pass of a training call has to know."""
    from vit_amd import _lib
    lib = _lib.load()
    n = ctypes.c_int64(0)
    assert lib.rvit_ssm_conv_bwd_workspace(ctypes.byref(n), 1 << 23, 1, 33, 4) == -1 and b"ssm_conv" in lib.rvit_last_error()
    assert lib.rvit_ssm_conv_bwd_workspace(ctypes.byref(n), (1 << 23) - 1, 1, 33, 4) == 0
    assert lib.rvit_ssm_conv_bwd_workspace(ctypes.byref(n), 1 << 23, 1, 36, 4) == 0
