"""AdamW over many tensors on the host emulator: gradients whose squares leave fp32's range, and the largest whose squares do not."""
import pytest
import torch

from open_flamingo_amd.train.optim import adamw_step
from tests.emu import harness


def state(bits, n=300):
    dt = torch.float32 if bits == 32 else torch.float8_e4m3fn
    sc = [[torch.zeros(-(-n // 256))] for _ in range(2)] if bits == 8 else [None, None]
    return dict(params=[torch.ones(n)], exp_avgs=[torch.zeros(n).to(dt)], exp_avg_sqs=[torch.zeros(n).to(dt)], exp_avg_scales=sc[0], exp_avg_sq_scales=sc[1],
                applied=torch.zeros(1, dtype=torch.int32))


def tensors(s):
    return [t for k in ("params", "exp_avgs", "exp_avg_sqs", "exp_avg_scales", "exp_avg_sq_scales") if s[k] for t in s[k]]


def grad(value, n=300):
    g = torch.ones(n)
    g[3] = value
    return [g]


@pytest.mark.parametrize("max_norm", [0.0, 1.0])
@pytest.mark.parametrize("bits", [8, 32])
def test_a_squared_norm_beyond_fp32_skips_the_step_and_says_so(bits, max_norm):
    s = state(bits)
    kw = dict(max_norm=max_norm, ops=harness.emu_ops())
    adamw_step(grads=grad(1.0), **s, **kw)
    before = [t.clone() for t in tensors(s)]
    n2 = adamw_step(grads=grad(1e21), **s, **kw)
    assert not torch.isfinite(n2) and int(s["applied"]) == 1
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, tensors(s)))
    adamw_step(grads=grad(1.0), **s, **kw)
    assert all(torch.isfinite(t.float()).all() for t in tensors(s)) and int(s["applied"]) == 2


@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.0, 0.0)])
@pytest.mark.parametrize("bits", [8, 32])
def test_the_largest_gradient_that_is_applied_leaves_finite_states(bits, betas):
    s = state(bits)
    n2 = adamw_step(grads=grad(1.7e19), betas=betas, **s, ops=harness.emu_ops())          # squared: 2.89e38
    assert abs(float(n2) / 2.89e38 - 1) < 1e-5
    for _ in range(3):
        adamw_step(grads=grad(1.0), betas=betas, **s, ops=harness.emu_ops())
        assert all(torch.isfinite(t.float()).all() for t in tensors(s))
    assert int(s["applied"]) == 4
