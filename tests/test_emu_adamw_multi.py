"""AdamW over many tensors (csrc/optim_multi.hip) on the host emulator, against the update in 64 bits, and its refusals."""
import pytest
import torch

from open_flamingo_amd.train.optim import adamw_step
from tests import vocab_reference as R
from tests.emu import harness

HYPER = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8)


def stepper(wd=0.1, max_norm=1.0, **kw):
    return lambda ps, gs, ms, vs, a, b, t: adamw_step(ps, gs, ms, vs, step=t, weight_decay=wd, max_norm=max_norm, exp_avg_scales=a, exp_avg_sq_scales=b,
                                                      ops=harness.emu_ops(), **HYPER, **kw)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("sizes,grad_dtype,max_norm,wd,offset", [
    ([1], torch.float32, 1.0, 0.1, 0),
    ([255, 256, 257, 3, 1024], torch.float32, 0.0, 0.0, 0),
    ([4097, 5], torch.bfloat16, 1.0, 0.1, 0),
    ([700, 300], torch.float32, 0.1, 0.1, 1),              # tensors that begin at odd addresses
    ([17] * 50, torch.bfloat16, 1.0, 0.0, 0),              # two launches
])
def test_against_64_bits(bits, sizes, grad_dtype, max_norm, wd, offset):
    R.adamw_check(stepper(wd, max_norm), sizes, bits, grad_dtype, max_norm=max_norm, wd=wd, steps=2 if len(sizes) > 9 else 3, offset=offset)


def fresh(sizes, bits, n_extra=0):
    ps = [torch.ones(n) for n in sizes]
    dt = torch.float32 if bits == 32 else torch.float8_e4m3fn
    ms, vs = ([torch.zeros(n).to(dt) for n in sizes] for _ in range(2))
    sc = [[torch.zeros(-(-n // 256)) for n in sizes] for _ in range(2)] if bits == 8 else (None, None)
    return ps, ms, vs, sc


@pytest.mark.parametrize("bits", [8, 32])
def test_a_norm_that_is_not_finite_leaves_everything_and_the_counter_as_it_was(bits):
    ps, ms, vs, sc = fresh([300, 5], bits)
    kw = dict(exp_avg_scales=sc[0], exp_avg_sq_scales=sc[1], ops=harness.emu_ops())
    applied = torch.zeros(1, dtype=torch.int32)
    adamw_step(ps, [torch.ones(300), torch.ones(5)], ms, vs, applied=applied, **kw)
    before = [t.clone() for ts in (ps, ms, vs) + tuple(s for s in sc if s) for t in ts]
    for bad in (float("nan"), float("inf"), 3e38):
        g = torch.ones(5)
        g[2] = bad
        adamw_step(ps, [torch.ones(300), g], ms, vs, applied=applied, **kw)
    after = [t for ts in (ps, ms, vs) + tuple(s for s in sc if s) for t in ts]
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, after)) and int(applied) == 1
    host = fresh([300, 5], bits)
    adamw_step(host[0], [torch.ones(300), torch.ones(5)], host[1], host[2], step=1, exp_avg_scales=host[3][0], exp_avg_sq_scales=host[3][1], ops=harness.emu_ops())
    assert all(torch.equal(a, b) for a, b in zip(host[0], ps))


def test_zeros_and_a_parameter_without_elements():
    ps, ms, vs, sc = fresh([300, 0], 8)
    n2 = adamw_step(ps, [torch.zeros(300), torch.zeros(0)], ms, vs, step=1, weight_decay=0.0, exp_avg_scales=sc[0], exp_avg_sq_scales=sc[1], ops=harness.emu_ops())
    assert float(n2) == 0 and (ps[0] == 1).all() and (ms[0].float() == 0).all() and (vs[0].float() == 0).all() and (sc[0][0] == 0).all()
    assert float(adamw_step(ps[1:], [torch.zeros(0)], ms[1:], vs[1:], step=1, exp_avg_scales=sc[0][1:], exp_avg_sq_scales=sc[1][1:], ops=harness.emu_ops())) == 0


def test_the_second_moment_moves_in_8_bits_on_average():
    """b2 = 0.999 moves the root of the second moment by less than half a code a step: at random in proportion it arrives all the same."""
    n = 256 * 8
    ps, ms, vs, sc = fresh([n], 8)
    kw = dict(betas=(0.9, 0.999), lr=0.0, weight_decay=0.0, exp_avg_scales=sc[0], exp_avg_sq_scales=sc[1], ops=harness.emu_ops())
    adamw_step(ps, [torch.full((n,), 1.0)], ms, vs, step=1, **kw)
    for t in range(2, 42):          # the gradient falls to a third; the largest of each block keeps its scale
        g = torch.full((n,), 1 / 3)
        g[::256] = 1.0
        adamw_step(ps, [g], ms, vs, step=t, **kw)
    v = ((R.blocks256(vs[0].float()) * sc[1][0][:, None]) ** 2)[:, 1:].mean()
    want = 0.001 * 0.999 ** 40 + (1 / 9) * (1 - 0.999 ** 40)
    # 2040 elements, each within one code (1/8) of its place: a mean within 1/8 / sqrt(2040) x 5 deviations of the root, twice that of its square,
    # and the mean of a square over the square of a mean by (1/8)^2 at most
    assert abs(float(v) / want - 1) < 2 * 5 * 0.125 / 2040 ** 0.5 + 0.125 ** 2, (float(v), want)


@pytest.mark.parametrize("change", [
    dict(step=0), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(grads=lambda g: [g[0].half(), g[1]]), dict(grads=lambda g: [g[0][:-1], g[1]]), dict(grads=lambda g: g[:1]),
    dict(params=lambda p: [p[0].bfloat16(), p[1]]), dict(params=lambda p: [torch.ones(600)[::2], p[1]]), dict(params=lambda p: []), dict(exp_avgs=lambda m: [x.float() for x in m]),
    dict(exp_avg_scales=None), dict(exp_avg_scales=lambda s: [torch.zeros(1), s[1]]), dict(lr=[1e-3]), dict(applied=torch.zeros(1)),
])
def test_refusals(change):
    ps, ms, vs, sc = fresh([300, 5], 8)
    args = dict(params=ps, grads=[torch.ones(300), torch.ones(5)], exp_avgs=ms, exp_avg_sqs=vs, step=1, exp_avg_scales=sc[0], exp_avg_sq_scales=sc[1], ops=harness.emu_ops())
    for k, v in change.items():
        args[k] = v(args[k]) if callable(v) else v
    with pytest.raises(ValueError):
        adamw_step(**args)
    assert all((p == 1).all() for p in ps)


def test_more_refusals():
    ps, ms, vs, sc = fresh([300, 300], 32)
    with pytest.raises(ValueError):          # the same parameter twice: two updates of it would race
        adamw_step([ps[0], ps[0]], [torch.ones(300)] * 2, ms, vs, step=1, ops=harness.emu_ops())
    with pytest.raises(RuntimeError):
        adamw_step(ps, [torch.ones(300)] * 2, ms, vs, step=1)
