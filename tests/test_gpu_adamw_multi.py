"""AdamW over many tensors on the GPU, against the update in 64 bits (tests/vocab_reference.py)."""
import pytest
import torch

from tests import vocab_reference as R

pytestmark = pytest.mark.gpu


def stepper(wd=0.1, max_norm=1.0):
    from open_flamingo_amd.train.optim import adamw_step
    return lambda ps, gs, ms, vs, a, b, t: adamw_step(ps, gs, ms, vs, step=t, lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=wd, max_norm=max_norm,
                                                      exp_avg_scales=a, exp_avg_sq_scales=b)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("sizes,grad_dtype,max_norm,wd,offset", [
    ([1], torch.float32, 1.0, 0.1, 0),
    ([255, 256, 257, 3, 1024], torch.float32, 0.0, 0.0, 0),
    ([4097, 5, 100003], torch.bfloat16, 1.0, 0.1, 0),
    ([70001, 300], torch.float32, 0.1, 0.1, 1),
    ([1777] * 170, torch.bfloat16, 1.0, 0.0, 0),
    ([3000017, 2048, 999], torch.float32, 1.0, 0.1, 0),
])
def test_against_64_bits(bits, sizes, grad_dtype, max_norm, wd, offset):
    R.adamw_check(stepper(wd, max_norm), sizes, bits, grad_dtype, max_norm=max_norm, wd=wd, device="cuda", offset=offset)


@pytest.mark.parametrize("bits", [8, 32])
def test_a_tensor_behind_32_bits(bits):
    """More than 2^31 elements, in whole blocks before its tail: the tail gets what it gets as a tensor of its own (without the clip, which
    takes the norm of everything; the second moment's codes draw by the element's index)."""
    from open_flamingo_amd.train.optim import adamw_step
    n, tail = (1 << 31) + 4096 + 77, 4096 + 77
    f8 = torch.float8_e4m3fn
    p, g = torch.empty(n, device="cuda").fill_(0.5), torch.empty(n, dtype=torch.bfloat16, device="cuda").fill_(1e-3)
    p[-tail:], g[-tail:] = torch.randn(tail, device="cuda"), torch.randn(tail, device="cuda").to(torch.bfloat16)
    dt = f8 if bits == 8 else torch.float32

    def step(p, g):
        m, v = (torch.zeros(p.numel(), dtype=torch.float32 if bits == 32 else torch.uint8, device="cuda").view(dt) for _ in range(2))
        sc = [torch.zeros(-(-p.numel() // 256), device="cuda") for _ in range(2)] if bits == 8 else [None, None]
        adamw_step([p], [g], [m], [v], step=1, lr=1e-2, exp_avg_scales=[sc[0]] if bits == 8 else None, exp_avg_sq_scales=[sc[1]] if bits == 8 else None)
        return m, v, sc
    p2, g2 = p[-tail:].clone(), g[-tail:].clone()
    m, v, sc = step(p, g)
    m2, v2, sc2 = step(p2, g2)
    raw = lambda t: t.view(torch.uint8) if t.dtype == f8 else t          # noqa: E731
    assert torch.equal(p[-tail:], p2) and torch.equal(raw(m)[-tail:], raw(m2))
    assert (p[:-tail] == p[0]).all() and float(p[0]) < 0.5
    if bits == 32:
        assert torch.equal(v[-tail:], v2)
    else:
        k = -(-tail // 256)
        assert torch.equal(sc[0][-k:], sc2[0]) and torch.equal(sc[1][-k:], sc2[1])
        a, b = v[-tail:].float(), v2.float()
        assert ((a - b).abs() <= torch.maximum(a, b) / 8 + 2.0 ** -9).all()          # neighbours: an eighth apart at most, 2^-9 below 2^-6
