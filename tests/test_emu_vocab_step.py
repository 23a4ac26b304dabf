"""The vocabulary-table operators together, as a training step uses them (host emulator): a tiny Flamingo whose whole table is trained, lookup
and loss on libofhip, gradients of the tied table from both ends, MultiTensorAdamW."""
import pytest
import torch

from open_flamingo_amd.hip.ops import Ops
from open_flamingo_amd.src import helpers
from open_flamingo_amd.train import step, synthetic, towers
from open_flamingo_amd.train.optim import MultiTensorAdamW
from open_flamingo_amd.train.vocab import use_libofhip_vocab
from tests.emu import harness as H


@pytest.fixture
def on_emulator(monkeypatch):
    monkeypatch.setattr(helpers, "_require_hip", lambda t, what: None)
    monkeypatch.setattr("open_flamingo_amd.train.optim._require_hip", lambda t, what: None)
    monkeypatch.setattr(Ops, "default", staticmethod(H.emu_ops))
    helpers._shared.items.clear()
    yield
    helpers._shared.items.clear()


def tiny(lm_loss):
    model, info = towers.build_flamingo("OF-tiny", device="cpu", seed=0, gates=0.5, fused_lm_attention=False, lm_loss=lm_loss,
                                        vision_kw=dict(width=64, layers=2, heads=2, patch=14, image=56), perceiver_depth=1)
    model.train()
    return model, info, synthetic.make_batch(2, 2, 24, info, "cpu", seed=5, image_size=56)


def test_loss_and_gradients_are_those_of_the_head_with_logits(on_emulator):
    got = []
    for lm_loss in ("hf", "libofhip_vocab"):
        model, info, batch = tiny(lm_loss)
        loss = step.forward_loss(model, batch, info, amp=True)
        loss.backward()
        got.append((loss.detach(), {k: p.grad.clone() for k, p in model.named_parameters() if p.requires_grad}))
    (l0, g0), (l1, g1) = got
    # logits of the first arm are rounded to bf16 (half a step, 2^-8 of values below 4); everything behind the loss is the same code
    assert abs(l1 - l0) <= 2 ** -8 * 4 / 8
    assert set(g0) == set(g1)
    for k in g0:
        if g0[k].numel() > 1:          # (a gate's gradient is one sum of terms of both signs: what is left of them says nothing about their rounding)
            assert (g1[k] - g0[k]).norm() <= 2e-2 * g0[k].norm() + 1e-8, k
    table = [k for k in g0 if k.endswith("wte.weight")]
    assert len(table) == 1 and (g1[table[0]].abs().sum(1) > 0).all()          # the head's part reaches every row


def test_output_without_labels_and_with(on_emulator):
    model, info, batch = tiny("libofhip_vocab")
    model.eval()
    kw = dict(vision_x=batch["vision_x"], lang_x=batch["lang_x"], attention_mask=batch["attention_mask"])
    with torch.no_grad(), torch.autocast("cpu", dtype=torch.bfloat16):
        plain = model(**kw)
        out = model(**kw, labels=batch["lang_x"])
    assert plain.loss is None and plain.logits.shape[:2] == batch["lang_x"].shape
    assert out.logits is None and out[0] is out.loss
    want = torch.nn.functional.cross_entropy(plain.logits[:, :-1].reshape(-1, plain.logits.shape[-1]).float(), batch["lang_x"][:, 1:].reshape(-1))
    assert abs(out.loss - want) <= 2 ** -8 * 4 / 8
    with torch.no_grad():          # fp32 without autocast: the LM's own loss
        assert model(**kw, labels=batch["lang_x"]).logits is not None
    assert use_libofhip_vocab(model.lang_encoder) is model.lang_encoder          # once is enough
    with pytest.raises(NotImplementedError):
        use_libofhip_vocab(torch.nn.Linear(2, 2))


def test_a_train_step_moves_like_torch_adamw(on_emulator):
    runs = []
    for own in (False, True):
        model, info, batch = tiny("libofhip_vocab")
        opt = step.build_optimizer(model, lr=1e-3, multi_tensor=own, state_bits=8 if own else 32)
        assert isinstance(opt, MultiTensorAdamW) == own
        start = {k: p.detach().clone() for k, p in model.named_parameters() if p.requires_grad}
        loss = float(step.train_step(model, None, opt, batch, info, mask_embedding_rows=False, nan_check="device" if own else True))
        runs.append((loss, start, {k: p.detach().clone() for k, p in model.named_parameters() if p.requires_grad}))
        assert not own or opt.applied_steps() == 1
    (l0, s0, p0), (l1, s1, p1) = runs
    assert l0 == l1
    for k in p0:          # the update itself uses the moments in front of their rounding to 8 bits: fp32 arithmetic, of lr at most an element
        assert ((p1[k] - p0[k]).abs() <= 1e-3 * 1e-3 + 2.0 ** -22 * p0[k].abs()).all(), k


def test_optimizer_states_go_through_a_file(on_emulator, tmp_path):
    g = torch.Generator().manual_seed(0)
    start = [torch.randn(300, generator=g), torch.randn(4, 5, generator=g)]
    grads = [[torch.randn(300, generator=g), torch.randn(4, 5, generator=g)] for _ in range(4)]

    def make(bits, values=start):
        ps = [torch.nn.Parameter(v.clone()) for v in values]
        return ps, MultiTensorAdamW([dict(params=ps[:1], weight_decay=0.1), dict(params=ps[1:], lr=1e-2)], lr=1e-3, state_bits=bits, max_norm=1.0)

    def go(ps, opt, gs):
        for g_ in gs:
            for p, x in zip(ps, g_):
                p.grad = x.clone()
            opt.step()

    for bits in (8, 32):
        ps, opt = make(bits)
        go(ps, opt, grads[:2])
        torch.save(opt.state_dict(), tmp_path / "o.pt")
        mid = [p.detach().clone() for p in ps]
        go(ps, opt, grads[2:])
        qs, opt2 = make(bits, mid)
        opt2.load_state_dict(torch.load(tmp_path / "o.pt", weights_only=True))
        go(qs, opt2, grads[2:])
        assert all(torch.equal(p, q) for p, q in zip(ps, qs)) and opt2.applied_steps() == 4
        with pytest.raises(ValueError):
            make(40 - bits)[1].load_state_dict(opt.state_dict())
        with pytest.raises(ValueError):
            MultiTensorAdamW([torch.nn.Parameter(torch.zeros(2))]).load_state_dict(opt.state_dict())
    # 32 bits: torch's own optimizer takes the state over
    ref = torch.optim.AdamW([dict(params=ps[:1], weight_decay=0.1), dict(params=ps[1:], lr=1e-2)], lr=1e-3)
    ref.load_state_dict(opt.state_dict())
    assert float(ref.state[ps[0]]["step"]) == 4


def test_optimizer_refusals_and_parameters_without_gradients(on_emulator):
    p, q = torch.nn.Parameter(torch.ones(8)), torch.nn.Parameter(torch.ones(8))
    with pytest.raises(ValueError):
        MultiTensorAdamW([p], state_bits=16)
    with pytest.raises(ValueError):
        MultiTensorAdamW([torch.nn.Parameter(torch.ones(8).bfloat16())])
    with pytest.raises(ValueError):
        step.build_optimizer(torch.nn.Linear(2, 2), state_bits=8)
    opt = MultiTensorAdamW([dict(params=[p]), dict(params=[q], betas=(0.5, 0.9))])
    with pytest.raises(ValueError):
        opt.step()
    opt = MultiTensorAdamW([p, q], lr=1e-2)
    opt.step()                                          # nothing has a gradient: nothing happens
    assert opt.applied_steps() == 0
    q.grad = torch.ones(8)
    opt.step()
    assert (p == 1).all() and (q < 1).all() and p not in opt.state and abs(float(opt.grad_norm()) - 8 ** 0.5) < 1e-5
