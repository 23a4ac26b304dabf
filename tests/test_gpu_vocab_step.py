"""The vocabulary-table operators together on the GPU: training steps of a tiny Flamingo whose whole table is trained, a captured and replayed
run of lookup, loss, both gradients and update, other streams, and lists of every kind."""
import pytest
import torch

from tests import vocab_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def tiny(lm_loss):
    from open_flamingo_amd.train import synthetic, towers
    model, info = towers.build_flamingo("OF-tiny", device=DEV, seed=0, gates=0.5, lm_loss=lm_loss)
    model.train()
    return model, info, synthetic.make_batch(4, 2, 64, info, DEV, seed=5)


def test_train_steps_of_the_whole_table():
    from open_flamingo_amd.train import step
    from open_flamingo_amd.train.reducer import GradReducer
    runs = []
    for lm_loss, multi, bits in (("libofhip", False, 32), ("libofhip_vocab", True, 32), ("libofhip_vocab", True, 8)):
        model, info, batch = tiny(lm_loss)
        red = GradReducer(model, embedding_rows=None)
        opt = step.build_optimizer(model, lr=1e-3, reducer=red, multi_tensor=multi, state_bits=bits)
        table = model.lang_encoder.get_input_embeddings().weight
        start = table.detach().clone()
        losses = [float(step.train_step(model, red, opt, batch, info, mask_embedding_rows=False, nan_check="device" if multi else True)) for _ in range(3)]
        runs.append((losses, (table.detach() - start)))
    (l0, d0), (l1, d1), (l2, d2) = runs
    # the first arm's logits are bf16 (half a step of values below 4, averaged over 8 labels at least); the others start from the same weights
    assert abs(l1[0] - l0[0]) <= 2 ** -8 * 4 / 8 and l1[0] == l2[0]
    assert all(torch.isfinite(d).all() for d in (d0, d1, d2)) and (d1.abs().sum(1) > 0).float().mean() > 0.9


def test_captured_and_replayed_beside_eager_work():
    from open_flamingo_amd.train.optim import adamw_step
    from open_flamingo_amd.train.vocab import embedding_lookup, linear_cross_entropy
    g = torch.Generator().manual_seed(0)
    vocab, d, n = 1003, 256, 300
    ids, labels = torch.randint(0, vocab, (n,), generator=g).cuda(), torch.randint(0, vocab, (n,), generator=g).cuda()
    labels[::5] = -100
    table = torch.randn(vocab, d, generator=g).cuda() * 0.05
    f8 = torch.float8_e4m3fn
    state = lambda: dict(p=table.clone(), m=torch.zeros(vocab, d, device=DEV).to(f8), v=torch.zeros(vocab, d, device=DEV).to(f8),          # noqa: E731
                         a=torch.zeros(vocab, device=DEV), b=torch.zeros(vocab, device=DEV), t=torch.zeros(1, dtype=torch.int32, device=DEV))

    def one(s, ids, labels):
        w = s["p"].detach().requires_grad_()
        with torch.autocast("cuda", dtype=torch.bfloat16, cache_enabled=False):
            h = embedding_lookup(ids, w, scale=4.0)
            loss = linear_cross_entropy(h, w, labels)
        grad, = torch.autograd.grad(loss, w)
        adamw_step([s["p"]], [grad], [s["m"]], [s["v"]], lr=1e-2, weight_decay=0.1, max_norm=1.0, exp_avg_scales=[s["a"]], exp_avg_sq_scales=[s["b"]],
                   applied=s["t"])
        return loss.detach(), grad

    side = torch.cuda.Stream()
    cap, eager, warm = state(), state(), state()
    ids_c, labels_c = ids.clone(), labels.clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one(warm, ids_c, labels_c)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss_c, grad_c = one(cap, ids_c, labels_c)
    for k in range(4):          # every replay against the eager step on the same inputs, which change from replay to replay
        i, l = ids.roll(k), labels.roll(2 * k)
        ids_c.copy_(i)
        labels_c.copy_(l)
        graph.replay()
        loss, grad = one(eager, i, l)
        torch.cuda.synchronize()
        assert torch.equal(loss, loss_c) and torch.equal(grad, grad_c), k
        assert all(torch.equal(cap[n_].view(torch.uint8), eager[n_].view(torch.uint8)) for n_ in cap), k
    assert int(cap["t"]) == 4


def test_another_stream_and_two_calls_at_once():
    from open_flamingo_amd.train.vocab import embedding_lookup, linear_cross_entropy
    x, w, y = R.ce_inputs(700, 512, 3001, device=DEV)
    table = torch.randn(3001, 512, device=DEV)

    def both():
        a, b, t = x.detach().requires_grad_(), w.detach().requires_grad_(), table.detach().requires_grad_()
        loss = linear_cross_entropy(a, b, y)
        ids = y.clamp(min=0)
        e = embedding_lookup(ids, t)
        return (loss.detach(),) + torch.autograd.grad(loss, (a, b)) + torch.autograd.grad(e, t, x.float())

    want = both()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams * 2:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(both())
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(a, b) for a, b in zip(r, want))
