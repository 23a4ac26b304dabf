"""Two threads in one language model's forward at once: each loss is taken from its own thread's hidden states."""
import threading

import torch

from open_flamingo_amd.train import vocab as V


class Base(torch.nn.Module):
    def __init__(self, meet):
        super().__init__()
        self.wte, self.meet = torch.nn.Embedding(10, 8), meet

    def forward(self, ids):
        h = self.wte(ids)
        self.meet.wait(20)          # both threads are inside before either leaves
        return (h,)


class MptForCausalLM(torch.nn.Module):
    def __init__(self, meet):
        super().__init__()
        self.transformer = Base(meet)
        self.lm_head = torch.nn.Linear(8, 10, bias=False)
        self.lm_head.weight = self.transformer.wte.weight

    base_model = property(lambda self: self.transformer)

    def get_input_embeddings(self):
        return self.transformer.wte

    def get_output_embeddings(self):
        return self.lm_head

    def forward(self, ids, labels=None, logits_to_keep=0):
        h = self.transformer(ids)[0]
        self.transformer.meet.wait(20)          # both hidden states are made before either loss is
        return (self.lm_head(h[:, logits_to_keep]),)


def test_each_thread_s_loss_is_its_own(monkeypatch):
    monkeypatch.setattr(V, "_runs_here", lambda t: t is not None and t.dtype is torch.bfloat16)
    monkeypatch.setattr(V, "embedding_lookup", lambda ids, w, padding_idx=None: torch.nn.functional.embedding(ids, w, padding_idx))
    monkeypatch.setattr(V, "linear_cross_entropy", lambda h, w, y: (h.float().sum(), h.shape))
    lm = V.use_libofhip_vocab(MptForCausalLM(threading.Barrier(2)).bfloat16())
    got, errors = {}, []

    def one(n):
        try:
            ids = torch.full((1, n), n)
            got[n] = lm(ids, labels=ids)[0]
        except BaseException as e:          # noqa: BLE001 (the thread's failure is the test's)
            errors.append(e)

    for _ in range(3):
        threads = [threading.Thread(target=one, args=(n,)) for n in (3, 5)]
        for t in threads:
            t.start()
        for t in threads:
            t.join(60)
        assert not errors
        for n in (3, 5):
            assert got[n][1] == (1, n, 8)
            assert abs(got[n][0] - lm.lm_head.weight[n].float().sum() * n) < 1e-4
    assert not lm.transformer._forward_hooks
