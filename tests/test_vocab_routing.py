"""Which calls of a routed language model go to the loss without logits, and which keep the LM's own head (no GPU and no kernel: the operator is
recorded in place of run)."""
import pytest
import torch

from open_flamingo_amd.train import vocab as V


class Base(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.wte = torch.nn.Embedding(10, 8)

    def forward(self, ids):
        return (self.wte(ids),)


class MptForCausalLM(torch.nn.Module):
    """the parts of a Hugging Face causal LM that the routing uses"""

    def __init__(self, head=None):
        super().__init__()
        self.transformer = Base()
        self.lm_head = head or torch.nn.Linear(8, 10, bias=False)

    base_model = property(lambda self: self.transformer)

    def get_input_embeddings(self):
        return self.transformer.wte

    def get_output_embeddings(self):
        return self.lm_head

    def forward(self, ids, labels=None, logits_to_keep=0):
        h = self.transformer(ids)[0]
        logits = self.lm_head(h if isinstance(logits_to_keep, int) else h[:, logits_to_keep])
        return (logits,) if labels is None else ("own", logits)


@pytest.fixture
def route(monkeypatch):
    monkeypatch.setattr(V, "_runs_here", lambda t: t is not None and t.dtype in (torch.bfloat16, torch.float32))
    monkeypatch.setattr(V, "embedding_lookup", lambda ids, w, padding_idx=None: torch.nn.functional.embedding(ids, w, padding_idx))
    monkeypatch.setattr(V, "linear_cross_entropy", lambda h, w, y: "operator")
    ids = torch.tensor([[1, 2, 3]])
    return lambda lm: lm(ids, labels=ids)[0]


def test_autocast_decides_the_heads_type_and_so_the_route(route):
    half, full = (V.use_libofhip_vocab(MptForCausalLM().to(t)) for t in (torch.bfloat16, torch.float32))
    assert route(half) == "operator" and route(full) == "own"
    with torch.autocast("cpu", dtype=torch.bfloat16):
        assert route(half) == route(full) == "operator"
    with torch.autocast("cpu", dtype=torch.float16):          # the LM's own head multiplies in fp16 here, also where its weight is bf16
        assert route(half) == route(full) == "own"


def test_a_head_that_does_more_than_multiply_is_not_passed_by(route):
    class Scaled(torch.nn.Linear):
        def forward(self, x):
            return 2 * super().forward(x)

    class Adapter(torch.nn.Module):          # a wrapper that shows its base's weight
        def __init__(self, base):
            super().__init__()
            self.base = base

        weight = property(lambda self: self.base.weight)
        bias = property(lambda self: self.base.bias)

        def forward(self, x):
            return self.base(x) + 1

    plain = torch.nn.Linear(8, 10, bias=False)
    patched, hooked, before = (torch.nn.Linear(8, 10, bias=False) for _ in range(3))
    patched.forward = lambda x: x @ patched.weight.t() * 3
    hook = hooked.register_forward_hook(lambda mod, args, out: out + 1)
    before.register_forward_pre_hook(lambda mod, args: (args[0] * 2,))
    tied = torch.nn.utils.parametrize.register_parametrization(torch.nn.Linear(8, 10, bias=False), "weight", torch.nn.Identity())
    want = [(plain, "operator"), (tied, "operator"), (Scaled(8, 10, bias=False), "own"), (Adapter(torch.nn.Linear(8, 10, bias=False)), "own"), (patched, "own"),
            (hooked, "own"), (before, "own"), (torch.nn.Linear(8, 10), "own")]
    for i, (head, path) in enumerate(want):
        assert route(V.use_libofhip_vocab(MptForCausalLM(head).bfloat16())) == path, i
    hook.remove()          # without it the head is a plain product again
    assert route(V.use_libofhip_vocab(MptForCausalLM(hooked).bfloat16())) == "operator"


def test_a_lookup_that_was_patched_before_stays(route):
    lm = MptForCausalLM()
    own = lm.transformer.wte.forward
    lm.transformer.wte.forward = lambda ids: 2 * own(ids)
    ids = torch.tensor([[1, 2]])
    assert torch.equal(V.use_libofhip_vocab(lm).transformer.wte(ids), 2 * lm.transformer.wte.weight[ids])
    first = V.use_libofhip_vocab(MptForCausalLM())
    third = MptForCausalLM()
    third.transformer.wte = first.transformer.wte          # a table of two LMs, routed by both
    V.use_libofhip_vocab(third)
    half = third.half().transformer.wte          # a type the operator does not take: the module's own lookup
    assert torch.equal(half(ids), half.weight[ids])
