"""What the vocabulary-table operators cost: their plain forms beside the kernels of this framework.

Three operators meet at the language model's (vocabulary x d) table when it is trained:

* ``ce``     -- the tied head's loss: softmax cross entropy of ``hidden @ table.T`` in pieces of the vocabulary, the logits never kept,
               with the gradients of the hidden states and of the table;
* ``embed``  -- the lookup ``scale * table[ids]`` and its gradient by sorted tokens;
* ``adamw``  -- clip + AdamW over many tensors at once, moments in 32 bits or in 8.

``own`` = False: elementary torch operations in 32 bits (64 for the long sums of the gradient norm), rounded once at the end.
``own`` = True: the calls that a user of the framework makes.
"""
import math

import torch

own = False

DEV = "cuda"
BF16, F32, F64, F8 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn

# ---------------------------------------------------------------------------------------------------------------- the cases
# Vocabulary 50435 = 50432 + 3 added tokens; d = 2048 / 2560 / 4096 of the three model families; the tiny test family is d = 256,
# vocabulary 1003.  `valid` = share of positions with a label (the rest are padding, media tokens and text in front of an image).


def listed():
    return [
        # 32 sequences of 256 tokens, the whole table trained (d = 2048): loss + both gradients
        dict(name="ce train 8192x2048", op="ce", rows=8192, d=2048, vocab=50435, valid=0.9, grad="both", ragged=False),
        # the widest family, 8192 tokens (d = 4096)
        dict(name="ce train 8192x4096", op="ce", rows=8192, d=4096, vocab=50435, valid=0.95, grad="both", ragged=False),
        # captions: 64 rows of 32 tokens cut to an odd count, half of them padding, frozen table: the hidden states' gradient alone
        dict(name="ce frozen table 1999x2560", op="ce", rows=1999, d=2560, vocab=50435, valid=0.5, grad="hidden", ragged=False),
        # the tiny test family's step: where launches count
        dict(name="ce tiny 64x256", op="ce", rows=64, d=256, vocab=1003, valid=0.8, grad="both", ragged=False),
        # scoring one next token (evaluation by likelihood): a single row, no gradient
        dict(name="ce score 1x2048", op="ce", rows=1, d=2048, vocab=50435, valid=1.0, grad="none", ragged=False),
        # fp32 table of the smallest family, 32 x 256 tokens, dense fp32 gradient
        dict(name="embed train 8192x2048", op="embed", n=8192, d=2048, vocab=50435, dtype="float32", scale=1.0, skew=1.0, grad=True),
        # bf16 table of the widest family, 16 sequences of 2048 tokens, the frequent ids very frequent, the lookup scaled
        dict(name="embed train bf16 32768x4096", op="embed", n=32768, d=4096, vocab=50435, dtype="bfloat16", scale=64.0, skew=2.0, grad=True),
        # one new token for each of 8 sequences (decode)
        dict(name="embed decode 8x2048", op="embed", n=8, d=2048, vocab=50435, dtype="float32", scale=1.0, skew=1.0, grad=False),
        # one trained vocabulary table and the matrices and vectors of gated blocks, moments in 32 bits
        dict(name="adamw 32 bits 160 tensors", op="adamw", tensors=160, elements=120_000_000, bits=32, clip=1.0, wd=0.1, grad_dtype="float32"),
        # the same in 8 bits
        dict(name="adamw 8 bits 160 tensors", op="adamw", tensors=160, elements=120_000_000, bits=8, clip=1.0, wd=0.1, grad_dtype="float32"),
        # a small trainable set, odd sizes: where launches count
        dict(name="adamw 8 bits 24 small", op="adamw", tensors=24, elements=60_007, bits=8, clip=1.0, wd=0.0, grad_dtype="bfloat16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ce", "ce", "embed", "adamw"])
    if op == "ce":
        while True:
            c = dict(op=op, rows=_log(rng, 1, 8192), d=64 * rng.randint(4, 64), vocab=_log(rng, 1000, 66000), valid=round(rng.uniform(0.3, 1.0), 3),
                     grad=rng.choice(["both", "both", "hidden", "none"]), ragged=rng.random() < 0.3)
            if c["rows"] * c["d"] * c["vocab"] <= 8192 * 4096 * 50435:
                return c
    if op == "embed":
        while True:
            c = dict(op=op, n=_log(rng, 1, 60000), d=8 * rng.randint(8, 512) + (rng.randint(1, 7) if rng.random() < 0.2 else 0),
                     vocab=_log(rng, 1000, 66000), dtype=rng.choice(["float32", "bfloat16"]), scale=rng.choice([1.0, 0.5, 45.25]),
                     skew=round(rng.uniform(0.5, 3.0), 2), grad=rng.random() < 0.75)
            if (c["n"] + c["vocab"]) * c["d"] <= (32768 + 50435) * 4096:
                return c
    n = _log(rng, 1000, 100_000_000)
    return dict(op=op, tensors=min(n // 50, _log(rng, 1, 200)), elements=n, bits=rng.choice([8, 32]), clip=rng.choice([0.0, 1.0]), wd=rng.choice([0.0, 0.1]),
                grad_dtype=rng.choice(["float32", "bfloat16"]))


# ---------------------------------------------------------------------------------------------------------------- inputs


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _sizes(case):
    """Element counts of the tensors: two matrices, then one vector of 1/500 of their size, and so on; odd sizes throughout."""
    t, n = case["tensors"], case["elements"]
    share = [1.0 if i % 3 != 2 else 0.002 for i in range(t)]
    total = sum(share)
    return [max(1, int(n * s / total) | 1) for s in share]


def _amax256(t):
    """The largest magnitude of each 256 elements."""
    return t.abs().view(-1, 256).amax(dim=1)


def _codes(t, top):
    """Elements in units of their block's largest / 448 (the largest e4m3 value)."""
    return (t.view(-1, 256) * (448.0 / top.clamp(min=1e-30))[:, None]).clamp_(-448.0, 448.0).view(-1)


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "ce":
        r, d, v = case["rows"], case["d"], case["vocab"]
        pad = 8 if case["ragged"] else 0                       # rows of a wider buffer: a stride that is not d
        x = torch.randn(r, d + pad, generator=g, device=DEV).to(BF16)[:, :d]      # behind the final norm: unit variance
        w = (torch.randn(v, d, generator=g, device=DEV) * (2.0 / math.sqrt(d))).to(BF16)
        labels = torch.randint(0, v, (r,), generator=g, device=DEV)
        drop = torch.rand(r, generator=g, device=DEV) >= case["valid"]
        drop[0] = False                                          # a step whose labels are all ignored is tested elsewhere
        labels = labels.masked_fill(drop, -100)
        return dict(case=case, x=x, w=w, labels=labels)
    if case["op"] == "embed":
        n, d, v = case["n"], case["d"], case["vocab"]
        dt = getattr(torch, case["dtype"])
        table = torch.randn(v, d, generator=g, device=DEV).to(dt)
        # text: small ids are frequent (skew 1: uniform); the last id stands for padding and takes a tenth of the positions
        ids = (torch.rand(n, generator=g, device=DEV, dtype=F64) ** (case["skew"] * 2 - 1 if case["skew"] > 1 else 1.0) * v).long().clamp_(max=v - 1)
        ids = torch.where(torch.rand(n, generator=g, device=DEV) < 0.1, torch.full_like(ids, v - 1), ids)
        dy = torch.randn(n, d, generator=g, device=DEV).to(dt) if case["grad"] else None
        return dict(case=case, table=table.requires_grad_(case["grad"]), ids=ids, dy=dy)
    sizes = _sizes(case)
    starts, at = [], 0
    for k in sizes:                                              # every tensor begins at a multiple of 256 elements of one buffer
        starts.append(at)
        at += -(-k // 256) * 256
    gd = getattr(torch, case["grad_dtype"])
    p = torch.randn(at, generator=g, device=DEV) * 0.02
    grad = (torch.randn(at, generator=g, device=DEV) * torch.rand(at, generator=g, device=DEV).pow_(4) * 1e-3).to(gd)
    m = torch.randn(at, generator=g, device=DEV) * 1e-4
    r = torch.rand(at, generator=g, device=DEV).pow_(2) * 1e-3 + 1e-6            # square root of the second moment
    for s, k in zip(starts, sizes):
        for t in (p, grad, m, r):
            t[s + k:s + -(-k // 256) * 256] = 0
    cut = lambda t: [t[s:s + k] for s, k in zip(starts, sizes)]  # noqa: E731
    st = dict(case=case, step=100, p=p, g=grad, starts=starts, sizes=sizes)
    if case["bits"] == 32:
        st.update(m=m, v=r * r, m_scales=None, v_scales=None)
    else:
        # what earlier steps left: 8-bit codes of the first moment and of the square root of the second, one scale per 256 elements
        tm, tr = _amax256(m), _amax256(r)
        blocks = lambda t: [t[s // 256:s // 256 + -(-k // 256)] for s, k in zip(starts, sizes)]  # noqa: E731
        st.update(m=_codes(m, tm).to(F8), v=_codes(r, tr).to(F8), m_scale=tm / 448.0, v_scale=tr / 448.0)
        st.update(m_scales=blocks(st["m_scale"]), v_scales=blocks(st["v_scale"]))
    st.update(ms=cut(st["m"]), vs=cut(st["v"]))
    st.update(ps=cut(p), gs=cut(grad))
    return st


# ---------------------------------------------------------------------------------------------------------------- one pass


def run(s):
    return dict(ce=_run_ce, embed=_run_embed, adamw=_run_adamw)[s["case"]["op"]](s)


def _run_ce(s):
    c, x, w, labels = s["case"], s["x"], s["w"], s["labels"]
    if own:
        from open_flamingo_amd.train.vocab import linear_cross_entropy
        if c["grad"] == "none":
            with torch.no_grad():
                return dict(loss=linear_cross_entropy(x, w, labels, reduction="none"))
        x = x.detach().requires_grad_(True)
        w = w.detach().requires_grad_(c["grad"] == "both")
        loss = linear_cross_entropy(x, w, labels)
        grads = torch.autograd.grad(loss, (x, w) if c["grad"] == "both" else (x,))
        return dict(loss=loss.detach(), **dict(zip(("dhidden", "dtable"), grads)))
    keep = labels != -100
    at = labels.clamp(min=0)
    xf, wf = x.float(), w.float()
    z = xf @ wf.t()
    top = z.max(dim=1, keepdim=True).values
    e = torch.exp(z - top)
    tot = e.sum(dim=1, keepdim=True)
    nll = (top + torch.log(tot)).squeeze(1) - z.gather(1, at[:, None]).squeeze(1)
    nll = torch.where(keep, nll, torch.zeros_like(nll))
    if c["grad"] == "none":
        return dict(loss=nll)
    n = keep.sum()
    loss = nll.sum() / n
    dz = e.div_(tot)
    dz.scatter_add_(1, at[:, None], torch.full_like(dz[:, :1], -1.0))
    dz.mul_((keep / n)[:, None])
    out = dict(loss=loss, dhidden=(dz @ wf).to(x.dtype))
    if c["grad"] == "both":
        out["dtable"] = (dz.t() @ xf).to(w.dtype)
    return out


def _run_embed(s):
    c, table, ids, dy = s["case"], s["table"], s["ids"], s["dy"]
    pad = c["vocab"] - 1
    if own:
        from open_flamingo_amd.train.vocab import embedding_lookup
        if not c["grad"]:
            with torch.no_grad():
                return dict(y=embedding_lookup(ids, table, scale=c["scale"], padding_idx=pad))
        y = embedding_lookup(ids, table, scale=c["scale"], padding_idx=pad)
        return dict(y=y.detach(), dtable=torch.autograd.grad(y, table, dy)[0])
    y = (table.detach()[ids].float() * c["scale"]).to(table.dtype)
    if not c["grad"]:
        return dict(y=y)
    d = torch.zeros(c["vocab"], c["d"], dtype=F32, device=table.device)
    d.index_add_(0, ids, torch.where((ids == pad)[:, None], torch.zeros((), device=ids.device), dy.float()) * c["scale"])
    return dict(y=y, dtable=d.to(table.dtype))


LR, B1, B2, EPS = 1e-4, 0.9, 0.999, 1e-8


def _uniform20(ordinal, index, step):
    """20 random bits per element: a fixed mixing of (tensor, element, step) in 32-bit integers."""
    m = 0xFFFFFFFF
    x = ((index ^ ((step * 0x9E3779B1 + ordinal * 0x85157AF5) & m)) * 0x9E3779B1) & m
    x = ((x ^ (x >> 15)) * 0x85157AF5) & m
    x = ((x ^ (x >> 13)) * 0x9E3779B1) & m
    return (x ^ (x >> 16)) & 0xFFFFF


def _run_adamw(s):
    c = s["case"]
    s["step"] += 1
    t = s["step"]
    if own:
        from open_flamingo_amd.train.optim import adamw_step
        adamw_step(s["ps"], s["gs"], s["ms"], s["vs"], step=t, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=c["wd"], max_norm=c["clip"],
                   exp_avg_scales=s["m_scales"], exp_avg_sq_scales=s["v_scales"])
    else:
        _plain_adamw(s, t)
    return dict(p=s["p"], m=s["m"], v=s["v"], **({} if c["bits"] == 32 else dict(m_scale=s["m_scale"], v_scale=s["v_scale"])))


def _plain_adamw(s, t):
    c, p = s["case"], s["p"]
    norm = s["g"].double().square().sum().sqrt().float()
    g = s["g"].float()
    if c["clip"] > 0:
        g = g * (c["clip"] / (norm + 1e-6)).clamp(max=1.0)
    if c["bits"] == 32:
        m, v = s["m"], s["v"]
    else:
        m = (s["m"].float().view(-1, 256) * s["m_scale"][:, None]).view(-1)
        v = (s["v"].float().view(-1, 256) * s["v_scale"][:, None]).view(-1).square()
    m = m * B1 + g * (1 - B1)
    v = v * B2 + g * (1 - B2) * g
    p.mul_(1 - LR * c["wd"]).sub_((m / (v.sqrt() * (1 / math.sqrt(1 - B2 ** t)) + EPS)) * (LR / (1 - B1 ** t)))
    if c["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return
    # first moment: to the nearest code; square root of the second: up or down at random in proportion (a mean that moves by 1/1000 a
    # step would stand still in 8 bits otherwise), never from above zero to zero
    r = v.sqrt()
    tm, tr = _amax256(m), _amax256(r)
    s["m"].copy_(_codes(m, tm).to(F8))
    q = _codes(r, tr)
    n = len(s["sizes"])
    first = torch.tensor(s["starts"] + [p.numel()], device=DEV)
    which = torch.repeat_interleave(torch.arange(n, device=DEV), first.diff(), output_size=p.numel())
    u = _uniform20(which, torch.arange(p.numel(), device=DEV) - first[which], t)
    up = ((q.view(torch.int32) + u.int()) & -0x100000).view(F32).clamp(max=448.0)             # 20 of the 23 mantissa bits go
    low = torch.floor(q * 512.0 + u.float() * 2.0 ** -20) / 512.0                             # below 2^-6 the codes are 2^-9 apart
    q8 = torch.where(q >= 2.0 ** -6, up, low)
    q8 = torch.where(q > 0, q8.clamp(min=2.0 ** -9), q8)
    s["v"].copy_(q8.to(F8))
    s["m_scale"].copy_(tm / 448.0)
    s["v_scale"].copy_(tr / 448.0)


# ---------------------------------------------------------------------------------------------------------------- costs


def work(case):
    if case["op"] == "ce":
        r, d, v = case["rows"], case["d"], case["vocab"]
        n = dict(none=1, hidden=2, both=3)[case["grad"]]                       # products of rows x d x vocab
        by = 2 * (r * d + v * d) + 8 * r + (0 if case["grad"] == "none" else 2 * r * d) + (2 * v * d if case["grad"] == "both" else 0)
        return dict(bytes=by, flops=2 * n * r * d * v)
    if case["op"] == "embed":
        n, d, v, e = case["n"], case["d"], case["vocab"], 4 if case["dtype"] == "float32" else 2
        by = 8 * n + 2 * n * d * e                                              # ids, the rows read and written
        if case["grad"]:
            by += n * d * e + v * d * e                                         # the upstream gradient read, the table's written whole
        return dict(bytes=by, flops=n * d * (3 if case["grad"] else 1))
    n = sum(_sizes(case))
    state = 16 if case["bits"] == 32 else 4 + 4 * 4 / 256                      # both moments read and written
    return dict(bytes=n * (8 + state + (4 if case["grad_dtype"] == "float32" else 2)), flops=16 * n)


# ---------------------------------------------------------------------------------------------------------------- in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "ce":
        x, w = s["x"].double(), s["w"].double()
        live = (s["labels"] >= 0).nonzero().squeeze(1)
        r = case["rows"]
        loss = torch.zeros(r, dtype=F64, device=DEV)
        dx, dw = torch.zeros_like(x), torch.zeros_like(w)
        for k in range(0, live.numel(), 2048):
            i = live[k:k + 2048]
            z = x[i] @ w.t()
            lp = torch.log_softmax(z, dim=1)
            lab = s["labels"][i]
            loss[i] = -lp.gather(1, lab[:, None]).squeeze(1)
            if case["grad"] != "none":
                dz = lp.exp_()
                dz[torch.arange(i.numel(), device=DEV), lab] -= 1.0
                dz /= live.numel()
                dx[i] = dz @ w
                dw += dz.t() @ x[i]
        if case["grad"] == "none":
            return dict(loss=loss)
        return dict(loss=loss.sum() / live.numel(), dhidden=dx, **(dict(dtable=dw) if case["grad"] == "both" else {}))
    if case["op"] == "embed":
        t, ids = s["table"].detach().double(), s["ids"]
        y = t[ids] * case["scale"]
        if not case["grad"]:
            return dict(y=y)
        keep = ids != case["vocab"] - 1
        order = torch.argsort(ids[keep], stable=True)
        dy = s["dy"].double()[keep][order] * case["scale"]
        which, count = torch.unique_consecutive(ids[keep][order], return_counts=True)
        d = torch.zeros(case["vocab"], case["d"], dtype=F64, device=DEV)
        d[which] = torch.segment_reduce(dy, "sum", lengths=count, axis=0) if which.numel() else d[which]
        return dict(y=y, dtable=d)
    return _exact_adamw(case, s)


def _exact_adamw(case, s):
    t = s["step"] + 1
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in s["gs"]))
    c = min(1.0, case["clip"] / (norm + 1e-6)) if case["clip"] > 0 else 1.0
    out = dict(p=torch.zeros(s["p"].numel(), dtype=F64, device=DEV))
    b32 = case["bits"] == 32
    if b32:
        out.update(m=torch.zeros_like(out["p"]), v=torch.zeros_like(out["p"]))
    else:
        out.update(m=None, v=None, m_scale=torch.zeros_like(s["m_scale"], dtype=F64), v_scale=torch.zeros_like(s["v_scale"], dtype=F64))
    for i, (a, k) in enumerate(zip(s["starts"], s["sizes"])):
        g = s["gs"][i].double() * c
        m, v = s["ms"][i].double(), s["vs"][i].double()
        if not b32:
            m = m * s["m_scales"][i].double().repeat_interleave(256)[:k]
            v = (v * s["v_scales"][i].double().repeat_interleave(256)[:k]) ** 2
        m = B1 * m + (1 - B1) * g
        v = B2 * v + (1 - B2) * g * g
        out["p"][a:a + k] = s["ps"][i].double() * (1 - LR * case["wd"]) - LR / (1 - B1 ** t) * m / (torch.sqrt(v / (1 - B2 ** t)) + EPS)
        if b32:
            out["m"][a:a + k], out["v"][a:a + k] = m, v
        else:
            b, n = a // 256, -(-k // 256)
            top = lambda z: torch.nn.functional.pad(z.abs(), (0, n * 256 - k)).view(n, 256).amax(1) / 448.0  # noqa: E731
            out["m_scale"][b:b + n], out["v_scale"][b:b + n] = top(m), top(v.sqrt())
    return out
