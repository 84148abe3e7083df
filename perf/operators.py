"""The workloads that the operators of the softmax anchor layers are measured on (the attention layers that a hybrid
model keeps between its recurrent ones): what each is, how its inputs are made, one pass of it, and the work it
cannot do without.

- ``attention``  causal attention over a packed batch of prompts with grouped heads, forward alone or with the
                 gradients of q, k and v;
- ``rotary``     rotary positions of q and k: halves or interleaved pairs, the whole head or its first part, plain or
                 scaled frequencies, and the inverse rotation (what gradients take);
- ``pages``      the paged cache: pages copied (forks that write, compaction), and new tokens' k and v put into it;
- ``tree``       attention of each sequence's new tokens (one, or a tree of drafts) over its pages and themselves.
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda:0"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _anchor():
    """The framework's operators (its modules are imported from its own folder, as its tests do)."""
    path = os.path.join(os.getcwd(), "kernel-deltanet_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from kdn import anchor
    return anchor


# ------------------------------------------------------------------------------------------------- the cases


def listed():
    return [
        # A few short prompts of one serving step, 64-wide heads as the recurrent layers have them.
        dict(name="prompt_packed", kind="attention", seqs=7, lo=33, hi=2048, H=16, KV=4, d=64, dtype="bf16", train=False),
        # One long prompt, 32 heads of 128 (the factored layers' heads) over 8 shared ones.
        dict(name="prompt_16k", kind="attention", seqs=1, lo=16384, hi=16384, H=32, KV=8, d=128, dtype="bf16", train=False),
        # The smallest training step: three ragged sequences in fp32, four heads.
        dict(name="train_small_f32", kind="attention", seqs=3, lo=101, hi=1024, H=4, KV=2, d=64, dtype="f32", train=True),
        # A training step of a long sequence.
        dict(name="train_8k", kind="attention", seqs=1, lo=8192, hi=8192, H=32, KV=8, d=128, dtype="bf16", train=True),
        # The positions of a decode step of nine streams far into their contexts: a launch's latency.
        dict(name="rotary_step", kind="rotary", tokens=9, lo=70000, hi=131072, H=16, KV=4, d=64, rot=32, pairs=True,
             scaling="none", inverse=False, dtype="bf16"),
        # A 64k prompt beyond the length its frequencies were trained at.
        dict(name="rotary_64k", kind="rotary", tokens=65536, lo=0, hi=65536, H=32, KV=8, d=128, rot=128, pairs=False,
             scaling="parts", inverse=False, dtype="bf16"),
        # Nine forked streams about to write: the last page of each is copied, all layers.
        dict(name="pages_fork", kind="pages", op="copy", pages=256, move=9, layers=4, KV=4, P=16, d=64, dtype="bf16"),
        # Compaction: a quarter of a pool of full-size pages moves down.
        dict(name="pages_compact", kind="pages", op="copy", pages=4096, move=1021, layers=4, KV=8, P=32, d=128, dtype="bf16"),
        # The keys and values of a step's prompts into their pages.
        dict(name="pages_append", kind="pages", op="append", pages=2048, tokens=16001, layers=2, KV=8, P=16, d=128, dtype="bf16"),
        # One token each of three streams, fp32: a decode step's latency.
        dict(name="decode_small_f32", kind="tree", seqs=3, lo=700, hi=2500, drafts=1, H=16, KV=4, P=16, d=64, dtype="f32"),
        # A full decode batch: 224 streams at contexts from 512 to 16384.
        dict(name="decode_full", kind="tree", seqs=224, lo=512, hi=16384, drafts=1, H=16, KV=4, P=16, d=128, dtype="bf16"),
        # Sixteen streams verify trees of 20 to 40 drafted tokens.
        dict(name="tree_verify", kind="tree", seqs=16, lo=1500, hi=16384, drafts=40, H=32, KV=8, P=32, d=128, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "rotary", "pages", "tree", "tree"])
    dtype = "f32" if rng.random() < 0.25 else "bf16"
    d = rng.choice([64, 128])
    H, KV = rng.choice([(4, 4), (4, 2), (8, 1), (12, 4), (16, 4), (16, 16), (32, 8)])
    if kind == "attention":
        train = rng.random() < 0.5
        seqs = _log_int(rng, 1, 16)
        top = _log_int(rng, 100, 8192 if H <= 16 and not train else 4096)
        top = min(top, int(16384 / math.sqrt(seqs)))
        if dtype == "f32":
            top = min(top, 2048)
        return dict(kind=kind, seqs=seqs, lo=max(1, int(top * rng.choice([0.02, 0.3, 0.9]))), hi=top, H=H, KV=KV, d=d, dtype=dtype,
                    train=train)
    if kind == "rotary":
        lo = rng.choice([0, 0, 5000, 100000])
        return dict(kind=kind, tokens=_log_int(rng, 1, 50000), lo=lo, hi=lo + _log_int(rng, 100, 130000), H=H, KV=KV, d=d,
                    rot=rng.choice([d, d, d // 2, d // 4]), pairs=rng.random() < 0.5,
                    scaling=rng.choice(["none", "linear", "base", "parts"]), inverse=rng.random() < 0.3, dtype=dtype)
    if kind == "pages":
        P, layers = rng.choice([16, 16, 32, 64]), rng.choice([1, 2, 4])
        if rng.random() < 0.5:
            pages = _log_int(rng, 64, 2048)
            return dict(kind=kind, op="copy", pages=pages, move=_log_int(rng, 1, pages // 3), layers=layers, KV=KV, P=P, d=d, dtype=dtype)
        tokens = _log_int(rng, 1, 20000)
        return dict(kind=kind, op="append", pages=tokens // P + _log_int(rng, 8, 500), tokens=tokens, layers=layers, KV=KV, P=P, d=d,
                    dtype=dtype)
    hi = _log_int(rng, 64, 16384)
    seqs = _log_int(rng, 1, max(1, min(128, 1000000 // hi // max(1, KV // 4))))
    return dict(kind=kind, seqs=seqs, lo=max(1, int(hi * rng.choice([0.05, 0.5]))), hi=hi, drafts=rng.choice([1, 1, 1, 5, 16, 33, 64]), H=H,
                KV=KV, P=rng.choice([16, 16, 32, 64]), d=d, dtype=dtype)


def _lens(case):
    """The lengths of a case's sequences: between lo and hi, spread over their logarithm, the longest first."""
    rng = random.Random("%d %d %d" % (case["seqs"], case["lo"], case["hi"]))
    return [case["hi"]] + [_log_int(rng, case["lo"], case["hi"]) for _ in range(case["seqs"] - 1)]


def _drafts(case):
    """How many new tokens each sequence has: one, or between half and all of `drafts`."""
    n = case["drafts"]
    rng = random.Random("%d %d" % (case["seqs"], n))
    return [n if n == 1 else rng.randint((n + 1) // 2, n) for _ in range(case["seqs"])]


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    d, KV = case["d"], case["KV"]
    if case["kind"] == "attention":
        lens, H = _lens(case), case["H"]
        rows, pairs = sum(lens), sum(n * (n + 1) // 2 for n in lens)
        once = rows * d * (2 * H + 2 * KV) * size  # q, y; k, v
        # two products forward; five backward, each over the visible pairs alone
        return {"bytes": once * (2 if case["train"] else 1), "flops": 2 * d * H * pairs * (7 if case["train"] else 2)}
    if case["kind"] == "rotary":
        n, heads = case["tokens"], case["H"] + KV
        return {"bytes": 2 * n * heads * d * size + 8 * n, "flops": 3 * n * heads * case["rot"]}
    if case["kind"] == "pages":
        if case["op"] == "copy":
            return {"bytes": 2 * case["move"] * case["layers"] * 2 * KV * case["P"] * d * size, "flops": 0}
        return {"bytes": 4 * case["tokens"] * KV * d * size + 8 * case["tokens"], "flops": 0}
    new, lens, H = _drafts(case), _lens(case), case["H"]
    rows = sum(new)
    pairs = sum(n * c for n, c in zip(new, lens)) + rows
    return {"bytes": 2 * (sum(lens) + rows) * KV * d * size + 2 * rows * H * d * size, "flops": 4 * d * H * pairs}


# ------------------------------------------------------------------------------------------------- inputs


def _offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int64, device=DEV)


def _frequencies(rot, scaling):
    """Radians a position for each pair of a rotated part of `rot` values, and the factor of its rotation: base 10000;
    scaled by 4 for contexts four times 4096: all of them, by a larger base, or only those that turn seldom."""
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
    if scaling == "linear":
        return f / 4, 1.0
    if scaling == "base":
        return (10000.0 * 4.0 ** (rot / max(1, rot - 2))) ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot), 1.0
    if scaling == "parts":
        keep = ((4096 * f / (2 * math.pi) - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        return f / 4 * (1 - keep) + f * keep, 0.1 * math.log(4.0) + 1.0
    return f, 1.0


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    host = random.Random(seed)
    dt, d, KV = DTYPES[case["dtype"]], case["d"], case["KV"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV).to(dt)

    s = dict(case=case)
    if case["kind"] in ("attention", "rotary", "tree"):
        H = case["H"]
        n = sum(_lens(case)) if case["kind"] == "attention" else case["tokens"] if case["kind"] == "rotary" else sum(_drafts(case))
        # one projection's output: q, k and v are views of its heads
        s["q"], s["k"], s["v"] = normal(n, H + 2 * KV, d).split([H, KV, KV], dim=1)
    if case["kind"] == "attention":
        lens = _lens(case)
        s.update(cu=_offsets(lens), longest=max(lens))
        if case["train"]:
            s["dy"] = normal(sum(lens), case["H"], d)
    elif case["kind"] == "rotary":
        pos = torch.randint(case["lo"], case["hi"], (case["tokens"],), generator=g, device=DEV)
        f, mag = _frequencies(case["rot"], case["scaling"])
        s.update(pos=pos, freq=f, mag=mag)
    elif case["kind"] == "pages":
        slab = torch.empty(case["pages"], case["layers"], 2, KV, case["P"], d, dtype=dt, device=DEV)
        for part in slab.split(256):
            part.copy_(torch.randn(part.shape, generator=g, device=DEV))
        order = list(range(case["pages"]))
        host.shuffle(order)
        s["slab"] = slab
        if case["op"] == "copy":  # pages that stay distinct, as a pool's bookkeeping on the host names them
            m = case["move"]
            s["moves"] = torch.tensor([[a, b] for a, b in zip(order[:m], order[m:2 * m])], dtype=torch.int32)
        else:  # whole pages in the order in which the pool gave them out
            n, P = case["tokens"], case["P"]
            s["k"], s["v"] = normal(n, 2 * KV, d).split([KV, KV], dim=1)
            at = torch.tensor(order[:-(-n // P)], dtype=torch.int64, device=DEV)
            t = torch.arange(n, device=DEV)
            s["rows"] = at[t // P] * P + t % P
    else:
        lens, new, P = _lens(case), _drafts(case), case["P"]
        counts = [-(-c // P) for c in lens]
        total = sum(counts)
        slab = torch.empty(total, 2, KV, P, d, dtype=dt, device=DEV)
        for part in slab.split(4096):
            part.copy_(torch.randn(part.shape, generator=g, device=DEV))
        order = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
        col = torch.arange(max(counts), device=DEV)
        first = _offsets(counts)[:-1]
        s["table"] = order[(first[:, None] + col[None]).clamp(max=total - 1)].contiguous()
        s.update(k_pages=slab[:, 0], v_pages=slab[:, 1], lens=torch.tensor(lens, dtype=torch.int32, device=DEV), cu=_offsets(new),
                 most=max(new), longest=max(lens))
        # each drafted token hangs on one before it, the first on the context
        s["parents"] = torch.tensor([host.randint(max(0, i - 6), i - 1) if i else -1 for m in new for i in range(m)], dtype=torch.int32,
                                    device=DEV)
    return s


# ------------------------------------------------------------------------------------------------- one pass


def run(s):
    kind = s["case"]["kind"]
    if own:
        return _own(s)
    return {"attention": _plain_attention, "rotary": _plain_rotary, "pages": _plain_pages, "tree": _plain_tree}[kind](s)


def _own(s):
    A, c = _anchor(), s["case"]
    if c["kind"] == "attention":
        if not c["train"]:
            return A.attention(s["q"], s["k"], s["v"], s["cu"])
        leaves = [s[n].detach().requires_grad_(True) for n in "qkv"]
        y = A.attention(*leaves, s["cu"])
        return [y.detach(), *torch.autograd.grad(y, leaves, s["dy"])]
    if c["kind"] == "rotary":
        return A.rotary(s["q"], s["k"], s["pos"], s["freq"], interleaved=c["pairs"], magnitude=s["mag"], inverse=c["inverse"])
    if c["kind"] == "pages":
        if c["op"] == "copy":
            A.page_copy(s["slab"], s["moves"])
        else:
            A.page_append(s["k"], s["v"], s["slab"][:, -1, 0], s["slab"][:, -1, 1], s["rows"])
        return s["slab"]
    return A.tree_attention(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["cu"], parents=s["parents"],
                            max_context=s["longest"], max_new=s["most"])


def _padded(x, cu, most):
    """The rows of a packed batch as (sequences, heads, most, d) in 32 bits (rows past a sequence's end: any)."""
    at = (cu[:-1, None] + torch.arange(most, device=DEV)[None]).clamp(max=x.shape[0] - 1)
    return x.float()[at].permute(0, 2, 1, 3)


def _packed(x, cu, n):
    """(sequences, heads, most, d) back to (n, heads, d)."""
    t = torch.arange(n, device=DEV)
    b = torch.bucketize(t, cu[1:], right=True)
    return x[b, :, t - cu[b]]


def _plain_attention(s):
    c, cu, most = s["case"], s["cu"], s["longest"]
    n, H, d = s["q"].shape
    KV, G, B = c["KV"], H // c["KV"], cu.numel() - 1
    q = _padded(s["q"], cu, most).reshape(B, KV, G * most, d)
    k, v = _padded(s["k"], cu, most), _padded(s["v"], cu, most)
    t = torch.arange(most, device=DEV)
    lens = cu[1:] - cu[:-1]
    hidden = (t[None, :] > t[:, None])[None] | (t[None, None, :] >= lens[:, None, None]) | (t[None, :, None] >= lens[:, None, None])
    scale = d ** -0.5
    p = q @ k.transpose(-1, -2)
    p.mul_(scale)
    pv = p.view(B, KV, G, most, most)
    pv.masked_fill_(hidden[:, None, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    p.div_(p.sum(-1, keepdim=True).clamp(min=1e-30))
    o = p @ v
    y = _packed(o.reshape(B, H, most, d), cu, n).to(s["q"].dtype)
    if not c["train"]:
        return y
    inside = (t[None] < lens[:, None])[:, None, :, None]
    do = (_padded(s["dy"], cu, most) * inside).reshape(B, KV, G * most, d)
    dv = p.transpose(-1, -2) @ do
    ds = do @ v.transpose(-1, -2)
    ds.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = (ds @ k).reshape(B, H, most, d)
    dk = ds.transpose(-1, -2) @ q
    return [y, _packed(dq, cu, n).to(y.dtype), _packed(dk, cu, n).to(y.dtype), _packed(dv, cu, n).to(y.dtype)]


def _plain_rotary(s):
    c = s["case"]
    rot, half = c["rot"], c["rot"] // 2
    # a position's angle needs more than 24 bits before it is reduced; its sine and cosine do not
    angle = torch.remainder(s["pos"].double()[:, None] * s["freq"][None], 2 * math.pi).float()
    cos, sin = (torch.cos(angle) * s["mag"])[:, None], (torch.sin(angle) * s["mag"])[:, None]
    sin = -sin if c["inverse"] else sin

    def turned(x):
        z = x.float()
        a, b = (z[..., 0:rot:2], z[..., 1:rot:2]) if c["pairs"] else (z[..., :half], z[..., half:rot])
        u, w = a * cos - b * sin, b * cos + a * sin
        part = torch.stack([u, w], dim=-1).flatten(-2) if c["pairs"] else torch.cat([u, w], dim=-1)
        return torch.cat([part, z[..., rot:]], dim=-1).to(x.dtype)

    return [turned(s["q"]), turned(s["k"])]


def _plain_pages(s):
    c, slab = s["case"], s["slab"]
    if c["op"] == "copy":
        src, dst = s["moves"].to(DEV, torch.int64).unbind(1)
        slab[dst] = slab[src]
    else:
        page, off = s["rows"] // c["P"], s["rows"] % c["P"]
        slab[:, -1, 0][page, :, off] = s["k"]
        slab[:, -1, 1][page, :, off] = s["v"]
    return slab


def _plain_tree(s):
    c, cu, most = s["case"], s["cu"], s["most"]
    n, H, d = s["q"].shape
    KV, G, B = c["KV"], H // c["KV"], cu.numel() - 1

    def context(pages):
        return pages[s["table"].long()].permute(0, 2, 1, 3, 4).reshape(B, KV, -1, d).float()

    q = _padded(s["q"], cu, most).reshape(B, KV, G * most, d)
    k, v = _padded(s["k"], cu, most), _padded(s["v"], cu, most)
    kc, vc = context(s["k_pages"]), context(s["v_pages"])
    # token i sees its parent and what that sees: the reachable entries of (one step or none) many times over
    t = torch.arange(most, device=DEV)
    at = (cu[:-1, None] + t[None]).clamp(max=n - 1)
    inside = t[None] < (cu[1:] - cu[:-1])[:, None]
    up = ((s["parents"].long()[at][:, :, None] == t[None, None, :]) & inside[:, :, None]).float() + torch.eye(most, device=DEV)
    seen = torch.linalg.matrix_power(up, most) > 0
    past = torch.arange(kc.shape[2], device=DEV)[None] >= s["lens"][:, None]
    sc = (q @ kc.transpose(-1, -2)).mul_(d ** -0.5).masked_fill_(past[:, None, None], -math.inf)
    sn = (q @ k.transpose(-1, -2)).mul_(d ** -0.5).view(B, KV, G, most, most).masked_fill_(~seen[:, None, None], -math.inf)
    sn = sn.view(B, KV, G * most, most)
    top = torch.maximum(sc.amax(-1, keepdim=True), sn.amax(-1, keepdim=True))
    sc.sub_(top).exp_()
    sn.sub_(top).exp_()
    o = (sc @ vc + sn @ v) / (sc.sum(-1, keepdim=True) + sn.sum(-1, keepdim=True))
    return _packed(o.reshape(B, H, most, d), cu, n).to(s["q"].dtype)


# ------------------------------------------------------------------------------------------------- in 64 bits


def _softmax64(z, hide):
    z = z.masked_fill(hide, -math.inf)
    e = torch.exp(z - z.max(dim=1, keepdim=True).values)
    return e / e.sum(dim=1, keepdim=True)


def exact(case, seed):
    """What run() returns, one sequence and one head at a time in 64 bits."""
    s = prepare(case, seed)
    kind, d = case["kind"], case["d"]
    if kind == "pages":  # moves bits, computes nothing
        return None
    if kind == "rotary":
        rot = case["rot"]
        z = torch.polar(torch.full((), s["mag"], dtype=torch.float64, device=DEV), s["pos"].double()[:, None] * s["freq"])[:, None]
        z = z.conj() if case["inverse"] else z
        outs = []
        for x in (s["q"], s["k"]):
            w = x.double().clone()
            i = torch.arange(rot // 2, device=DEV)
            a, b = (2 * i, 2 * i + 1) if case["pairs"] else (i, i + rot // 2)
            r = torch.complex(w[..., a], w[..., b]) * z
            w[..., a], w[..., b] = r.real, r.imag
            outs.append(w)
        return outs
    G, cu, scale = case["H"] // case["KV"], s["cu"].tolist(), 1.0 / math.sqrt(d)
    q, k, v = (s[n].double() for n in "qkv")
    y = torch.zeros_like(q)
    if kind == "tree":
        table, lens, parents = s["table"].tolist(), s["lens"].tolist(), s["parents"].tolist()
        for b, (lo, hi) in enumerate(zip(cu, cu[1:])):
            own_pages = torch.tensor(table[b][:-(-lens[b] // case["P"])], device=DEV)
            hide = torch.ones(hi - lo, lens[b] + hi - lo, dtype=torch.bool)
            hide[:, :lens[b]] = False
            for i in range(hi - lo):
                j = i
                while j >= 0:
                    hide[i, lens[b] + j] = False
                    j = parents[lo + j]
            hide = hide.to(DEV)
            kc = s["k_pages"][own_pages].transpose(1, 2).reshape(-1, case["KV"], d)[:lens[b]].double()
            vc = s["v_pages"][own_pages].transpose(1, 2).reshape(-1, case["KV"], d)[:lens[b]].double()
            for h in range(case["H"]):
                kk, vv = torch.cat([kc[:, h // G], k[lo:hi, h // G]]), torch.cat([vc[:, h // G], v[lo:hi, h // G]])
                y[lo:hi, h] = _softmax64(q[lo:hi, h] @ kk.T * scale, hide) @ vv
        return y
    grads = [torch.zeros_like(x) for x in (q, k, v)]
    for lo, hi in zip(cu, cu[1:]):
        hide = torch.ones(hi - lo, hi - lo, dtype=torch.bool, device=DEV).triu(1)
        for h in range(case["H"]):
            e = h // G
            p = _softmax64(q[lo:hi, h] @ k[lo:hi, e].T * scale, hide)
            y[lo:hi, h] = p @ v[lo:hi, e]
            if case["train"]:
                dy = s["dy"][lo:hi, h].double()
                dp = dy @ v[lo:hi, e].T
                ds = p * (dp - (p * dp).sum(dim=1, keepdim=True)) * scale
                grads[0][lo:hi, h] = ds @ k[lo:hi, e]
                grads[1][lo:hi, e] += ds.T @ q[lo:hi, h]
                grads[2][lo:hi, e] += p.T @ dy
    return [y, *grads] if case["train"] else y
