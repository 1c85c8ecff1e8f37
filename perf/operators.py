"""Workloads of the operators that surround the gated delta rule in a serving stack.

The short causal convolution (packed prompts, and tokens over a pool of convolution states), the selective
state-space scan (packed prompts, and tokens over a pool of states) and the root-mean-square norm (with the
residual's addition, an output gate, and an 8-bit output with scales).

``run`` computes a case in its plain form (elementary torch operations in 32 bits) or, with ``own`` set, by the
framework's entry points; ``exact`` is the definition in 64 bits.
"""
import math
import os
import sys

import torch

own = False

PKG = "mlsys-flashlinfer-contest_b200"


def _gdn():
    path = os.path.join(os.getcwd(), PKG)
    if path not in sys.path:
        sys.path.insert(0, path)
    import gdn_b200
    return gdn_b200


# ---------------------------------------------------------------------------------------------------- cases

# Sequence lengths of a packed batch: "even" divides the tokens evenly, "ragged" draws the shares (some of
# them empty or one token long), "long" gives the first sequence half of the tokens.
def lengths(case):
    n, total = case["seqs"], case["tokens"]
    if case["spread"] == "even":
        return [total // n + (1 if i < total % n else 0) for i in range(n)]
    g = torch.Generator().manual_seed(1000 + 7 * n + total)
    share = torch.rand(n, generator=g, dtype=torch.float64) ** 2 + 0.02
    if n > 8:
        share[n // 2] = 0.0
    if case["spread"] == "long":
        share[0] = float(share[1:].sum()) if n > 1 else 1.0
    cum = (share.cumsum(0) / share.sum() * total).round().long().tolist()
    return [b - a for a, b in zip([0] + cum[:-1], cum)]


def listed():
    return [
        # q|k|v of a delta-rule layer (16 q/k heads, 32 v heads of 128) over a batch of mixed prompts that
        # continue from cached convolution states
        dict(name="conv_prompts_ragged", op="conv", tokens=7648, seqs=16, spread="ragged", parts="2048,2048,4096",
             width=4, bias=False, state=True, pad=0, dtype="bf16"),
        # x|B|C of a scan layer inside a wider projection (rows with a stride), four long prompts
        dict(name="conv_prompts_long", op="conv", tokens=32768, seqs=4, spread="even", parts="4096,1024,1024",
             width=4, bias=True, state=False, pad=4160, dtype="bf16"),
        # one user's next token: latency
        dict(name="conv_token_one", op="conv_pool", batch=1, tokens=1, parts="2048,2048,4096", width=4, bias=False,
             pad=0, dtype="bf16"),
        # a full decode batch verifying four drafted tokens each
        dict(name="conv_token_batch", op="conv_pool", batch=256, tokens=4, parts="2048,2048,4096", width=4, bias=True,
             pad=0, dtype="fp16"),
        # one prompt of a long document: few (sequence, head) pairs
        dict(name="scan_prompt_one", op="scan", tokens=8192, seqs=1, spread="even", heads=64, head=64, state_dim=128,
             groups=8, state=False, skip=True),
        # a batch of mixed prompts continuing from cached states, wide heads
        dict(name="scan_prompts_ragged", op="scan", tokens=7648, seqs=16, spread="ragged", heads=32, head=128,
             state_dim=128, groups=16, state=True, skip=True),
        # four prompts at full length
        dict(name="scan_prompts_long", op="scan", tokens=65536, seqs=4, spread="even", heads=64, head=64,
             state_dim=128, groups=8, state=True, skip=True),
        # one user's next token
        dict(name="scan_token_one", op="scan_pool", batch=1, tokens=1, heads=64, head=64, state_dim=128, groups=8,
             state_dtype="fp32"),
        # a full decode batch
        dict(name="scan_token_batch", op="scan_pool", batch=256, tokens=1, heads=64, head=64, state_dim=128, groups=8,
             state_dtype="fp32"),
        # the norm before a projection in 8 bits, small decode batch
        dict(name="norm_rows_few", op="norm", rows=8, dim=4096, residual=True, gate="", out="e4m3", group=0,
             dtype="bf16"),
        # the same for packed prompts, scales by 128 columns
        dict(name="norm_rows_many", op="norm", rows=16384, dim=4096, residual=True, gate="", out="e4m3", group=128,
             dtype="bf16"),
        # the gated norm of every head's output of a delta-rule layer (32 heads of 128), mixed prompts
        dict(name="norm_heads_gated", op="norm", rows=7648 * 32, dim=128, residual=False, gate="after", out="same",
             group=0, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["conv", "conv_pool", "scan", "scan", "scan_pool", "norm"])
    if op in ("conv", "conv_pool"):
        c = dict(op=op, parts=",".join(str(8 * _log(rng, 8, 512)) for _ in range(rng.choice([1, 2, 3]))),
                 width=rng.choice([2, 3, 4, 4]), bias=rng.random() < 0.5, pad=8 * rng.choice([0, 0, rng.randint(1, 400)]),
                 dtype=rng.choice(["bf16", "bf16", "fp16"]))
        if op == "conv":
            seqs = _log(rng, 1, 64)
            c.update(tokens=max(seqs, _log(rng, 16, 16384)), seqs=seqs, spread=rng.choice(["even", "ragged", "long"]),
                     state=rng.random() < 0.6)
        else:
            c.update(batch=_log(rng, 1, 256), tokens=rng.choice([1, 1, 2, 3, 5, 8]))
        return c
    if op in ("scan", "scan_pool"):
        groups = rng.choice([1, 2, 4, 8])
        c = dict(op=op, heads=groups * rng.choice([1, 2, 3, 4, 8]), head=rng.choice([64, 64, 128]),
                 state_dim=rng.choice([64, 128, 128]), groups=groups)
        if op == "scan":
            seqs = _log(rng, 1, 32)
            c.update(tokens=max(seqs, _log(rng, 16, 16384)), seqs=seqs, spread=rng.choice(["even", "ragged", "long"]),
                     state=rng.random() < 0.6, skip=rng.random() < 0.7)
        else:
            c.update(batch=_log(rng, 1, 128), tokens=rng.choice([1, 1, 1, 2, 3, 4]),
                     state_dtype=rng.choice(["fp32", "fp32", "bf16"]))
        return c
    gate = rng.choice(["", "", "after", "before"])
    group = rng.choice([0, 128])
    dim = 128 * _log(rng, 1, 64) if group or rng.random() < 0.5 else 8 * _log(rng, 4, 1000)
    return dict(op="norm", rows=_log(rng, 1, 16384 * 4096 // (2 * dim)), dim=dim, residual=not gate and rng.random() < 0.6,
                gate=gate, out=rng.choice(["same", "e4m3", "e4m3"]), group=group, dtype=rng.choice(["bf16", "bf16", "fp16"]))


def _types(case):
    return {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[case]


def _parts(case):
    return [int(p) for p in case["parts"].split(",")]


# ---------------------------------------------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    def uniform(n, lo, hi):
        return torch.rand(n, generator=g, device="cuda") * (hi - lo) + lo

    def slots(batch, pool):  # a batch's sequences lie anywhere in the pool
        return torch.randperm(pool, generator=g, device="cuda")[:batch].to(torch.int32)

    s = dict(case)
    op = case["op"]
    if op in ("conv", "conv_pool"):
        dt, parts = _types(case["dtype"]), _parts(case)
        dim, w = sum(parts), case["width"]
        s.update(parts=parts, weight=normal(dim, w, dtype=dt, scale=0.5),
                 bias=normal(dim, dtype=dt, scale=0.2) if case["bias"] else None)
        if op == "conv":
            lens = lengths(case)
            wide = normal(case["tokens"], dim + case["pad"], dtype=dt)
            s.update(x=wide[:, :dim], state=normal(len(lens), w - 1, dim, dtype=dt) if case["state"] else None,
                     cu=torch.tensor([0] + lens, device="cuda").cumsum(0))
        else:
            b, t = case["batch"], case["tokens"]
            wide = normal(b, t, dim + case["pad"], dtype=dt)
            s.update(x=wide[:, :, :dim], pool=normal(b + 3, w - 1, dim, dtype=dt), slots=slots(b, b + 3))
    elif op in ("scan", "scan_pool"):
        h, p, n, gr = case["heads"], case["head"], case["state_dim"], case["groups"]
        lead = (case["tokens"],) if op == "scan" else (case["batch"], case["tokens"])
        step = torch.exp(uniform(h, math.log(1e-3), math.log(0.1)))
        s.update(x=normal(*lead, h, p), B=normal(*lead, gr, n), C=normal(*lead, gr, n), a=normal(*lead, h, scale=0.7),
                 A_log=torch.log(uniform(h, 1.0, 16.0)), dt_bias=step + torch.log(-torch.expm1(-step)),
                 D=uniform(h, 0.5, 1.5) if case.get("skip", True) else None)
        if op == "scan":
            lens = lengths(case)
            s.update(state=normal(len(lens), h, p, n, dtype=torch.float32) if case["state"] else None,
                     cu=torch.tensor([0] + lens, device="cuda").cumsum(0))
        else:
            b = case["batch"]
            s.update(pool=normal(b + 3, h, p, n, dtype=_types(case["state_dtype"])), slots=slots(b, b + 3))
    else:
        dt, shape = _types(case["dtype"]), (case["rows"], case["dim"])
        s.update(x=normal(*shape, dtype=dt), weight=(1 + normal(case["dim"], dtype=torch.float32, scale=0.1)).to(dt),
                 residual=normal(*shape, dtype=dt, scale=3.0) if case["residual"] else None,
                 gate_in=normal(*shape, dtype=dt) if case["gate"] else None)
    return s


# ---------------------------------------------------------------------------------------------------- plain forms

def _silu(x):
    return x / (1 + torch.exp(-x))


def _softplus(x):
    return torch.where(x > 20, x, torch.log1p(torch.exp(x)))


def _conv_rows(src, index, s):
    """Rows of the convolution: index [rows, width] into src [positions, dim]."""
    acc = (src[index].float() * s["weight"].float().t()).sum(1)
    if s["bias"] is not None:
        acc = acc + s["bias"].float()
    return [p.contiguous() for p in _silu(acc).to(src.dtype).split(s["parts"], -1)]


def _conv(s):
    x, cu, w = s["x"], s["cu"], s["width"]
    total, dim = x.shape
    n = cu.numel() - 1
    old = s["state"] if s["state"] is not None else x.new_zeros(n, w - 1, dim)
    src = torch.cat([x, old.reshape(n * (w - 1), dim)])
    t = torch.arange(total, device=x.device)
    seq = torch.searchsorted(cu, t, right=True) - 1
    tap = torch.arange(w, device=x.device)

    def source(pos, q):  # a position before its sequence lies in that sequence's state
        return torch.where(pos >= cu[q], pos, total + q * (w - 1) + pos - cu[q] + w - 1)

    out = _conv_rows(src, source(t[:, None] - (w - 1) + tap, seq[:, None]), s)
    q = torch.arange(n, device=x.device)
    return out, src[source(cu[1:, None] - (w - 1) + tap[:-1], q[:, None])]


def _conv_pool(s):
    x, pool, w = s["x"], s["pool"], s["width"]
    b, t, dim = x.shape
    at = s["slots"].long()
    src = torch.cat([pool[at], x], 1)
    index = torch.arange(t, device=x.device)[:, None] + torch.arange(w, device=x.device)
    row = (torch.arange(b, device=x.device) * (t + w - 1))[:, None, None] + index
    out = _conv_rows(src.reshape(-1, dim), row.reshape(-1, w), s)
    pool[at] = src[:, t:]
    return [o.reshape(b, t, -1) for o in out], pool


def _scan(s, chunk=128):
    """Chunks of one sequence each: products within a chunk, and the chunks' states joined by one product with the
    decays between them."""
    x, cu = s["x"], s["cu"]
    total, h, p = x.shape
    n, gr = s["state_dim"], s["groups"]
    dev, seqs = x.device, cu.numel() - 1
    dt = _softplus(s["a"].float() + s["dt_bias"])
    l = -torch.exp(s["A_log"]).double() * dt.double()
    # the chunks: sequence, first token, and the tokens of each (all of them one past the last where a chunk is short)
    count = (cu[1:] - cu[:-1] + chunk - 1) // chunk
    ends = count.cumsum(0)
    c = torch.arange(total // chunk + seqs, device=dev)
    seq = torch.searchsorted(ends, c, right=True).clamp(max=seqs - 1)
    within = c - (ends - count)[seq]
    tok = (cu[seq] + within * chunk)[:, None] + torch.arange(chunk, device=dev)
    live = (tok < cu[seq + 1][:, None]) & (c < ends[-1])[:, None]
    tok = torch.where(live, tok, total)

    def take(v):
        return torch.cat([v, v.new_zeros(1, *v.shape[1:])])[tok]

    xc, bc, cc, dc = take(x).float(), take(s["B"]).float(), take(s["C"]).float(), take(dt)
    gam = take(l).cumsum(1)                                                       # [c, q, h], 64 bits
    rel = (gam[:, :, None] - gam[:, None]).float()                                # [c, i, j, h]
    tri = torch.ones(chunk, chunk, dtype=torch.bool, device=dev).tril()[None, :, :, None]
    dec = torch.where(tri, torch.exp(torch.where(tri, rel, 0.0)), 0.0)
    cb = torch.einsum("cign,cjgn->cijg", cc, bc).repeat_interleave(h // gr, -1)
    y = torch.einsum("cijh,cjhp->cihp", cb * dec * dc[:, None], xc)
    last = gam[:, -1:]                                                            # [c, 1, h]
    wx = xc * (torch.exp((last - gam).float()) * dc)[..., None]
    add = torch.einsum("cjgep,cjgn->cgepn", wx.reshape(*wx.shape[:2], gr, h // gr, p), bc).reshape(-1, h, p, n)
    # states at the chunks' starts
    upto = last[:, 0].cumsum(0)                                                   # [c, h], through chunk c
    before = upto - last[:, 0]
    first = (ends - count)[seq]
    joined = (seq[:, None] == seq) & (c[None] < c[:, None])
    between = (before[:, None] - upto[None]).float()
    between = torch.where(joined[..., None], torch.exp(torch.where(joined[..., None], between, 0.0)), 0.0)
    start = torch.einsum("cdh,dhe->che", between, add.reshape(len(c), h, p * n)).reshape(len(c), h, p, n)
    old = s["state"] if s["state"] is not None else torch.zeros(seqs, h, p, n, device=dev)
    live_c = (c < ends[-1])[:, None]
    lead = torch.exp(torch.where(live_c, before - before[first.clamp(max=len(c) - 1)], 0.0)).float()
    start = start + old[seq] * lead[..., None, None]
    ys = torch.einsum("cign,cgepn->cigep", cc, start.reshape(-1, gr, h // gr, p, n)).reshape(y.shape)
    y = y + ys * torch.exp(gam.float())[..., None]
    if s["D"] is not None:
        y = y + xc * s["D"][:, None]
    out = x.new_empty(total + 1, h, p)
    out[tok] = y.to(x.dtype)
    end = start * torch.exp(last[:, 0].float())[..., None, None] + add
    final = torch.where((count > 0)[:, None, None, None], end[(ends - 1).clamp(min=0)], old)
    return out[:total], final


def _scan_pool(s):
    """The tokens of a sequence by products with the decays between them; the state by one more."""
    x, pool = s["x"], s["pool"]
    b, t, h, p = x.shape
    gr = s["groups"]
    at = s["slots"].long()
    old = pool[at].float()
    xf = x.float()
    bh, ch = (s[k].float().repeat_interleave(h // gr, 2) for k in ("B", "C"))
    dt = _softplus(s["a"].float() + s["dt_bias"])
    gam = (-torch.exp(s["A_log"]) * dt).cumsum(1)                                 # [b, t, h]
    tri = torch.ones(t, t, dtype=torch.bool, device=x.device).tril()[:, :, None]
    rel = gam[:, :, None] - gam[:, None]
    m = torch.where(tri, torch.exp(torch.where(tri, rel, 0.0)), 0.0) * dt[:, None]
    y = torch.einsum("bijh,bihn,bjhn,bjhp->bihp", m, ch, bh, xf) if t > 1 else \
        xf * ((ch * bh).sum(-1) * dt)[..., None]
    y = y + (old[:, None] * ch[:, :, :, None]).sum(-1) * torch.exp(gam)[..., None]
    if s["D"] is not None:
        y = y + xf * s["D"][:, None]
    w = xf * (torch.exp(gam[:, -1:] - gam) * dt)[..., None]
    new = old * torch.exp(gam[:, -1])[..., None, None] + (w[..., None] * bh[:, :, :, None]).sum(1)
    pool[at] = new.to(pool.dtype)
    return y.to(x.dtype), pool


def _norm(s):
    x, dt = s["x"].float(), s["x"].dtype
    new = None
    if s["residual"] is not None:
        x = x + s["residual"].float()
        new = x.to(dt)
    if s["gate"] == "before":
        x = x * _silu(s["gate_in"].float())
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * s["weight"].float()
    if s["gate"] == "after":
        y = y * _silu(s["gate_in"].float())
    if s["out"] == "same":
        return [y.to(dt), new]
    rows, dim = y.shape
    blocks = y.reshape(rows, dim // s["group"] if s["group"] else 1, -1)
    amax = blocks.abs().amax(-1)
    scale = torch.where(amax == 0, 1.0, amax / 448)
    q = (blocks / scale[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).reshape(rows, dim)
    return [q, scale if s["group"] else scale[:, 0], new]


def run(s):
    op = s["op"]
    if own:
        f = _gdn()
        if op == "conv":
            out, new = f.conv.run(s["x"], s["weight"], s["bias"], s["state"], s["cu"], splits=s["parts"])
            return list(out), new
        if op == "conv_pool":
            out = f.conv.run_pool(s["x"], s["weight"], s["bias"], s["pool"], s["slots"], splits=s["parts"])
            return list(out), s["pool"]
        if op == "scan":
            return f.ssm.run(s["x"], s["B"], s["C"], s["state"], s["A_log"], s["a"], s["dt_bias"], s["D"], s["cu"])
        if op == "scan_pool":
            y = f.ssm.run_pool(s["x"], s["B"], s["C"], s["A_log"], s["a"], s["dt_bias"], s["D"], s["pool"], s["slots"])
            return y, s["pool"]
        kw = dict(residual=s["residual"], gate=s["gate_in"], gate_first=s["gate"] == "before")
        if s["out"] == "same":
            out = f.norm.run(s["x"], s["weight"], 1e-6, **kw)
            return list(out) if s["residual"] is not None else [out, None]
        out = f.norm.run_fp8(s["x"], s["weight"], 1e-6, group_size=s["group"], **kw)
        return list(out) if s["residual"] is not None else [*out, None]
    return {"conv": _conv, "conv_pool": _conv_pool, "scan": _scan, "scan_pool": _scan_pool, "norm": _norm}[op](s)


# ---------------------------------------------------------------------------------------------------- work

def work(case):
    op = case["op"]
    if op in ("conv", "conv_pool"):
        dim, w = sum(_parts(case)), case["width"]
        rows = case["tokens"] * (case["batch"] if op == "conv_pool" else 1)
        states = 2 * case["batch"] if op == "conv_pool" else case["seqs"] * (2 if case["state"] else 1)
        return {"bytes": 2 * dim * (2 * rows + (w - 1) * states + w), "flops": rows * dim * (2 * w + 4)}
    if op in ("scan", "scan_pool"):
        h, p, n, gr = case["heads"], case["head"], case["state_dim"], case["groups"]
        rows = case["tokens"] * (case["batch"] if op == "scan_pool" else 1)
        if op == "scan":
            states = 4 * case["seqs"] * (2 if case["state"] else 1)
        else:
            states = 2 * case["batch"] * (2 if case["state_dtype"] == "bf16" else 4)
        return {"bytes": rows * (4 * h * p + 4 * gr * n + 2 * h) + states * h * p * n, "flops": rows * h * p * (5 * n + 2)}
    size = case["rows"] * case["dim"]
    out = 2 * size if case["out"] == "same" else size + 4 * case["rows"] * (case["dim"] // case["group"] if case["group"] else 1)
    return {"bytes": 2 * size + out + (4 * size if case["residual"] else 0) + (2 * size if case["gate"] else 0) + 2 * case["dim"],
            "flops": 6 * size}


# ---------------------------------------------------------------------------------------------------- 64 bits

def _sigmoid64(v):
    return torch.sigmoid(v.double())


def _conv_one64(s, before, rows):
    """One sequence: rows [t, dim] after the width - 1 rows `before`."""
    full = torch.cat([before.double(), rows.double()])
    t, w = rows.shape[0], s["width"]
    out = sum(full[j:j + t] * s["weight"][:, j].double() for j in range(w))
    if s["bias"] is not None:
        out = out + s["bias"].double()
    return out * _sigmoid64(out), full[t:]


def _scan64(x, B, C, a, s, S):
    """Token by token over a batch of sequences: x [b, t, h, p] -> y, and the states after each sequence's tokens
    (a of -inf beyond a sequence's end leaves its state)."""
    h, gr = x.shape[2], B.shape[2]
    ys = []
    A = -torch.exp(s["A_log"].double())
    z = a.double() + s["dt_bias"].double()
    dt = torch.clamp(z, min=0) + torch.log1p(torch.exp(-z.abs()))
    for t in range(x.shape[1]):
        d = dt[:, t]
        xt = x[:, t].double()
        S.mul_(torch.exp(A * d)[..., None, None])
        S.view(S.shape[0], gr, h // gr, *S.shape[2:]).addcmul_(
            (d[..., None] * xt).view(S.shape[0], gr, h // gr, -1, 1), B[:, t].double()[:, :, None, None])
        y = torch.matmul(S.view(S.shape[0], gr, -1, S.shape[3]), C[:, t].double()[..., None]).view(xt.shape)
        ys.append(y + xt * s["D"].double()[:, None] if s["D"] is not None else y)
    return torch.stack(ys, 1), S


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "conv":
        cu = s["cu"].tolist()
        outs, news = [], []
        for i, (b, e) in enumerate(zip(cu, cu[1:])):
            before = s["state"][i] if s["state"] is not None else s["x"].new_zeros(s["width"] - 1, s["x"].shape[1])
            o, nw = _conv_one64(s, before, s["x"][b:e])
            outs.append(o)
            news.append(nw)
        return list(torch.cat(outs).split(s["parts"], -1)), torch.stack(news)
    if op == "conv_pool":
        outs, pool = [], s["pool"].double()
        for i, at in enumerate(s["slots"].tolist()):
            o, nw = _conv_one64(s, s["pool"][at], s["x"][i])
            outs.append(o)
            pool[at] = nw
        return list(torch.stack(outs).split(s["parts"], -1)), pool
    if op == "scan_pool":
        at = s["slots"].long()
        y, S = _scan64(s["x"], s["B"], s["C"], s["a"], s, s["pool"][at].double())
        pool = s["pool"].double()
        pool[at] = S
        return y, pool
    if op == "scan":
        lens = lengths(case)
        longest = max(lens)
        if longest * len(lens) * case["heads"] * case["head"] * case["state_dim"] > 6e11 or longest > 40000:
            return None
        tok = torch.arange(longest, device="cuda") + s["cu"][:-1, None]
        live = tok < s["cu"][1:, None]
        tok = torch.where(live, tok, 0)
        a = torch.where(live[..., None], s["a"][tok].double(), -math.inf)
        S = torch.zeros(len(lens), case["heads"], case["head"], case["state_dim"], dtype=torch.float64, device="cuda")
        if s["state"] is not None:
            S += s["state"]
        y, S = _scan64(s["x"][tok], s["B"][tok], s["C"][tok], a, s, S)
        return y[live], S
    x = s["x"].double()
    new = None
    if s["residual"] is not None:
        x = new = x + s["residual"].double()
    if s["gate"] == "before":
        x = x * s["gate_in"].double() * _sigmoid64(s["gate_in"])
    y = x * torch.rsqrt(x.square().mean(1, True) + 1e-6) * s["weight"].double()
    if s["gate"] == "after":
        y = y * s["gate_in"].double() * _sigmoid64(s["gate_in"])
    if s["out"] == "same":
        return [y, new]
    scale = y.unflatten(1, (-1, s["group"] or case["dim"])).abs().amax(2) / 448
    scale[scale == 0] = 1
    q = (y.unflatten(1, (scale.shape[1], -1)) / scale[..., None]).flatten(1)
    return [q, scale if s["group"] else scale[:, 0], new]
