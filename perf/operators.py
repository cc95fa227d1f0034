"""The sequence operators over feature rows -- the gated recurrence and its single-step form, the
running normalisation, the dropout whose mask is never stored -- as measured cases, each with the
same operation in elementary torch products, sums and comparisons."""
import math
import random

import numpy as np
import torch

own = False  # True: run() calls mfcc_amd, False: the plain forms below

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
DEV = "cuda"


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
def listed():
    return [
        # serving: one frame of 64 live streams through one recurrent layer; latency is all there is
        dict(name="step 64x512 f32", op="step", n=64, d=512, dtype="f32", form="sigmoid"),
        # a batch of utterances of ordinary lengths scored by one layer, the state carried in
        dict(name="scan 32x512 bf16", op="scan", train=False, n=32, lo=97, hi=700, d=512, dtype="bf16", form="sigmoid",
             padded=False, reverse=False, h0=True),
        # a training step's share of one layer: a large batch, forward and backward
        dict(name="scan train 64x1024 bf16", op="scan", train=True, n=64, lo=100, hi=1500, d=1024, dtype="bf16", form="sigmoid",
             padded=False, reverse=False, h0=True),
        # the backward-running half of a bidirectional layer on a padded batch of 257-bin spectrum rows
        dict(name="scan train pad rev 32x257 f32", op="scan", train=True, n=32, lo=0, hi=700, d=257, dtype="f32", form="decay",
             padded=True, reverse=True, h0=False),
        # one hour of 10 ms frames through one layer
        dict(name="scan 1h 1x256 f16", op="scan", train=False, n=1, lo=360000, hi=360000, d=256, dtype="f16", form="sigmoid",
             padded=False, reverse=False, h0=False),
        # training on two long recordings
        dict(name="scan train long 2x384 bf16", op="scan", train=True, n=2, lo=47001, hi=60000, d=384, dtype="bf16", form="decay",
             padded=False, reverse=False, h0=True),
        # one 10 ms hop of 64 live streams, normalised from a carried state
        dict(name="norm hop 64x39", op="norm", n=64, lo=1, hi=1, d=39, out="f32", decay=0.995, state=True),
        # ten thousand utterances of 3 s
        dict(name="norm 10000x3s 39", op="norm", n=10000, lo=299, hi=299, d=39, out="f32", decay=0.995, state=False),
        # one hour in one piece, cumulative statistics
        dict(name="norm 1h 39", op="norm", n=1, lo=360000, hi=360000, d=39, out="f32", decay=1.0, state=True),
        # spectrum rows of a ragged batch for a model that computes in bfloat16
        dict(name="norm 200x257 to bf16", op="norm", n=200, lo=1, hi=1200, d=257, out="bf16", decay=0.99, state=False),
        # a CTC batch whose coefficients are dropped for whole utterances, the mask of a recurrent model
        dict(name="dropout seq 64x39 f32", op="dropout", train=False, n=64, lo=50, hi=700, d=39, dtype="f32", p=0.2, per="sequence"),
        # stacked 17 x 257 windows on their way into a dense model, forward and backward
        dict(name="dropout train 20000x4369 bf16", op="dropout", train=True, n=1, lo=20000, hi=20000, d=4369, dtype="bf16", p=0.3,
             per="element"),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(["step", "scan", "scan", "scan", "norm", "norm", "dropout"])
    if op == "step":
        return dict(op=op, n=_log(rng, 1, 512), d=rng.choice([_log(rng, 16, 2048), 39, 256, 512]), dtype=rng.choice(list(DTYPES)),
                    form=rng.choice(["decay", "sigmoid"]))
    if op == "dropout":
        d = rng.choice([39, 257, 429, 4369, _log(rng, 8, 2048)])
        hi = max(1, min(_log(rng, 10, 2000), 40000000 // (d * 40)))
        return dict(op=op, train=rng.random() < 0.5, n=rng.randint(1, 40), lo=rng.randint(0, hi), hi=hi, d=d, dtype=rng.choice(list(DTYPES)),
                    p=rng.choice([0.05, 0.1, 0.25, 0.5, 0.75]), per=rng.choice(["element", "sequence", "frame"]))
    if op == "norm":
        d = rng.choice([13, 39, 257, _log(rng, 4, 600)])
        n, hi = rng.choice([(_log(rng, 1, 256), 1), (_log(rng, 2, 4000), 0), (rng.randint(1, 4), 0)])
        if hi == 0:
            hi = max(2, min(_log(rng, 20, 2000) if n > 4 else _log(rng, 2000, 300000), 50000000 // (n * d)))
        return dict(op=op, n=n, lo=rng.randint(1, hi), hi=hi, d=d, out=rng.choice(list(DTYPES)), decay=rng.choice([0.9, 0.99, 0.995, 0.999, 1.0]),
                    state=rng.random() < 0.5)
    train = rng.random() < 0.6
    d = rng.choice([39, 257, 512, 1024, _log(rng, 8, 1500)])
    n = rng.choice([_log(rng, 4, 256), rng.randint(1, 3)])
    hi = _log(rng, 30, 1500) if n > 3 else _log(rng, 1000, 100000)
    hi = max(2, min(hi, 24000000 // (n * d)))
    return dict(op="scan", train=train, n=n, lo=rng.randint(0, hi), hi=hi, d=d, dtype=rng.choice(list(DTYPES)),
                form=rng.choice(["decay", "sigmoid"]), padded=rng.random() < 0.3, reverse=rng.random() < 0.4, h0=rng.random() < 0.5)


def lengths_of(case):
    """Frames of every sequence: uniform between lo and hi, the first one hi."""
    rng = random.Random(case["n"] * 1000003 + case["lo"] * 1009 + case["hi"])
    return [case["hi"]] + [rng.randint(case["lo"], case["hi"]) for _ in range(case["n"] - 1)]


def work(case):
    d = case["d"]
    if case["op"] == "step":
        e = DTYPES[case["dtype"]].itemsize
        v = case["n"] * d
        return {"bytes": v * (3 * e + 8), "flops": v * (3 if case["form"] == "decay" else 10)}
    v = sum(lengths_of(case)) * d
    if case["op"] == "norm":
        ends = case["n"] * (1 + 2 * d) * 4
        return {"bytes": v * (4 + DTYPES[case["out"]].itemsize) + ends * (2 if case["state"] else 1), "flops": 15 * v}
    e = DTYPES[case["dtype"]].itemsize
    if case["op"] == "dropout":
        return {"bytes": v * e * (4 if case["train"] else 2), "flops": v * (2 if case["train"] else 1)}
    written = (case["n"] * case["hi"] * d if case["padded"] else v) * e  # the rows behind a padded sequence are zeroed
    ends = case["n"] * d * 4
    fwd = 2 * v * e + written + ends * (2 if case["h0"] else 1)
    bwd = 3 * v * e + 2 * written + ends * (2 if case["h0"] else 1)
    flops = v * (3 if case["form"] == "decay" else 10)
    return {"bytes": fwd + (bwd if case["train"] else 0), "flops": flops * (3 if case["train"] else 1)}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    d, n = case["d"], case["n"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEV)

    s = dict(case=case)
    if case["op"] == "step":
        dt = DTYPES[case["dtype"]]
        g = normal(n, d) * 1.5 + 3
        s.update(x=normal(n, d).to(dt), gate=(g if case["form"] == "sigmoid" else torch.sigmoid(g)).to(dt), h=normal(n, d),
                 h_out=torch.empty(n, d, device=DEV))
        return s
    lens = lengths_of(case)
    rows = sum(lens)
    s["lens"] = lens
    if own:
        import mfcc_amd
        s["layout"] = mfcc_amd.Layout.from_frame_counts(torch.device("cuda", torch.cuda.current_device()), lens)
    else:
        s["index"] = _index(lens, case)
    if case["op"] == "norm":
        # feature columns: each its own level and spread
        s["x"] = normal(rows, d) * (0.5 + 3 * torch.rand(d, generator=gen, device=DEV)) + 6 * normal(d)
        if case["state"]:
            w = 20 + 100 * torch.rand(n, 1, generator=gen, device=DEV)
            s["state"] = torch.cat([w, 6 * normal(n, d), w * (0.5 + 4 * torch.rand(n, d, generator=gen, device=DEV))], 1)
        return s
    dt = DTYPES[case["dtype"]]
    if case["op"] == "dropout":
        s.update(x=normal(rows, d).to(dt), seed=int(torch.randint(1 << 62, (1,), generator=torch.Generator().manual_seed(seed)).item()),
                 step=1000 + seed % 1000)
        if case["train"]:
            s["gy"] = normal(rows, d).to(dt)
            s["x"].requires_grad_(True)
        return s
    shape = (n, case["hi"], d) if case["padded"] else (rows, d)
    g = normal(*shape) * 1.5 + 3  # a memory of some tens of frames
    s.update(x=normal(*shape).to(dt), gate=(g if case["form"] == "sigmoid" else torch.sigmoid(g)).to(dt))
    s["h0"] = normal(n, d) if case["h0"] else None
    if case["train"]:
        s.update(gy=normal(*shape).to(dt), glast=normal(n, d))
        for k in ("x", "gate", "h0"):
            if s[k] is not None:
                s[k].requires_grad_(True)
    return s


# --------------------------------------------------------------------------
# the framework's calls
# --------------------------------------------------------------------------
def _run_own(s):
    import mfcc_amd
    case = s["case"]
    if case["op"] == "step":
        return mfcc_amd.gated_scan_step(s["x"], s["gate"], s["h"], form=case["form"], state_out=s["h_out"])
    if case["op"] == "norm":
        return mfcc_amd.running_norm(s["x"], s["layout"], decay=case["decay"], state=s.get("state"), dtype=DTYPES[case["out"]])
    if case["op"] == "dropout":
        y = mfcc_amd.feature_dropout(s["x"], case["p"], s["seed"], step=s["step"], per=case["per"], frame_counts=s["layout"])
        return (y.detach(), *torch.autograd.grad(y, s["x"], s["gy"])) if case["train"] else y
    y, last = mfcc_amd.gated_scan(s["x"], s["gate"], s["layout"], h0=s["h0"], form=case["form"], reverse=case["reverse"])
    if not case["train"]:
        return y, last
    leaves = [s[k] for k in ("x", "gate", "h0") if s[k] is not None]
    return (y.detach(), last.detach(), *torch.autograd.grad((y, last), leaves, (s["gy"], s["glast"])))


# --------------------------------------------------------------------------
# the plain forms
# --------------------------------------------------------------------------
def _index(lens, case):
    """Index tensors of a ragged batch: the rows of every sequence in the order in which the recurrence visits them."""
    n = torch.tensor(lens, device=DEV)
    end = torch.cumsum(n, 0)
    seq = torch.repeat_interleave(torch.arange(len(lens), device=DEV), n)
    t = torch.arange(int(end[-1]), device=DEV) - (end - n)[seq]
    src = seq * case["hi"] + t if case.get("padded") else (end - n)[seq] + t
    if case.get("reverse"):
        back = (end - n)[seq] + n[seq] - 1 - t
        src = src[back]
    return dict(n=n, end=end, seq=seq, t=t, src=src, first=(t == 0), longest=max(lens))


def _scan(a, b, longest):
    """h_t = a_t h_{t-1} + b_t along the rows by doubling: log2(longest) sweeps; a is 0 where a sequence begins."""
    k = 1
    while k < longest:
        b = torch.cat([b[:k], b[k:] + a[k:] * b[:-k]])
        a = torch.cat([a[:k], a[k:] * a[:-k]])
        k *= 2
    return b


def _plain_scan(s):
    case, ix = s["case"], s["index"]
    d, dt = case["d"], DTYPES[case["dtype"]]
    shape = s["x"].shape
    x = s["x"].detach().reshape(-1, d)[ix["src"]].float()
    g = s["gate"].detach().reshape(-1, d)[ix["src"]].float()
    if case["form"] == "sigmoid":
        a, na = 1 / (1 + torch.exp(-g)), 1 / (1 + torch.exp(g))
        b = na * x
    else:
        a, b = g, x
    h0 = s["h0"].detach() if s["h0"] is not None else torch.zeros(case["n"], d, device=DEV)
    some = ix["n"] > 0
    first, final = (ix["end"] - ix["n"])[some], ix["end"][some] - 1
    b = b.clone()
    b[first] += a[first] * h0[some]
    a0 = a.clone()
    a0[first] = 0
    h = _scan(a0, b, ix["longest"])
    last = h0.clone()
    last[some] = h[final]

    def back(v):
        out = torch.zeros(math.prod(shape[:-1]), d, dtype=dt, device=DEV)
        out[ix["src"]] = v.to(dt)
        return out.reshape(shape)

    y = back(h)
    if not case["train"]:
        return y, last
    gy = s["gy"].reshape(-1, d)[ix["src"]].float()
    gy[final] += s["glast"][some]
    link = torch.cat([a[1:], a[:1]])
    link[final] = 0
    delta = _scan(link.flip(0), gy.flip(0), ix["longest"]).flip(0)
    hp = torch.cat([h[:1], h[:-1]])
    hp[first] = h0[some]
    if case["form"] == "sigmoid":
        dx, dg = na * delta, delta * a * na * (hp - x)
    else:
        dx, dg = delta, delta * hp
    grads = [back(dx), back(dg)]
    if s["h0"] is not None:
        dh0 = s["glast"].clone()
        dh0[some] = a[first] * delta[first]
        grads.append(dh0)
    return (y, last, *grads)


def _plain_norm(s, eps=1e-5):
    # in 64 bits: a weight of 1e5 rows leaves 1 - 1 / W too few digits in 32
    case, ix = s["case"], s["index"]
    d, lam, n = case["d"], case["decay"], case["n"]
    x = s["x"].double()
    st = s["state"].double() if case["state"] else torch.zeros(n, 1 + 2 * d, dtype=torch.float64, device=DEV)
    w0, m0, s0 = st[:, :1], st[:, 1:1 + d], st[:, 1 + d:]
    k = (ix["t"] + 1).double().unsqueeze(1)
    grown = k if lam == 1.0 else (1 - lam ** k) / (1 - lam)
    w = (lam ** k) * w0[ix["seq"]] + grown
    some = ix["n"] > 0
    first, final = (ix["end"] - ix["n"])[some], ix["end"][some] - 1
    a, b = (1 - 1 / w).expand(-1, d).clone(), x / w
    b[first] += a[first] * m0[some]
    a[first] = 0
    m = _scan(a, b, ix["longest"])
    mp = torch.cat([m[:1], m[:-1]])
    mp[first] = m0[some]
    b = (x - mp) * (x - m)
    b[first] += lam * s0[some]
    a = torch.full_like(b, lam)
    a[first] = 0
    sq = _scan(a, b, ix["longest"])
    y = (x - m) / torch.sqrt(sq / w + eps)
    out = st.clone()
    out[some] = torch.cat([w[final], m[final], sq[final]], 1)
    return y.to(DTYPES[case["out"]]), out.float()


def _philox(q, step, seed):
    """Philox4x32-10 blocks of the counters (q, step) under the key seed: int64 tensor [len(q), 4] of 32-bit words."""
    low = 0xFFFFFFFF
    c = [q & low, q >> 32, torch.full_like(q, step & low), torch.full_like(q, step >> 32)]
    k0, k1 = seed & low, seed >> 32

    def wide(m, v):  # high and low word of m * v
        lo, hi = m * (v & 0xFFFF), m * (v >> 16)
        return (hi + (lo >> 16)) >> 16, (((hi & 0xFFFF) << 16) + lo) & low

    for _ in range(10):
        h0, l0 = wide(0xD2511F53, c[0])
        h1, l1 = wide(0xCD9E8D57, c[2])
        c = [h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack(c, 1)


def _fields(count, step, seed):
    """The first `count` 16-bit fields of the stream."""
    words = _philox(torch.arange((count + 7) // 8, device=DEV), step, seed)
    return torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:count]


def _plain_dropout(s):
    case, ix = s["case"], s["index"]
    rows, d = s["x"].shape
    thr = int(round(case["p"] * 65536))
    if case["per"] == "element":
        keep = (_fields(rows * d, s["step"], s["seed"]) >= thr).reshape(rows, d)
    elif case["per"] == "frame":
        keep = (_fields(rows, s["step"], s["seed"]) >= thr).unsqueeze(1)
    else:
        wide = (d + 7) // 8 * 8
        keep = (_fields(case["n"] * wide, s["step"], s["seed"]) >= thr).reshape(case["n"], wide)[:, :d][ix["seq"]]
    scale = 65536 / (65536 - thr)

    def apply(v):
        return torch.where(keep, v.float() * scale, 0.0).to(v.dtype)

    y = apply(s["x"].detach())
    return (y, apply(s["gy"])) if case["train"] else y


def _plain_step(s):
    x, g, h = s["x"].float(), s["gate"].float(), s["h"]
    if s["case"]["form"] == "sigmoid":
        h = h / (1 + torch.exp(-g)) + x / (1 + torch.exp(g))
    else:
        h = g * h + x
    return h.to(s["x"].dtype), h


def run(state):
    if own:
        return _run_own(state)
    return {"step": _plain_step, "scan": _plain_scan, "norm": _plain_norm, "dropout": _plain_dropout}[state["case"]["op"]](state)


# --------------------------------------------------------------------------
# the definitions, frame by frame in 64 bits on the host
# --------------------------------------------------------------------------
def _host(t):
    return None if t is None else t.detach().double().cpu().numpy()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "step":
        h = _exact_cell(_host(s["x"]), _host(s["gate"]), _host(s["h"]), case["form"])[0]
        return h, h
    if case["op"] == "scan":
        return _exact_scan(case, s)
    if case["op"] == "norm":
        return _exact_norm(case, s)
    return _exact_dropout(case, s)


def _exact_cell(x, g, h, form):
    if form == "decay":
        return g * h + x, g, 1.0
    a, na = 1 / (1 + np.exp(-g)), 1 / (1 + np.exp(g))
    return a * h + na * x, a, na


def _exact_scan(case, s):
    lens, d, form = s["lens"], case["d"], case["form"]
    n, top = case["n"], max(lens)
    # sequences in order of falling length, so that those still running at frame t are the first few
    order = sorted(range(n), key=lambda u: -lens[u])
    running = [sum(1 for v in lens if v > t) for t in range(top)]
    if n == 1:
        running = [1] * top
    start = np.concatenate([[0], np.cumsum(lens)])[:n] if not case["padded"] else np.arange(n) * case["hi"]

    def row(u, t):
        return start[u] + (lens[u] - 1 - t if case["reverse"] else t)

    at = [np.array([row(u, t) for u in order[:running[t]]]) for t in range(top)]
    flat = {k: _host(s[k]).reshape(-1, d) for k in ("x", "gate") + (("gy",) if case["train"] else ())}
    h = np.zeros((n, d)) if s["h0"] is None else _host(s["h0"])[order]
    y = np.zeros_like(flat["x"])
    before = np.zeros_like(y) if case["train"] else None
    for t in range(top):
        r, i = running[t], at[t]
        if before is not None:
            before[i] = h[:r]
        h[:r] = _exact_cell(flat["x"][i], flat["gate"][i], h[:r], form)[0]
        y[i] = h[:r]
    last = np.zeros_like(h)
    last[order] = h
    shape = tuple(s["x"].shape)
    if not case["train"]:
        return y.reshape(shape), last
    eps = _host(s["glast"])[order]  # a_{t+1} delta_{t+1}
    dx, dg = np.zeros_like(y), np.zeros_like(y)
    for t in reversed(range(top)):
        r, i = running[t], at[t]
        _, a, na = _exact_cell(flat["x"][i], flat["gate"][i], before[i], form)
        delta = flat["gy"][i] + eps[:r]
        dx[i] = delta * na
        dg[i] = delta * before[i] if form == "decay" else delta * a * na * (before[i] - flat["x"][i])
        eps[:r] = a * delta
    out = [y.reshape(shape), last, dx.reshape(shape), dg.reshape(shape)]
    if s["h0"] is not None:
        dh0 = np.zeros_like(eps)
        dh0[order] = eps
        out.append(dh0)
    return tuple(out)


def _exact_norm(case, s, eps=1e-5):
    lens, d, n, lam = s["lens"], case["d"], case["n"], case["decay"]
    x, y = _host(s["x"]), np.zeros((sum(lens), d))
    st = _host(s["state"]) if case["state"] else np.zeros((n, 1 + 2 * d))
    order = sorted(range(n), key=lambda u: -lens[u])
    start = np.concatenate([[0], np.cumsum(lens)])[:n][order]
    falling = np.array(lens)[order]
    w, m, q = st[order, :1], st[order, 1:1 + d], st[order, 1 + d:]
    for t in range(int(falling[0])):
        r = 1 if n == 1 else int(np.searchsorted(-falling, -t, side="left"))
        v = x[start[:r] + t]
        w[:r] = lam * w[:r] + 1
        off = v - m[:r]
        m[:r] += off / w[:r]
        q[:r] = lam * q[:r] + off * (v - m[:r])
        y[start[:r] + t] = (v - m[:r]) / np.sqrt(q[:r] / w[:r] + eps)
    out = np.zeros_like(st)
    out[order] = np.concatenate([w, m, q], 1)
    return y, out


def _exact_dropout(case, s):
    x, d = _host(s["x"]), case["d"]
    rows = x.shape[0]
    if case["per"] == "element":
        e = np.arange(rows * d, dtype=np.uint64).reshape(rows, d)
    elif case["per"] == "frame":
        e = np.broadcast_to(np.arange(rows, dtype=np.uint64)[:, None], (rows, d))
    else:
        u = np.repeat(np.arange(case["n"], dtype=np.uint64), s["lens"])
        e = u[:, None] * np.uint64(-(-d // 8) * 8) + np.arange(d, dtype=np.uint64)
    word = np.uint64(0xFFFFFFFF)
    shift = np.uint64(32)
    blocks = np.arange(int(e.max(initial=0)) // 8 + 1, dtype=np.uint64)
    c = [blocks & word, blocks >> shift, np.full_like(blocks, s["step"] % 2**32), np.full_like(blocks, s["step"] >> 32)]
    for i in range(10):
        key = [np.uint64((s["seed"] % 2**32 + i * 0x9E3779B9) % 2**32), np.uint64(((s["seed"] >> 32) + i * 0xBB67AE85) % 2**32)]
        a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(b >> shift) ^ c[1] ^ key[0], b & word, (a >> shift) ^ c[3] ^ key[1], a & word]
    field = np.stack([c[k // 2] >> np.uint64(16 * (k % 2)) & np.uint64(0xFFFF) for k in range(8)], 1).reshape(-1)
    thr = int(round(case["p"] * 65536))
    factor = np.where(field[e] >= thr, 65536 / (65536 - thr), 0.0)
    return (x * factor, _host(s["gy"]) * factor) if case["train"] else x * factor
