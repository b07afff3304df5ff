"""Cases of the sequence-training operators: the gated linear recurrence along an axis, 8-bit activation
checkpoints with their use in the backward pass, and the softmax cross-entropy with its gradient map.

`own = False` computes the plain forms (elementary torch operations), `own = True` calls the library."""
import math

import numpy as np
import torch

own = False

BLOCK = 128          # elements that share one magnitude in an 8-bit checkpoint
MOST = 1 << 26       # elements of the largest recurrence and of the largest checkpoint in f32
MOST_LOGITS = 1 << 28


def listed():
    return [
        # one token for each of 64 sequences being generated: the state of 2048 channels moves one step in place
        _scan("scan step 64x2048", "step", 64, 1, 2048),
        # a short batch, forward only (evaluation)
        _scan("scan fwd 16x256x512", "fwd", 16, 256, 512),
        # an ordinary training batch, forward and backward
        _scan("scan train 8x8192x1024", "train", 8, 8192, 1024),
        # one long document, a scalar decay for each of 16 heads: the states are kept in 8 bits, the backward pass reads them
        _scan("scan back8 1x65536x1024 h16", "back8", 1, 65536, 1024, heads=16),
        # the reverse direction of a bidirectional model in f64, odd sizes, interpolating gate, initial state
        _scan("scan train 3x1537x250 f64", "train", 3, 1537, 250, dtype="f64", coupled=True, reverse=True, h0=True),
        # channels first: the recurrence runs along the contiguous axis
        _scan("scan fwd 4x512x8192 rows", "fwd", 4, 8192, 512, layout="bdt"),
        # one hidden activation of the dense MLP at its batch, kept in 8 bits and restored
        _ckpt("ckpt restore 4096x1024", "restore", 4096 * 1024),
        # the saved result of a sigmoid over a large batch, kept and used by its backward pass
        _ckpt("ckpt sigmoid 8192x8192", "sigmoid", 8192 * 8192),
        # an odd length in f64, the saved result of a tanh
        _ckpt("ckpt tanh 1000003 f64", "tanh", 1000003, dtype="f64"),
        # the ten-class head of the dense MLP at its batch
        _ce("ce train 4096x10", True, 4096, 10),
        # next-token loss over an ordinary vocabulary
        _ce("ce train 8192x32000", True, 8192, 32000),
        # odd sizes in f64, some rows are padding
        _ce("ce train 517x5003 f64", True, 517, 5003, dtype="f64", padded=True),
    ]


def _scan(name, way, b, t, d, heads=0, dtype="f32", coupled=False, reverse=False, h0=False, layout="btd"):
    return {"name": name, "op": "scan", "way": way, "b": b, "t": t, "d": d, "heads": heads, "dtype": dtype, "coupled": coupled,
            "reverse": reverse, "h0": h0, "layout": layout}


def _ckpt(name, way, n, dtype="f32"):
    return {"name": name, "op": "ckpt", "way": way, "n": n, "dtype": dtype}


def _ce(name, train, rows, classes, dtype="f32", padded=False):
    return {"name": name, "op": "ce", "train": train, "rows": rows, "classes": classes, "dtype": dtype, "padded": padded}


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("scan", "scan", "ckpt", "ce"))
    dtype = "f64" if rng.random() < 0.2 else "f32"
    half = 2 if dtype == "f64" else 1
    if op == "ckpt":
        c = _ckpt("", rng.choice(("restore", "mul", "sigmoid", "tanh", "square")), _log_int(rng, 1000, MOST // half), dtype)
    elif op == "ce":
        classes = _log_int(rng, 2, 131072)
        rows = _log_int(rng, 1, max(1, min(16384, MOST_LOGITS // half // classes)))
        if dtype == "f64":
            rows = max(1, min(rows, (1 << 24) // classes))
        c = _ce("", rng.random() < 0.75, rows, classes, dtype, rng.random() < 0.5)
    else:
        way = rng.choice(("fwd", "train", "back8", "step"))
        heads = rng.choice((0, 0, 0, 4, 16)) if way != "step" else 0
        d = heads * rng.choice((16, 31, 64, 100, 128)) if heads else _log_int(rng, 8, 4096)
        t = 1 if way == "step" else _log_int(rng, 1, 65536)
        b = _log_int(rng, 1, max(1, min(2048 if way == "step" else 256, MOST // half // (t * d))))
        t = min(t, max(1, MOST // half // (b * d)))
        layout = "bdt" if way != "step" and not heads and rng.random() < 0.3 else "btd"
        c = _scan("", way, b, t, d, heads, dtype, rng.random() < 0.4, way != "step" and rng.random() < 0.3,
                  way != "step" and rng.random() < 0.5, layout)
    del c["name"]
    return c


def _torch_dtype(case):
    return torch.float64 if case["dtype"] == "f64" else torch.float32


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    dt = _torch_dtype(case)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", dtype=dt, generator=g)

    s = {"case": case, "seed": seed}
    if case["op"] == "ckpt":
        n, way = case["n"], case["way"]
        x = normal(n)
        s["x"] = torch.sigmoid_(x) if way == "sigmoid" else torch.tanh_(x) if way == "tanh" else x
        if way != "restore":
            s["up"] = normal(n)
    elif case["op"] == "ce":
        rows, classes = case["rows"], case["classes"]
        s["logits"] = normal(rows, classes).mul_(2.0)
        s["targets"] = torch.randint(0, classes, (rows,), device="cuda", generator=g)
        if case["padded"] and rows > 1:
            pad = torch.rand(rows, device="cuda", generator=g) < 0.1
            pad[0] = False
            s["targets"][pad] = -1
    else:
        b, t, d, heads = case["b"], case["t"], case["d"], case["heads"]
        if case["layout"] == "bdt":
            shape, gate_shape, s["axis"] = (b, d, t), (b, d, t), 2
        elif heads:
            shape, gate_shape, s["axis"] = (b, t, heads, d // heads), (b, t, heads, 1), 1
        else:
            shape, gate_shape, s["axis"] = (b, t, d), (b, t, d), 1
        s["x"] = normal(*shape)
        s["gate"] = torch.sigmoid_(normal(*gate_shape).add_(3.0))
        first = tuple(1 if k == s["axis"] else n for k, n in enumerate(shape))
        s["h0"] = normal(*first) if case["h0"] or case["way"] == "step" else None
        if case["way"] in ("train", "back8"):
            s["up"] = normal(*shape)
        if case["way"] == "back8":   # the forward pass's states, some layers earlier in the program
            s["h"] = normal(*shape).mul_(3.0)
    return s


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


def work(case):
    es = 8 if case["dtype"] == "f64" else 4
    if case["op"] == "ckpt":
        n = case["n"]
        return {"bytes": n * es * (2 if case["way"] == "restore" else 3), "flops": 6.0 * n}
    if case["op"] == "ce":
        n = case["rows"] * case["classes"]
        return {"bytes": n * es * (2 if case["train"] else 1) + 8 * case["rows"], "flops": 6.0 * n}
    n = case["b"] * case["t"] * case["d"]
    gate = case["b"] * case["t"] * case["heads"] if case["heads"] else n
    ends = case["b"] * case["d"] if case["h0"] else 0
    if case["way"] == "step":
        return {"bytes": es * (3 * n + gate), "flops": 2.0 * n}
    if case["way"] == "fwd":
        return {"bytes": es * (2 * n + gate + ends), "flops": 2.0 * n}
    read = (3 if case["coupled"] else 2) if case["way"] == "back8" else 2
    wrote = 1 if case["way"] == "back8" else 2
    return {"bytes": es * ((read + wrote) * n + 2 * gate + 2 * ends), "flops": 6.0 * n}


# ---- plain forms --------------------------------------------------------------------------------------

def _prefix(a, b):
    """h_s = a_s h_{s-1} + b_s from zero along dim 1, by doubling: pairs of steps, of pairs, and so on."""
    span = 1
    while span < a.shape[1]:
        b = torch.cat((b[:, :span], b[:, span:] + a[:, span:] * b[:, :-span]), 1)
        if span * 2 < a.shape[1]:
            a = torch.cat((a[:, :span], a[:, span:] * a[:, :-span]), 1)
        span *= 2
    return b


def _ahead(v, first):
    """`v` one step later along dim 1, `first` in the first place."""
    return torch.cat((first, v[:, :-1]), 1)


def _quantise(x):
    """Codes (-127 .. 127) and the magnitude of each block; in 64 bits, where a code's border is never missed."""
    n = x.numel()
    v = torch.nn.functional.pad(x.reshape(-1).double(), (0, -n % BLOCK)).view(-1, BLOCK)
    top = v.abs().amax(1, keepdim=True)
    return torch.round(127.0 * v / torch.where(top > 0, top, 1.0)), top


def _restored(x):
    codes, top = _quantise(x)
    return (codes * top / 127.0).reshape(-1)[: x.numel()].to(x.dtype).view(x.shape)


def _plain_scan(s):
    c, axis = s["case"], s["axis"]
    x, gate, h0 = s["x"], s["gate"], s["h0"]
    if c["way"] == "step":
        h0.copy_(gate * h0 + ((1.0 - gate) * x if c["coupled"] else x))
        return h0
    a = gate.expand(x.shape)

    def turn(v):   # time at dim 1, in the order of processing
        v = v.movedim(axis, 1)
        return v.flip(1) if c["reverse"] else v

    def back(v):
        return (v.flip(1) if c["reverse"] else v).movedim(1, axis).contiguous()

    a, xs = turn(a), turn(x)
    b = (1.0 - a) * xs if c["coupled"] else xs
    first = turn(h0) if h0 is not None else torch.zeros_like(b[:, :1])
    if h0 is not None:
        b = torch.cat((b[:, :1] + a[:, :1] * first, b[:, 1:]), 1)
    if c["way"] == "back8":
        h = turn(_restored(s["h"]))
    else:
        h = _prefix(a, b)
    if c["way"] == "fwd":
        return back(h)
    up = turn(s["up"])
    later = torch.cat((a[:, 1:], torch.zeros_like(a[:, :1])), 1)
    g = _prefix(later.flip(1), up.flip(1)).flip(1)
    before = _ahead(h, first)
    if c["coupled"]:
        dx, da = (1.0 - a) * g, g * (before - xs)
    else:
        dx, da = g, g * before
    da = back(da)
    if c["heads"]:
        da = da.sum(-1, keepdim=True)
    grads = {"dx": back(dx), "dgate": da}
    if c["way"] == "train":
        grads["h"] = back(h)
    if h0 is not None:
        grads["dh0"] = (a[:, :1] * g[:, :1]).movedim(1, axis).contiguous()
    return grads


def _plain_ckpt(s):
    x, way = s["x"], s["case"]["way"]
    r = _restored(x)
    if way == "restore":
        return r
    up = s["up"]
    if way == "mul":
        return r * up
    if way == "sigmoid":
        return r * (1.0 - r) * up
    if way == "tanh":
        return (1.0 - r * r) * up
    return 2.0 * r * up


def _plain_ce(s):
    x, t = s["logits"], s["targets"]
    counted = t >= 0
    at = torch.where(counted, t, 0)[:, None]
    v = x - x.amax(1, keepdim=True)
    e = v.exp()
    total = e.sum(1, keepdim=True)
    n = counted.sum()
    rows = torch.where(counted[:, None], total.log() - v.gather(1, at), 0.0)
    loss = (rows.double().sum() / n).to(x.dtype)
    if not s["case"]["train"]:
        return loss
    e.div_(total)
    e.scatter_add_(1, at, torch.full_like(at, -1, dtype=x.dtype))
    e.mul_(counted[:, None] / n.to(x.dtype))
    return {"loss": loss, "map": e}


_PLAIN = {"scan": _plain_scan, "ckpt": _plain_ckpt, "ce": _plain_ce}


# ---- the library's calls ------------------------------------------------------------------------------

def _tensor(buf):
    from rtensors_b200.meta import Meta
    from rtensors_b200.tensor import Tensor, default_backend
    return Tensor(default_backend(), buf.view(-1), Meta.contiguous(buf.shape))


def _own_scan(s):
    from rtensors_b200.tensor import gated_scan_backward
    c, axis = s["case"], s["axis"]
    x, gate = _tensor(s["x"]), _tensor(s["gate"])
    h0 = _tensor(s["h0"]) if s["h0"] is not None else None
    if c["way"] == "step":
        h0.gated_step_inplace(gate, x, coupled=c["coupled"])
        return s["h0"]
    if c["way"] == "back8":
        h = _tensor(s["h"]).checkpoint8()
    else:
        h = x.gated_scan_at(axis, gate, h0, reverse=c["reverse"], coupled=c["coupled"])
    if c["way"] == "fwd":
        return h.buf.view(s["x"].shape)
    dx, dgate, dh0 = gated_scan_backward(_tensor(s["up"]), axis, gate, h, x=x if c["coupled"] else None, h0=h0,
                                         reverse=c["reverse"], coupled=c["coupled"])
    grads = {"dx": dx.buf.view(s["x"].shape), "dgate": dgate.buf.view(s["gate"].shape)}
    if c["way"] == "train":
        grads["h"] = h.buf.view(s["x"].shape)
    if h0 is not None:
        grads["dh0"] = dh0.buf.view(s["h0"].shape)
    return grads


def _own_ckpt(s):
    kept = _tensor(s["x"]).checkpoint8()
    if s["case"]["way"] == "restore":
        return kept.restore().buf
    return kept.grad(s["case"]["way"], _tensor(s["up"])).buf


def _own_ce(s):
    from rtensors_b200.tensor import cross_entropy_loss
    logits, targets = _tensor(s["logits"]), _tensor(s["targets"])
    if not s["case"]["train"]:
        return cross_entropy_loss(logits, targets).buf.view(())
    loss, gmap = cross_entropy_loss(logits, targets, with_grad=True)
    return {"loss": loss.buf.view(()), "map": gmap.buf.view(s["logits"].shape)}


_OWN = {"scan": _own_scan, "ckpt": _own_ckpt, "ce": _own_ce}


# ---- from the definitions, step by step in 64 bits ------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"scan": _exact_scan, "ckpt": _exact_ckpt, "ce": _exact_ce}[case["op"]](s)


def _exact_kept(v):
    """What an 8-bit checkpoint of `v` (as it is stored, in its own type) stands for, on the host."""
    flat = v.detach().reshape(-1).cpu().numpy().astype(np.float64)
    blocks = np.zeros((-(-flat.size // BLOCK), BLOCK))
    blocks.reshape(-1)[: flat.size] = flat
    top = np.abs(blocks).max(axis=1, keepdims=True)
    t = np.divide(blocks * 127.0, top, out=np.zeros_like(blocks), where=top > 0)
    low = np.floor(t)
    odd = np.abs(np.fmod(low, 2.0))
    codes = low + np.where((t - low > 0.5) | ((t - low == 0.5) & (odd == 1.0)), 1.0, 0.0)
    return torch.from_numpy((codes / 127.0 * top).reshape(-1)[: flat.size].copy()).view(v.shape)


def _exact_scan(s):
    c, axis = s["case"], s["axis"]
    x, a = s["x"].double(), s["gate"].double().expand(s["x"].shape)
    x, a = x.movedim(axis, 0).contiguous(), a.movedim(axis, 0).contiguous()
    n = x.shape[0]
    start = torch.zeros_like(x[0]) if s["h0"] is None else s["h0"].double().select(axis, 0).clone()
    if c["way"] == "step":
        h = a[0] * start + ((1 - a[0]) * x[0] if c["coupled"] else x[0])
        return h.unsqueeze(axis).contiguous()
    order = range(n - 1, -1, -1) if c["reverse"] else range(n)
    if c["way"] == "back8":
        h = _exact_kept(s["h"]).cuda().movedim(axis, 0).contiguous()
    else:
        h, last = torch.empty_like(x), start
        for t in order:
            last = a[t] * last
            last += (1 - a[t]) * x[t] if c["coupled"] else x[t]
            h[t] = last
    if c["way"] == "fwd":
        return h.movedim(0, axis).contiguous()
    up = s["up"].double().movedim(axis, 0).contiguous()
    dx, da = torch.empty_like(x), torch.empty_like(x)
    g = torch.zeros_like(start)
    order = list(order)
    for k in range(n - 1, -1, -1):
        t = order[k]
        g = g + up[t]
        before = h[order[k - 1]] if k else start
        dx[t] = (1 - a[t]) * g if c["coupled"] else g
        da[t] = g * (before - x[t]) if c["coupled"] else g * before
        g = g * a[t]
    da = da.movedim(0, axis)
    if c["heads"]:
        da = da.sum(-1, keepdim=True)
    grads = {"dx": dx.movedim(0, axis).contiguous(), "dgate": da.contiguous()}
    if c["way"] == "train":
        grads["h"] = h.movedim(0, axis).contiguous()
    if s["h0"] is not None:
        grads["dh0"] = g.unsqueeze(axis).contiguous()
    return grads


def _exact_ckpt(s):
    way = s["case"]["way"]
    r = _exact_kept(s["x"]).cuda()
    if way == "restore":
        return r
    d = {"mul": lambda: r, "sigmoid": lambda: r - r ** 2, "tanh": lambda: 1 - r ** 2, "square": lambda: r + r}[way]()
    return d * s["up"].double()


def _exact_ce(s):
    t = s["targets"].cpu().numpy()
    rows, classes = s["logits"].shape
    if rows * classes > (1 << 25):   # in parts, to stay within the card's memory
        step = max(1, (1 << 25) // classes)
    else:
        step = rows
    count = int((t >= 0).sum())
    loss, parts = 0.0, []
    for r in range(0, rows, step):
        x = s["logits"][r: r + step].double()
        tt = s["targets"][r: r + step]
        lse = torch.logsumexp(x, 1)
        ok = tt >= 0
        hit = torch.arange(classes, device="cuda")[None, :] == tt[:, None]
        loss += float(((lse * ok) - (x * hit).sum(1)).sum())
        if s["case"]["train"]:
            parts.append(((torch.exp(x - lse[:, None]) - hit.double()) * ok[:, None] / count))
    loss = torch.tensor(loss / count, dtype=torch.float64)
    return {"loss": loss, "map": torch.cat(parts)} if s["case"]["train"] else loss
