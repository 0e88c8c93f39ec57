"""Low-rank adapters beside a shared projection, and the residual's addition with its norm and 8-bit output: what is measured.

Both operators sit at a W4A8 linear.  The residual stream takes a sub-layer's output in, is normalised, modulated and
quantised for the next linear; the requests of a batch add their own adapters' products to what that linear gives.  Four
kinds of case:

  adapt        out_i = base_i + s_g (x_i A_g^T) B_g^T, g the adapter of row i (rows without one keep base_i)
  adapt_train  the same, then the gradients of x, A and B from the output's gradient
  norm         t = x + gate y, h = t rsqrt(mean t^2 + eps) w (1 + scale) + shift, 8-bit codes of h (rotated by blocks) with a
               scale per row, and h itself where it is asked for
  norm_train   t and h, then the gradients of x, y and w

`run` computes them either in plain torch operations in 32 bits (`own` false) or through the package's entry points
(`own` true); `exact` restates the definitions in 64 bits.
"""
import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_DEV = "cuda"
_EPS = 1e-5
_MAX_ADAPT = 59440 * (5120 + 2 * 5120)  # elements of x, base and out of the largest listed adapter case
_MAX_TRAIN = 12090 * (2 * 5120 + 3 * 5120)
_MAX_NORM = 59440 * 5120


def listed():
    return [
        # one new row of each of four requests, their own adapters: launch latency only
        {"name": "adapt_4rows", "kind": "adapt", "dtype": "bf16", "M": 4, "K": 5120, "N": 5120, "r": 16, "R": 4, "map": "mixed",
         "none": False},
        # one row of each of 64 requests, 64 adapters of rank 64 beside the qkv projection: all time goes into reading them
        {"name": "adapt_64rows", "kind": "adapt", "dtype": "bf16", "M": 64, "K": 5120, "N": 15360, "r": 64, "R": 64,
         "map": "mixed", "none": False},
        # odd sizes: fp16, a rank that is no power of two, three requests and rows without an adapter
        {"name": "adapt_odd_fp16", "kind": "adapt", "dtype": "fp16", "M": 1031, "K": 1288, "N": 2056, "r": 24, "R": 3,
         "map": "runs", "none": True},
        # the 5 s video's rows, two requests, beside the qkv projection
        {"name": "adapt_12090", "kind": "adapt", "dtype": "bf16", "M": 12090, "K": 5120, "N": 15360, "r": 16, "R": 2,
         "map": "runs", "none": False},
        # the whole 40 s sequence over four adapters of rank 64, beside the output projection: the largest forward
        {"name": "adapt_59440", "kind": "adapt", "dtype": "bf16", "M": 59440, "K": 5120, "N": 5120, "r": 64, "R": 4,
         "map": "runs", "none": False},
        # a training step of odd sizes, rows of two adapters mixed, some without
        {"name": "adapt_train_odd_fp16", "kind": "adapt_train", "dtype": "fp16", "M": 517, "K": 640, "N": 1288, "r": 8, "R": 2,
         "map": "mixed", "none": True},
        # a training step of one adapter over the 5 s video's rows
        {"name": "adapt_train_12090", "kind": "adapt_train", "dtype": "bf16", "M": 12090, "K": 5120, "N": 5120, "r": 32, "R": 1,
         "map": "runs", "none": False},
        # one row of each of eight requests: launch latency only
        {"name": "norm_8rows", "kind": "norm", "dtype": "bf16", "M": 8, "K": 5120, "mods": 2, "none": False, "hidden": False},
        # odd row count, fp16, codes and the normalised stream too (adapters read it), rows outside every segment
        {"name": "norm_odd_fp16", "kind": "norm", "dtype": "fp16", "M": 1031, "K": 1280, "mods": 3, "none": True,
         "hidden": True},
        # the whole 40 s sequence into the codes of the next linear: the largest
        {"name": "norm_59440", "kind": "norm", "dtype": "bf16", "M": 59440, "K": 5120, "mods": 2, "none": False,
         "hidden": False},
        # a training step of odd sizes without gate or modulation
        {"name": "norm_train_odd_fp16", "kind": "norm_train", "dtype": "fp16", "M": 517, "K": 1288, "mods": 0, "none": False},
        # a training step over the 5 s video's rows at the official width
        {"name": "norm_train_12090", "kind": "norm_train", "dtype": "bf16", "M": 12090, "K": 5376, "mods": 2, "none": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["adapt", "adapt", "adapt", "adapt_train", "norm", "norm", "norm_train"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind.startswith("adapt"):
        r = rng.choice([4, 8, 16, 16, 24, 32, 64, 128])
        k, n = 8 * _log_int(rng, 16, 1920), 8 * _log_int(rng, 16, 1920)
        few = rng.random() < 0.4
        train = kind == "adapt_train"
        cap = _MAX_TRAIN // (2 * k + 3 * n) if train else _MAX_ADAPT // (k + 2 * n)
        # products and the listed ones' rank and rows bound the work as well as the bytes do
        cap = min(cap, (12090 * 32 if train else 59440 * 64) * 10240 // (r * (k + n)))
        m = rng.randint(1, 64) if few else _log_int(rng, 16 if train else 1, max(16, min(59440, cap)))
        big = rng.choice([1, 2, 4, 8]) if m > 512 else rng.randint(1, 64)
        return {"kind": kind, "dtype": dtype, "M": m, "K": k, "N": n, "r": r, "R": big,
                "map": rng.choice(["runs", "mixed"]), "none": rng.random() < 0.3}
    k = 256 * rng.randint(1, 56) if kind == "norm" else 8 * _log_int(rng, 16, 1792)
    m = _log_int(rng, 1, max(1, min(59440, _MAX_NORM // (2 if kind == "norm_train" else 1) // k)))
    case = {"kind": kind, "dtype": dtype, "M": m, "K": k, "mods": rng.randint(0, 4), "none": rng.random() < 0.3}
    if kind == "norm":
        case["hidden"] = rng.random() < 0.4
    return case


def _counts(case):
    """Rows of each adapter, ragged: in proportion to 1, 2, 3, ... R (and as many rows without one as the first has more)."""
    m, n = case["M"], case["R"] + (1 if case["none"] else 0)
    total = n * (n + 1) // 2
    ends = [m * ((i + 1) * (i + 2) // 2) // total for i in range(n)]
    return [e - s for s, e in zip([0] + ends[:-1], ends)]


def _segments(case):
    """(first row, end row, modulation row): even runs; with "none" the last rows are outside every segment."""
    m, n = case["M"], case["mods"]
    if n == 0:
        return []
    end = m - (m + 4) // 5 if case["none"] else m
    return [(end * i // n, end * (i + 1) // n, (i + 1) % n) for i in range(n)]


def _package():
    name = "minimax_h3_turbo_b200"
    if name not in sys.modules:
        root = Path(__file__).resolve().parent.parent / "minimax-h3-turbo_b200"
        spec = importlib.util.spec_from_file_location(name, root / "__init__.py", submodule_search_locations=[str(root)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    from minimax_h3_turbo_b200.h3 import adapters, residual

    return adapters, residual


def prepare(case, seed):
    g = torch.Generator(device=_DEV).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device=_DEV) * std).to(dt)

    m, k = case["M"], case["K"]
    st = {"case": case, "x": normal(m, k)}
    if case["kind"].startswith("adapt"):
        n, r, adapters = case["N"], case["r"], case["R"]
        counts = _counts(case)
        rows = torch.repeat_interleave(torch.arange(len(counts), device=_DEV), torch.tensor(counts, device=_DEV))
        if case["map"] == "mixed":
            rows = rows[torch.randperm(m, generator=g, device=_DEV)]
        # the rows of each adapter, a line per adapter, filled up with a row past the end: what the plain form gathers by
        first = torch.tensor([sum(counts[:i]) for i in range(adapters)], device=_DEV).view(-1, 1)
        many = torch.tensor(counts[:adapters], device=_DEV).view(-1, 1)
        at = torch.arange(max(1, max(counts[:adapters])), device=_DEV).view(1, -1)
        order = torch.argsort(rows, stable=True)
        st["lines"] = torch.where(at < many, order[(first + at).clamp(max=m - 1)], torch.full_like(first, m))
        st["rows"] = torch.where(rows < adapters, rows, torch.full_like(rows, -1)).to(torch.int32)
        st["a"] = normal(adapters, r, k, std=k ** -0.5)
        st["b"] = normal(adapters, n, r, std=r ** -0.5)
        st["scales"] = torch.rand(adapters, generator=g, device=_DEV) * 1.5 + 0.5
        st["base"] = normal(m, n)
        if case["kind"] == "adapt_train":
            st["do"] = normal(m, n)
    else:
        st["y"] = normal(m, k)
        st["w"] = (1.0 + 0.1 * torch.randn(k, generator=g, device=_DEV)).to(dt)
        mods = case["mods"]
        st["gate"] = normal(mods, k, std=0.5) if mods else None
        st["shift"] = normal(mods, k, std=0.2) if mods else None
        st["scale"] = normal(mods, k, std=0.2) if mods else None
        st["segments"] = _segments(case)
        if case["kind"] == "norm_train":
            st["dt"], st["dh"] = normal(m, k), normal(m, k)
    if own:
        st["adapters"], st["residual"] = _package()
        if case["kind"].startswith("adapt"):
            st["plan"] = st["adapters"].plan(st["rows"], case["R"])
    return st


# ------------------------------------------------------------------------------------------------ plain forms, 32 bits
def _plain_adapt(st):
    case = st["case"]
    m, n, k = case["M"], case["N"], case["K"]
    dt, at = st["x"].dtype, st["lines"]
    a, b, s = st["a"].float(), st["b"].float(), st["scales"].view(-1, 1, 1)

    def gather(t):  # [R, rows, width], the lines' ends filled with zeros
        return torch.cat([t.float(), torch.zeros(1, t.shape[1], device=_DEV)])[at]

    def scatter(t):  # back to [M, width], zeros where no line has the row
        out = torch.zeros(m + 1, t.shape[-1], device=_DEV)
        out[at.reshape(-1)] = t.reshape(-1, t.shape[-1])
        return out[:m]

    x = gather(st["x"])
    h = torch.bmm(x, a.transpose(1, 2)).mul_(s)
    out = scatter(torch.bmm(h, b.transpose(1, 2))).add_(st["base"].float()).to(dt)
    if case["kind"] == "adapt":
        return out
    go = gather(st["do"])
    dh = torch.bmm(go, b).mul_(s)
    return [out, scatter(torch.bmm(dh, a)).to(dt), torch.bmm(dh.transpose(1, 2), x).to(dt),
            torch.bmm(go.transpose(1, 2), h).to(dt)]


def _plain_rows(t, segments, m, fill):
    """[M, K] in 32 bits: each row's modulation row of t, `fill` outside every segment."""
    index = torch.full((m,), t.shape[0], device=_DEV, dtype=torch.int64)
    for first, end, row in segments:
        index[first:end] = row
    return torch.cat([t.float(), torch.full((1, t.shape[1]), fill, device=_DEV)])[index]


def _plain_norm(st):
    case = st["case"]
    m, k = case["M"], case["K"]
    dt, w = st["x"].dtype, st["w"].float()
    gate = up = None
    t = st["y"].float()
    if case["mods"]:
        gate = _plain_rows(st["gate"], st["segments"], m, 0.0)
        up = _plain_rows(st["scale"], st["segments"], m, 0.0).add_(1.0)
        t = t * gate
    t = t.add_(st["x"].float()).to(dt)
    tf = t.float()
    rstd = torch.rsqrt(tf.square().mean(-1, keepdim=True) + _EPS)
    n = tf * rstd
    h = n * w
    if case["mods"]:
        h = (h * up).add_(_plain_rows(st["shift"], st["segments"], m, 0.0))
    if case["kind"] == "norm_train":
        dn = st["dh"].float()
        if case["mods"]:
            dn = dn * up
        dw = (dn * n).sum(0)
        u = dn * w
        d = st["dt"].float() + rstd * (u - n * (u * n).mean(-1, keepdim=True))
        dy = d * gate if case["mods"] else d
        return [t, h.to(dt), d.to(dt), dy.to(dt), dw.to(dt)]
    h4 = torch.tensor([[1, 1, 1, -1], [1, 1, -1, 1], [1, -1, 1, 1], [-1, 1, 1, 1]], dtype=torch.float32, device=_DEV)
    h16 = torch.kron(h4, h4)
    z = torch.matmul(h.view(m, k // 256, 256), torch.kron(h16, h16) / 16.0).view(m, k)
    step = z.abs().amax(-1, keepdim=True) / 127.0
    codes = torch.round(z / step.clamp_min(1e-30))
    out = [t, codes.to(torch.bfloat16), step]  # codes: whole numbers up to 127, exact in bf16
    return out + [h.to(dt)] if case["hidden"] else out


def run(state):
    st, case = state, state["case"]
    if not own:
        return _plain_adapt(st) if case["kind"].startswith("adapt") else _plain_norm(st)
    if case["kind"].startswith("adapt"):
        low_rank, args = st["adapters"].low_rank, (st["x"], st["a"], st["b"], st["plan"])
        if case["kind"] == "adapt":
            return low_rank(*args, base=st["base"], scales=st["scales"])
        out, hidden = low_rank(*args, base=st["base"], scales=st["scales"], return_hidden=True)
        return [out, *st["adapters"].low_rank_backward(st["do"], *args, hidden, scales=st["scales"])]
    mod = {"gate": st["gate"], "scale": st["scale"], "segments": st["segments"]}
    norm = st["residual"].residual_norm
    if case["kind"] == "norm":
        r = norm(st["x"], st["y"], st["w"], _EPS, shift=st["shift"], codes=True, hidden=case["hidden"], **mod)
        out = [r.x, r.codes.to(torch.bfloat16), r.scales]
        return out + [r.hidden] if case["hidden"] else out
    r = norm(st["x"], st["y"], st["w"], _EPS, shift=st["shift"], codes=False, hidden=True, **mod)
    grads = st["residual"].residual_norm_backward(st["dt"], st["dh"], r.x, r.rstd, st["w"], **mod)
    return [r.x, r.hidden, *grads]


def work(case):
    m, k = case["M"], case["K"]
    if case["kind"].startswith("adapt"):
        n, r, counts = case["N"], case["r"], _counts(case)[:case["R"]]
        rows, used = sum(counts), sum(1 for c in counts if c)
        weights = used * r * (k + n)
        data = rows * k + 2 * m * n + weights  # x, base, out, the adapters in use
        flops = 2 * rows * r * (k + n)
        if case["kind"] == "adapt_train":  # g, dx, dA, dB as well; three times the products
            data += rows * n + m * k + case["R"] * r * (k + n)
            flops *= 3
        return {"bytes": 2 * data + 4 * m, "flops": flops}
    mod = 2 * (3 * case["mods"] + 1) * k
    if case["kind"] == "norm":  # x, y, t; codes and scales; h where it is asked for
        # a butterfly stage is two sums a value for each of the four base-4 digits of the rotation
        return {"bytes": m * k * (7 + (2 if case["hidden"] else 0)) + 4 * m + mod, "flops": 17 * m * k}
    return {"bytes": 2 * m * k * (7 + (1 if case["mods"] else 0)) + mod + 2 * k, "flops": 20 * m * k}


# ------------------------------------------------------------------------------------------------ definitions, 64 bits
def _exact_adapt(case, st):
    m, n, k = case["M"], case["N"], case["K"]
    out = st["base"].double()
    dx = torch.zeros(m, k, dtype=torch.float64, device=_DEV)
    da = torch.zeros(st["a"].shape, dtype=torch.float64, device=_DEV)
    db = torch.zeros(st["b"].shape, dtype=torch.float64, device=_DEV)
    for i in range(case["R"]):
        sel = (st["rows"] == i).nonzero().flatten()
        w = float(st["scales"][i]) * (st["b"][i].double() @ st["a"][i].double()) if sel.numel() > 4096 else None
        for part in sel.split(8192):
            x = st["x"][part].double()
            low = x @ st["a"][i].double().T
            out[part] += float(st["scales"][i]) * low @ st["b"][i].double().T
            if case["kind"] == "adapt_train":
                g = st["do"][part].double() * float(st["scales"][i])
                db[i] += g.T @ low
                da[i] += (g @ st["b"][i].double()).T @ x
                dx[part] = st["do"][part].double() @ w if w is not None else (g @ st["b"][i].double()) @ st["a"][i].double()
    return [out, dx, da, db] if case["kind"] == "adapt_train" else out


def _exact_norm(case, st):
    m, k = case["M"], case["K"]
    dt, w = st["x"].dtype, st["w"].double()
    t, h, z = (torch.empty(m, k, dtype=torch.float64, device=_DEV) for _ in range(3))
    d, dy, dw = torch.empty_like(t), torch.empty_like(t), torch.zeros(k, dtype=torch.float64, device=_DEV)
    owner = [-1] * m
    for first, end, row in st["segments"]:
        owner[first:end] = [row] * (end - first)
    owner = torch.tensor(owner, device=_DEV)
    for row in ([-1] + list(range(case["mods"]))):
        for sel in (owner == row).nonzero().flatten().split(8192):
            plain = row < 0
            gate = (torch.ones(k, device=_DEV) if case["mods"] == 0 else torch.zeros(k, device=_DEV)).double() if plain else \
                st["gate"][row].double()
            up = 1.0 if plain else 1.0 + st["scale"][row].double()
            # the sum is the stream as it is held: rounded to the type, and read back from there
            v = (st["x"][sel].double() + gate * st["y"][sel].double()).to(dt).double()
            t[sel] = v
            size = torch.sqrt((v ** 2).sum(1, keepdim=True) / k + _EPS)
            unit = v / size
            h[sel] = unit * w * up + (0.0 if plain else st["shift"][row].double())
            if case["kind"] == "norm_train":
                g = st["dh"][sel].double() * up
                dw += (g * unit).sum(0)
                g = g * w
                full = st["dt"][sel].double() + (g - unit * ((g * unit).sum(1, keepdim=True) / k)) / size
                d[sel], dy[sel] = full, full * gate
    if case["kind"] == "norm_train":
        return [t, h, d, dy, dw]
    x = h.view(m, -1, 4, 4, 4, 4)
    for axis in range(2, 6):  # one base-4 digit after the other: half the digit's sum less the value at the mirrored place
        x = x.sum(axis, keepdim=True) / 2.0 - x.flip(axis)
    z = x.reshape(m, k)
    step = z.abs().max(dim=1, keepdim=True).values / 127
    codes = torch.round(z / torch.where(step > 0, step, torch.ones_like(step)))
    out = [t, codes, step]
    return out + [h] if case["hidden"] else out


def exact(case, seed):
    st = prepare(case, seed)
    return _exact_adapt(case, st) if case["kind"].startswith("adapt") else _exact_norm(case, st)
