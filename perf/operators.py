"""The state-space and adapter operators as users give them work: a fixed list of timed cases and a generator of more of them.

Three kinds, each one call of the library's public entry points:
  conv   the short causal convolution before a state-space scan (ops.ssm_conv), whole behaviour lists or one new behaviour a user
  scan   the selective state-space scan (ops.ssm_scan), whole lists or one new behaviour a user
  lora   a projection shared by all rows with a low-rank adapter of each row's own scene (ops.lora_gemm)

The plain forms below are elementary torch operations in 32 bits, rounded once at the end.
"""
import math

import torch

own = False

_T = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"f16": 2, "bf16": 2, "f32": 4}
_SCAN_MOST = 70_000 * 256 * 16      # values of the plain form's [rows, D, N] intermediates in the largest listed case
_CONV_MOST = 262_144 * 512
_LORA_MOST = 65536 * 1280 * 1024


def listed():
    return [
        # one new behaviour each of four users, interest extractor of twice the DIN width: the latency of a single token
        dict(name="scan_step_small", kind="scan", rows=4, batch=4, ragged=False, D=72, N=16, groups=1, dtype="f16", gate=True, carry=True),
        # one new behaviour of every active user: the states' traffic
        dict(name="scan_step_bulk", kind="scan", rows=8192, batch=8192, ragged=False, D=256, N=16, groups=1, dtype="bf16", gate=True, carry=True),
        # the headline batch's behaviour lists: 74 requests of 100 steps
        dict(name="scan_history", kind="scan", rows=7400, batch=74, ragged=False, D=72, N=16, groups=1, dtype="f16", gate=True, carry=False),
        # lists of every length packed one after the other, some continued from kept states
        dict(name="scan_ragged", kind="scan", rows=70_000, batch=256, ragged=True, D=256, N=16, groups=1, dtype="bf16", gate=True, carry=True),
        # one life-long list at odd sizes, in fp32, two groups of B and C
        dict(name="scan_long", kind="scan", rows=30_011, batch=1, ragged=True, D=202, N=10, groups=2, dtype="f32", gate=False, carry=True),
        # one new behaviour each of 74 users
        dict(name="conv_step", kind="conv", rows=74, batch=74, ragged=False, D=72, K=4, dtype="f16", carry=True),
        # packed lists of every length, bulk scoring
        dict(name="conv_ragged", kind="conv", rows=262_144, batch=1024, ragged=True, D=512, K=4, dtype="bf16", carry=True),
        # one life-long list at odd sizes, in fp32
        dict(name="conv_long", kind="conv", rows=30_011, batch=1, ragged=True, D=205, K=3, dtype="f32", carry=False),
        # 64 rows of as many scenes at the large tower's first layer: single tokens, each with an adapter of its own
        dict(name="lora_rows", kind="lora", requests=64, rows=64, K=1280, N=1024, adapters=64, rank=16, dtype="f16", out="f16", packed=True),
        # the DIN tower's first layer for 74 requests of 1000 candidates, a scene a request
        dict(name="lora_tower", kind="lora", requests=74, rows=74_000, K=324, N=200, adapters=12, rank=8, dtype="f16", out="f16", packed=True),
        # the large tower's first layer on a full batch, the compute-bound case
        dict(name="lora_bulk", kind="lora", requests=256, rows=65536, K=1280, N=1024, adapters=32, rank=16, dtype="bf16", out="bf16", packed=True),
        # ragged requests at odd sizes, weights as Blaze holds them, fp32 results
        dict(name="lora_odd", kind="lora", requests=37, rows=5003, K=250, N=131, adapters=5, rank=12, dtype="bf16", out="f32", packed=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["scan", "scan", "conv", "lora", "lora"])
    dtype = rng.choice(["f16", "bf16", "f32"])
    if kind == "lora":
        while True:
            K, N = _log(rng, 16, 1280), _log(rng, 8, 1024)
            if rng.random() < 0.7:
                K, N = (K + 7) // 8 * 8, (N + 7) // 8 * 8
            rows, rank, adapters = _log(rng, 1, 80_000), rng.choice([1, 4, 8, 16, 24, 32, 64]), _log(rng, 1, 64)
            if rows * (K * N + adapters * rank * (K + N)) <= _LORA_MOST:
                break
        return dict(kind=kind, requests=_log(rng, 1, min(rows, 1024)), rows=rows, K=K, N=N, adapters=adapters, rank=rank, dtype=dtype,
                    out=rng.choice([dtype, "f32"]), packed=rng.random() < 0.6)
    step, cut = rng.random() < 0.35, rng.random() < 0.2        # single tokens; lists that were cut to one length
    while True:
        D = _log(rng, 16, 1024)
        if rng.random() < 0.6:
            D = (D + 7) // 8 * 8
        batch = _log(rng, 1, 8192) if step else _log(rng, 1, 1024)
        rows = batch if step else _log(rng, max(batch // 2, 1), 70_000 if kind == "scan" else 262_144)
        if cut and not step:
            rows = max(rows // batch, 1) * batch
        if kind == "conv":
            if rows * D <= _CONV_MOST:
                return dict(kind=kind, rows=rows, batch=batch, ragged=not (step or cut), D=D, K=rng.choice([2, 3, 4, 5]), dtype=dtype, carry=rng.random() < 0.6)
            continue
        N, groups = rng.choice([4, 8, 13, 16, 16, 16, 32, 64]), rng.choice([1, 1, 2, 4])
        if D % groups == 0 and rows * D * N <= _SCAN_MOST:
            return dict(kind=kind, rows=rows, batch=batch, ragged=not (step or cut), D=D, N=N, groups=groups, dtype=dtype, gate=rng.random() < 0.7,
                        carry=rng.random() < 0.6)


def _lengths(rows, batch, seed):
    """`batch` list lengths that add up to `rows`: mostly of the mean's order, some long, some empty."""
    g = torch.Generator().manual_seed(seed)
    w = torch.empty(batch, dtype=torch.float64).exponential_(1.0, generator=g) + 1e-3
    ends = (w.cumsum(0) / w.sum() * rows).floor().to(torch.int64)
    ends[-1] = rows
    return torch.diff(ends, prepend=torch.zeros(1, dtype=torch.int64))


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _T[c["dtype"]]

    def normal(*shape, mean=0.0, std=1.0, to=torch.float32):
        return (torch.randn(shape, device="cuda", generator=gen) * std + mean).to(to)

    s = dict(c)
    if c["kind"] == "lora":
        # rows of the operands start on 16 bytes where the layers are kept packed, as the library lays its weights out
        pad = (c["K"] + 7) // 8 * 8 if c["packed"] else c["K"]
        s["X"] = normal(c["rows"], pad, to=dt)[:, :c["K"]]
        s["W"] = (normal(c["N"], pad, std=c["K"] ** -0.5, to=dt)[:, :c["K"]] if c["packed"] else
                  normal(c["K"], c["N"], std=c["K"] ** -0.5, to=dt))
        s["A"] = normal(c["adapters"], c["rank"], pad, std=c["K"] ** -0.5, to=dt)[:, :, :c["K"]]
        s["B"] = normal(c["adapters"], c["N"], c["rank"], std=0.5 * c["rank"] ** -0.5, to=dt)
        s["bias"] = normal(c["N"], std=0.1)
        s["scale"] = torch.rand(c["adapters"], device="cuda", generator=gen) + 0.5
        g = torch.Generator().manual_seed(seed)
        scene = torch.randint(-1, c["adapters"], (c["requests"],), generator=g)     # -1: a request without an adapter
        if c["requests"] == c["rows"]:
            scene = torch.randperm(c["rows"], generator=g) % c["adapters"]
        s["adapter"] = torch.repeat_interleave(scene, _lengths(c["rows"], c["requests"], seed) if c["requests"] < c["rows"] else 1).to(
            device="cuda", dtype=torch.int32)
        return s
    rows, batch, D = c["rows"], c["batch"], c["D"]
    lengths = torch.full((batch,), rows // batch) if not c["ragged"] else _lengths(rows, batch, seed)
    s["equal"] = int(lengths[0]) if bool((lengths == lengths[0]).all()) else 0
    s["longest"] = int(lengths.max())
    s["lengths"] = lengths
    offsets = torch.zeros(batch + 1, dtype=torch.int32)
    offsets[1:] = lengths.cumsum(0)
    s["offsets"] = offsets.cuda()
    # users lie anywhere in the table of kept states
    s["slots"] = torch.randperm(batch, device="cuda", generator=gen).to(torch.int32) if c["carry"] else None
    s["x"] = normal(rows, D, to=dt)
    if c["kind"] == "conv":
        s["w"], s["b"] = normal(D, c["K"], std=c["K"] ** -0.5, to=dt), normal(D, std=0.1, to=dt)
        s["state"] = normal(batch, c["K"] - 1, D, to=dt) if c["carry"] else None
        s["state_out"] = torch.zeros((batch, c["K"] - 1, D), device="cuda", dtype=dt)
        return s
    N, G = c["N"], c["groups"]
    s["delta"] = normal(rows, D, std=0.5, to=dt)
    step0 = torch.exp(torch.rand(D, device="cuda", generator=gen) * math.log(100.0) + math.log(1e-3))   # steps of 0.001 to 0.1
    s["delta_bias"] = step0 + torch.log(-torch.expm1(-step0))
    s["A"] = -torch.arange(1, N + 1, device="cuda", dtype=torch.float32) * torch.exp(normal(D, N, std=0.1))
    s["B"], s["C"] = normal(rows, G * N, to=dt), normal(rows, G * N, to=dt)
    s["Dskip"] = normal(D, mean=1.0, std=0.1)
    s["z"] = normal(rows, D, to=dt) if c["gate"] else None
    s["h"] = normal(batch, D, N, std=0.3) if c["carry"] else None
    s["h_out"] = torch.zeros((batch, D, N), device="cuda")
    return s


def _ops():
    from __graft_entry__ import load_package
    load_package()
    from x_deeplearning_b200 import ops
    return ops


def run(s):
    if own:
        ops = _ops()
        if s["kind"] == "lora":
            return ops.lora_gemm(s["X"], s["W"], s["A"], s["B"], s["adapter"], bias=s["bias"], scale=s["scale"], trans_b=s["packed"],
                                 out_dtype=_T[s["out"]])
        lists = dict(T=s["equal"]) if s["equal"] else dict(offsets=s["offsets"])
        if s["kind"] == "conv":
            y = ops.ssm_conv(s["x"], s["w"], s["b"], state_in=s["state"], state_out=s["state_out"], slots=s["slots"], **lists)
            return y, s["state_out"]
        y = ops.ssm_scan(s["x"], s["delta"], s["A"], s["B"], s["C"], D=s["Dskip"], z=s["z"], delta_bias=s["delta_bias"], groups=s["groups"],
                         h_in=s["h"], h_out=s["h_out"], slots=s["slots"], longest=s["longest"], **lists)
        return y, s["h_out"]
    return {"lora": _plain_lora, "conv": _plain_conv, "scan": _plain_scan}[s["kind"]](s)


def _plain_lora(s):
    X, A, B = s["X"].float(), s["A"].float(), s["B"].float()
    n, r, _ = A.shape
    a = s["adapter"].long()
    Y = X @ (s["W"].float().t() if s["packed"] else s["W"].float()) + s["bias"]
    # every row against every adapter, then its own alone is kept
    U = (X @ A.reshape(n * r, -1).t()).view(-1, n, r)
    keep = torch.arange(n, device=X.device) == a[:, None]
    U = torch.where(keep[:, :, None], U * s["scale"][None, :, None], 0.0)
    Y = Y + U.view(-1, n * r) @ B.transpose(1, 2).reshape(n * r, -1)
    return Y.to(_T[s["out"]])


def _sequence_of_rows(s):
    """The list that each row belongs to, and its place in it."""
    off = s["offsets"].long()
    rows = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(off[1:].contiguous(), rows, right=True)
    return off, rows, seq, rows - off[seq]


def _plain_conv(s):
    x, w, K = s["x"].float(), s["w"].float(), s["K"]
    off, rows, seq, place = _sequence_of_rows(s)
    slots = s["slots"].long() if s["slots"] is not None else torch.arange(s["batch"], device="cuda")
    state = s["state"].float() if s["state"] is not None else torch.zeros((s["batch"], K - 1, s["D"]), device="cuda")
    # with its state ahead of each list the inputs are one padded sequence
    ahead = torch.zeros((s["rows"] + s["batch"] * (K - 1), s["D"]), device="cuda")
    begin = off[:-1] + (K - 1) * torch.arange(s["batch"], device="cuda")
    at = torch.arange(K - 1, device="cuda")
    ahead[(begin[:, None] + at).reshape(-1)] = state[slots].reshape(-1, s["D"])
    mine = begin[seq] + (K - 1) + place
    ahead[mine] = x
    y = s["b"].float() + sum(ahead[mine - (K - 1) + j] * w[:, j] for j in range(K))
    end = begin + (off[1:] - off[:-1])
    out = torch.zeros_like(state)
    out[slots] = ahead[(end[:, None] + at).reshape(-1)].view(-1, K - 1, s["D"])
    return (y / (1 + torch.exp(-y))).to(s["x"].dtype), out.to(s["x"].dtype)


def _plain_scan(s):
    x, N, G, D = s["x"].float(), s["N"], s["groups"], s["D"]
    off, rows, seq, place = _sequence_of_rows(s)
    v = s["delta"].float() + s["delta_bias"]
    d = torch.where(v > 20, v, torch.log1p(torch.exp(v.clamp(max=20))))
    per = D // G
    Bm, Cm = s["B"].float().view(-1, G, 1, N), s["C"].float().view(-1, G, 1, N)
    a = torch.exp(d[:, :, None] * s["A"])
    b = ((d * x).view(-1, G, per, 1) * Bm).reshape(-1, D, N)
    # the state of a list's beginning goes into its first row, which then looks back no further
    slots = s["slots"].long() if s["slots"] is not None else torch.arange(s["batch"], device="cuda")
    held = s["h"][slots] if s["h"] is not None else torch.zeros((s["batch"], D, N), device="cuda")
    first = place == 0
    b[first] += a[first] * held[seq[first]]
    a[first] = 0.0
    # a scan by doubling: after a pass of width w every row holds the sum of the 2 w rows up to it
    w = 1
    while w < s["longest"]:
        b[w:] += a[w:] * b[:-w]
        a[w:] *= a[:-w].clone()
        w *= 2
    y = torch.einsum("mgpn,mgqn->mgp", b.view(-1, G, per, N), Cm).reshape(-1, D) + s["Dskip"] * x
    if s["z"] is not None:
        z = s["z"].float()
        y = y * (z / (1 + torch.exp(-z)))
    out = held
    some = off[1:] > off[:-1]
    out[some] = b[off[1:][some] - 1]
    h_out = torch.zeros_like(out)
    h_out[slots] = out
    return y.to(s["x"].dtype), h_out


def work(case):
    c = case
    e = _SIZE[c["dtype"]]
    if c["kind"] == "lora":
        used = min(c["adapters"], c["requests"])
        return {"bytes": e * (c["rows"] * c["K"] + c["K"] * c["N"] + used * c["rank"] * (c["K"] + c["N"])) + _SIZE[c["out"]] * c["rows"] * c["N"]
                + 4 * (c["rows"] + c["N"] + c["adapters"]),
                "flops": 2 * c["rows"] * (c["K"] * c["N"] + c["rank"] * (c["K"] + c["N"]))}
    if c["kind"] == "conv":
        states = c["batch"] * (c["K"] - 1) * c["D"] * (2 if c["carry"] else 1)
        return {"bytes": e * (2 * c["rows"] * c["D"] + states + c["D"] * (c["K"] + 1)), "flops": c["rows"] * c["D"] * (2 * c["K"] + 4)}
    states = c["batch"] * c["D"] * c["N"] * (2 if c["carry"] else 1)
    return {"bytes": e * c["rows"] * (c["D"] * (4 if c["gate"] else 3) + 2 * c["groups"] * c["N"]) + 4 * (states + c["D"] * (c["N"] + 2)),
            "flops": c["rows"] * c["D"] * (7 * c["N"] + 12)}


def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "lora":
        X = s["X"].double()
        W = s["W"].double()
        Y = X.matmul(W.T if s["packed"] else W).add_(s["bias"].double())
        for a in range(s["adapters"]):
            mine = (s["adapter"] == a).nonzero().flatten()
            Y[mine] += s["scale"][a].double() * X[mine].matmul(s["A"][a].double().T).matmul(s["B"][a].double().T)
        return Y
    starts = s["offsets"][:-1].long()
    lengths = s["lengths"].cuda()
    slots = torch.arange(s["batch"], device="cuda") if s["slots"] is None else s["slots"].long()
    x = s["x"].double()
    if s["kind"] == "conv":
        K, w = s["K"], s["w"].double()
        held = s["state"].double()[slots] if s["state"] is not None else x.new_zeros((s["batch"], K - 1, s["D"]))

        def at(seq, place):
            """The input at a place of its list, where the places before the first are those of the state."""
            before = (place < 0)[:, None]
            return torch.where(before, held[seq, (place + K - 1).clamp(0, K - 2)], x[(starts[seq] + place).clamp(0, s["rows"] - 1)])
        seq = torch.repeat_interleave(torch.arange(s["batch"], device="cuda"), lengths)
        place = torch.arange(s["rows"], device="cuda") - starts[seq]
        v = s["b"].double() + torch.zeros_like(x)
        for back in range(K):
            v += w[:, K - 1 - back] * at(seq, place - back)
        out = torch.zeros_like(held)
        every = torch.arange(s["batch"], device="cuda")
        out[slots] = torch.stack([at(every, lengths - back) for back in range(K - 1, 0, -1)], 1)
        return v * torch.sigmoid(v), out
    # position t of every list that has one, one after the other
    y = torch.zeros_like(x)
    order = torch.argsort(lengths, descending=True)
    longer = (s["batch"] - torch.bincount(s["lengths"], minlength=s["longest"] + 1).cumsum(0)).tolist()
    h = s["h"].double()[slots] if s["h"] is not None else torch.zeros((s["batch"], s["D"], s["N"]), dtype=torch.float64, device="cuda")
    group = torch.arange(s["D"], device="cuda") // (s["D"] // s["groups"])
    delta = torch.nn.functional.softplus(s["delta"].double() + s["delta_bias"].double())
    A, skip = s["A"].double(), s["Dskip"].double()
    Bm, Cm = (s[k].double().view(-1, s["groups"], s["N"]) for k in "BC")
    for t in range(s["longest"]):
        i = order[:longer[t]]
        r = starts[i] + t
        dt = delta[r][:, :, None]
        h[i] = torch.exp(dt * A) * h[i] + dt * Bm[r][:, group] * x[r][:, :, None]
        y[r] = (Cm[r][:, group] * h[i]).sum(2) + skip * x[r]
    if s["z"] is not None:
        z = s["z"].double()
        y *= z * torch.sigmoid(z)
    out = torch.zeros_like(h)
    out[slots] = h
    return y, out
