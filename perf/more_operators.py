"""Attention over behaviour lists as users give it work: a fixed list of timed cases and a generator of more of them.

Three kinds, each one call of the library's public entry points:
  rope   norms of queries and keys for each head and the position rotation (ops.qk_norm_rope)
  lin    linear attention with a decay for each head (ops.linear_attention), whole lists or one new behaviour a user
  att    softmax attention of lists that share a prefix (ops.prefix_attention): the candidates of a request against the user's kept
         behaviours and their own rows

The plain forms below are elementary torch operations in 32 bits, rounded once at the end.
"""
import math

import torch

own = False

_T = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"f16": 2, "bf16": 2, "f32": 4}
_ROPE_MOST = 70_000 * 16 * 128      # values of the largest listed case
_LIN_MOST = 70_000 * 8 * 128        # rows x heads x (dk + dv)
_STATES_MOST = 2048 * 8 * 64 * 64
_ATT_FLOPS = 4 * 128 * 512 * 4 * 100_003
_ATT_BYTES = 4 * 128 * 8 * 108_800


def listed():
    return [
        # one new behaviour each of four users: the latency of a single token
        dict(name="rope_step", kind="rope", rows=4, Hq=8, Hk=2, d=64, rot=64, dtype="f16", fused=True, norm=True, adjacent=False),
        # packed behaviour lists in bulk, sliced from one projection of queries, keys and values
        dict(name="rope_bulk", kind="rope", rows=70_000, Hq=8, Hk=8, d=128, rot=128, dtype="bf16", fused=True, norm=True, adjacent=False),
        # one new behaviour each of four users: the latency of a single token
        dict(name="lin_step_small", kind="lin", rows=4, batch=4, ragged=False, H=4, Hkv=4, dk=64, dv=64, dtype="f16", carry=True),
        # one new behaviour of every active user: the states' traffic
        dict(name="lin_step_bulk", kind="lin", rows=2048, batch=2048, ragged=False, H=8, Hkv=8, dk=64, dv=64, dtype="bf16", carry=True),
        # the headline batch's behaviour lists, 74 requests of 100 steps, heads of the recurrent extractor's width, in fp32
        dict(name="lin_history", kind="lin", rows=7400, batch=74, ragged=False, H=2, Hkv=2, dk=36, dv=36, dtype="f32", carry=False),
        # lists of every length packed one after the other, some continued from kept states
        dict(name="lin_ragged", kind="lin", rows=70_000, batch=256, ragged=True, H=8, Hkv=8, dk=64, dv=64, dtype="bf16", carry=True),
        # one life-long list, wide heads that share keys and values in pairs
        dict(name="lin_long", kind="lin", rows=30_011, batch=1, ragged=True, H=8, Hkv=4, dk=128, dv=128, dtype="f16", carry=True),
        # one request, four branches of a few rows on a kept list: the latency of a single token
        dict(name="att_step_small", kind="att", mode="step", groups=1, lists=4, own=16, prefix=1000, ragged=False, H=8, Hkv=2, d=64, dtype="f16"),
        # the headline batch: 74 requests of 1000 candidates, each against the user's 100 behaviours and itself
        dict(name="att_candidates", kind="att", mode="step", groups=74, lists=74_000, own=1, prefix=100, ragged=False, H=4, Hkv=4, d=64, dtype="f16"),
        # 512 candidates of one request against a life-long list, the compute-bound case
        dict(name="att_life", kind="att", mode="step", groups=1, lists=512, own=1, prefix=100_003, ragged=False, H=4, Hkv=4, d=128, dtype="bf16"),
        # one new row of each of 256 branches of every length on eight kept lists of every length, keys shared by four heads
        dict(name="att_step_ragged", kind="att", mode="step", groups=8, lists=256, own=300, prefix=4000, ragged=True, H=32, Hkv=8, d=128, dtype="bf16"),
        # whole branches of every length on kept lists of every length
        dict(name="att_whole", kind="att", mode="whole", groups=16, lists=64, own=500, prefix=1000, ragged=True, H=8, Hkv=8, d=64, dtype="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi, unit):
    """A head's width: mostly whole pieces of 8."""
    w = _log(rng, lo, hi)
    return (w + 7) // 8 * 8 if rng.random() < 0.7 else (w + unit - 1) // unit * unit


def draw(rng):
    kind = rng.choice(["rope", "lin", "lin", "att", "att"])
    if kind == "rope":
        while True:
            rows, Hq, d = _log(rng, 1, 70_000), _log(rng, 1, 32), _width(rng, 16, 256, 2)
            Hk = rng.choice([h for h in range(0, Hq + 1) if h == 0 or Hq % h == 0])
            if rows * (Hq + Hk) * d <= _ROPE_MOST:
                break
        return dict(kind=kind, rows=rows, Hq=Hq, Hk=Hk, d=d, rot=d if rng.random() < 0.6 else rng.randrange(1, d // 2 + 1) * 2,
                    dtype=rng.choice(["f16", "bf16", "f32"]), fused=rng.random() < 0.6, norm=rng.random() < 0.8, adjacent=rng.random() < 0.3)
    if kind == "lin":
        step, cut = rng.random() < 0.35, rng.random() < 0.2         # single tokens; lists that were cut to one length
        while True:
            H, dk, dv = rng.choice([1, 2, 3, 4, 6, 8, 16]), _width(rng, 16, 128, 1), _width(rng, 16, 128, 1)
            Hkv = rng.choice([h for h in range(1, H + 1) if H % h == 0])
            batch = _log(rng, 1, 4096) if step else _log(rng, 1, 512)
            rows = batch if step else _log(rng, max(batch // 2, 1), 70_000)
            if cut and not step:
                rows = max(rows // batch, 1) * batch
            if rows * H * (dk + dv) <= _LIN_MOST and batch * H * dk * dv <= _STATES_MOST:
                return dict(kind=kind, rows=rows, batch=batch, ragged=not (step or cut), H=H, Hkv=Hkv, dk=dk, dv=dv,
                            dtype=rng.choice(["f16", "bf16", "f32"]), carry=rng.random() < 0.6)
    while True:
        Hkv, share, d = rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 2, 3, 4, 8]), (_log(rng, 16, 128) + 7) // 8 * 8
        groups = _log(rng, 1, 128)
        whole = rng.random() < 0.4
        lists = groups * _log(rng, 1, 8 if whole else 1000)
        c = dict(kind=kind, mode="whole" if whole else "step", groups=groups, lists=lists, own=_log(rng, 1, 2000 if whole else 500),
                 prefix=rng.choice([0, 1, 1, 1, 1, 1]) * _log(rng, 1, 100_000), ragged=rng.random() < 0.7, H=Hkv * share, Hkv=Hkv, d=d,
                 dtype=rng.choice(["f16", "bf16"]))
        rows = lists * c["own"] if whole else lists
        keys = lists * c["own"] + groups * c["prefix"]
        # what a list sees, where a ragged one may be several times the mean
        flops = 4 * d * c["H"] * rows * (c["prefix"] + c["own"]) * (3 if c["ragged"] else 1)
        bytes_ = 4 * d * (Hkv * keys + c["H"] * rows)
        if flops <= _ATT_FLOPS and bytes_ <= _ATT_BYTES and rows * c["H"] // groups * (c["prefix"] + lists // groups * c["own"]) * 3 <= 1 << 30:
            return c


def _lengths(rows, batch, seed, least=0):
    """`batch` lengths that add up to `rows`: mostly of the mean's order, some long, some empty (or of `least`)."""
    g = torch.Generator().manual_seed(seed)
    w = torch.empty(batch, dtype=torch.float64).exponential_(1.0, generator=g) + 1e-3
    ends = (w.cumsum(0) / w.sum() * (rows - batch * least)).floor().to(torch.int64)
    ends[-1] = rows - batch * least
    return torch.diff(ends, prepend=torch.zeros(1, dtype=torch.int64)) + least


def _offsets(lengths):
    o = torch.zeros(len(lengths) + 1, dtype=torch.int64)
    o[1:] = lengths.cumsum(0)
    return o


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _T[c["dtype"]]

    def normal(*shape, mean=0.0, std=1.0, to=torch.float32):
        return (torch.randn(shape, device="cuda", generator=gen) * std + mean).to(to)

    s = dict(c)
    if c["kind"] == "rope":
        rows, Hq, Hk, d = c["rows"], c["Hq"], c["Hk"], c["d"]
        if c["fused"]:                  # slices of one projection, whose last part are the values
            qkv = normal(rows, Hq + 2 * Hk, d, std=1.5, to=dt)
            s["q"], s["k"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hk] if Hk else None
        else:
            s["q"], s["k"] = normal(rows, Hq, d, std=1.5, to=dt), normal(rows, Hk, d, std=1.5, to=dt) if Hk else None
        s["wq"], s["wk"] = (normal(d, mean=1.0, std=0.1), normal(d, mean=1.0, std=0.1)) if c["norm"] else (None, None)
        s["freqs"] = torch.exp(torch.arange(c["rot"] // 2, dtype=torch.float64) * (-math.log(10000.0) / (c["rot"] // 2))).float().cuda()
        # places in lists that go on from kept ones
        s["positions"] = (torch.arange(rows, device="cuda") % 1000 + torch.randint(0, 200_000, (rows,), device="cuda", generator=gen)).to(torch.int32)
        return s
    if c["kind"] == "lin":
        rows, batch, H, dk, dv = c["rows"], c["batch"], c["H"], c["dk"], c["dv"]
        lengths = _lengths(rows, batch, seed) if c["ragged"] else torch.full((batch,), rows // batch)
        s["equal"] = int(lengths[0]) if bool((lengths == lengths[0]).all()) else 0
        s["longest"] = int(lengths.max())
        s["offsets"] = _offsets(lengths).to(device="cuda", dtype=torch.int32)
        s["lengths"] = lengths
        # users lie anywhere in the table of kept states
        s["slots"] = torch.randperm(batch, device="cuda", generator=gen).to(torch.int32) if c["carry"] else None
        s["q"], s["k"], s["v"] = normal(rows, H, dk, to=dt), normal(rows, c["Hkv"], dk, to=dt), normal(rows, c["Hkv"], dv, to=dt)
        # decays of 1 - 1/16 to 1 - 1/1024 over the heads
        s["log_decay"] = torch.log1p(-torch.exp2(-4 - 6 * torch.arange(H, dtype=torch.float64) / max(H - 1, 1))).float().cuda()
        s["scale"] = dk ** -0.5
        s["h"] = normal(batch, H, dk, dv) if c["carry"] else None
        s["h_out"] = torch.zeros((batch, H, dk, dv), device="cuda")
        return s
    groups, lists, H, Hkv, d = c["groups"], c["lists"], c["H"], c["Hkv"], c["d"]
    each = _lengths(lists, groups, seed, 1 if lists >= groups else 0) if c["ragged"] else torch.full((groups,), lists // groups)
    members = _offsets(each)
    own_len = _lengths(lists * c["own"], lists, seed + 1, 1) if c["ragged"] else torch.full((lists,), c["own"])
    prefix_len = _lengths(groups * c["prefix"], groups, seed + 2) if c["ragged"] else torch.full((groups,), c["prefix"])
    own_off, prefix_off = _offsets(own_len), _offsets(prefix_len)
    rows = int(own_off[-1]) if c["mode"] == "whole" else lists
    s["rows_at"] = (own_off if c["mode"] == "whole" else torch.arange(lists + 1)).tolist()
    s["own_at"], s["prefix_at"], s["members_at"] = own_off.tolist(), prefix_off.tolist(), members.tolist()
    to = lambda t: t.to(device="cuda", dtype=torch.int32)
    s["own_off"], s["prefix_off"], s["members"] = to(own_off), to(prefix_off), to(members)
    s["q"] = normal(rows, H, d, to=dt)
    s["k"], s["v"] = normal(int(own_off[-1]), Hkv, d, to=dt), normal(int(own_off[-1]), Hkv, d, to=dt)
    s["pk"], s["pv"] = (normal(int(prefix_off[-1]), Hkv, d, to=dt), normal(int(prefix_off[-1]), Hkv, d, to=dt)) if c["prefix"] else (None, None)
    s["scale"] = d ** -0.5
    return s


def _ops():
    from __graft_entry__ import load_package
    load_package()
    from x_deeplearning_b200 import ops
    return ops


def run(s):
    if own:
        ops = _ops()
        if s["kind"] == "rope":
            return ops.qk_norm_rope(s["q"], s["k"], s["positions"], s["freqs"], q_weight=s["wq"],
                                    k_weight=s["wk"] if s["k"] is not None else None, norm=s["norm"],
                                    adjacent=s["adjacent"])
        if s["kind"] == "lin":
            lists = dict(T=s["equal"]) if s["equal"] else dict(offsets=s["offsets"])
            y = ops.linear_attention(s["q"], s["k"], s["v"], s["log_decay"], scale=s["scale"], h_in=s["h"], h_out=s["h_out"], slots=s["slots"],
                                     longest=s["longest"], **lists)
            return y, s["h_out"]
        lists = dict(offsets=s["own_off"]) if s["mode"] == "whole" else dict(T=1, own_offsets=s["own_off"])
        if s["pk"] is not None:
            lists.update(prefix_k=s["pk"], prefix_v=s["pv"], prefix_offsets=s["prefix_off"], members=s["members"])
        return ops.prefix_attention(s["q"], s["k"], s["v"], scale=s["scale"], **lists)
    return {"rope": _plain_rope, "lin": _plain_lin, "att": _plain_att}[s["kind"]](s)


def _plain_rope(s):
    def one(x, w):
        if x is None:
            return None
        t, half = x.float(), s["rot"] // 2
        if s["norm"]:
            t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * w
        angle = s["positions"].double()[:, None] * s["freqs"].double()
        cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
        a, b = (t[..., 0:s["rot"]:2], t[..., 1:s["rot"]:2]) if s["adjacent"] else (t[..., :half], t[..., half:s["rot"]])
        first, second = a * cos - b * sin, b * cos + a * sin
        turned = torch.stack([first, second], -1).flatten(-2) if s["adjacent"] else torch.cat([first, second], -1)
        return torch.cat([turned, t[..., s["rot"]:]], -1).to(x.dtype)
    return one(s["q"], s["wq"]), one(s["k"], s["wk"])


def _plain_lin(s):
    H, dk, dv, batch = s["H"], s["dk"], s["dv"], s["batch"]
    share = H // s["Hkv"]
    off = s["offsets"].long()
    slots = s["slots"].long() if s["slots"] is not None else torch.arange(batch, device="cuda")
    h = s["h"][slots] if s["h"] is not None else torch.zeros((batch, H, dk, dv), device="cuda")
    y = torch.zeros((s["rows"], H, dv), device="cuda")
    ld = s["log_decay"].double()
    C = min(128, s["longest"])          # rows of every list at a time, from the state that they begin with
    place = torch.arange(C, device="cuda")
    back = place[:, None] - place
    D = torch.where(back >= 0, torch.exp(back.clamp(min=0) * ld[:, None, None]), 0.0).float()
    into = torch.exp((place + 1) * ld[:, None]).float()
    for t in range(0, s["longest"], C):
        at = off[:-1, None] + t + place
        there = at < off[1:, None]
        r = at.clamp(max=s["rows"] - 1)
        q = s["q"][r].float().transpose(1, 2)
        k, v = ((s[n][r].float() * there[:, :, None, None]).transpose(1, 2).repeat_interleave(share, 1) for n in "kv")
        o = (torch.matmul(q, k.transpose(2, 3)) * D) @ v + into[:, :, None] * torch.matmul(q, h)
        y[r[there]] = (o * s["scale"]).transpose(1, 2)[there]
        n = there.sum(1)                # the state moves on by the rows that the list still has
        left = (n[:, None] - 1 - place).clamp(min=0)
        w = torch.exp(left[:, None] * ld[:, None]).float()
        h = torch.exp(n[:, None] * ld).float()[:, :, None, None] * h + torch.matmul((k * w[:, :, :, None]).transpose(2, 3), v)
    h_out = torch.zeros_like(h)
    h_out[slots] = h
    return y.to(s["q"].dtype), h_out


def _plain_att(s):
    share = s["H"] // s["Hkv"]
    y = torch.zeros(s["q"].shape, device="cuda")
    own_off, rows_off = s["own_off"].long(), torch.tensor(s["rows_at"], device="cuda")

    def heads(t):
        return t.float().transpose(0, 1).repeat_interleave(share, 0)
    for g in range(s["groups"]):
        l0, l1 = s["members_at"][g], s["members_at"][g + 1]
        r0, r1, k0, k1 = s["rows_at"][l0], s["rows_at"][l1], s["own_at"][l0], s["own_at"][l1]
        if r0 == r1:
            continue
        q = s["q"][r0:r1].float().transpose(0, 1)
        k, v = heads(s["k"][k0:k1]), heads(s["v"][k0:k1])
        # the own keys of a row's list, up to the row's place counted from the end
        row = torch.arange(r0, r1, device="cuda")
        mine = torch.searchsorted(rows_off[1:].contiguous(), row, right=True)
        last = own_off[mine + 1] - (rows_off[mine + 1] - row)
        key = torch.arange(k0, k1, device="cuda")
        seen = (key >= own_off[mine][:, None]) & (key <= last[:, None])
        score = (torch.matmul(q, k.transpose(1, 2)) * s["scale"]).masked_fill(~seen, float("-inf"))
        if s["pk"] is not None:
            p0, p1 = s["prefix_at"][g], s["prefix_at"][g + 1]
            score = torch.cat([torch.matmul(q, heads(s["pk"][p0:p1]).transpose(1, 2)) * s["scale"], score], 2)
            v = torch.cat([heads(s["pv"][p0:p1]), v], 1)
        p = torch.exp(score - score.amax(2, keepdim=True))
        y[r0:r1] = (torch.matmul(p, v) / p.sum(2, keepdim=True)).transpose(0, 1)
    return y.to(s["q"].dtype)


def _lists_of(case):
    """(rows, own rows, pairs of a query row and a key that it sees) of an attention case, of mean lengths where they are ragged."""
    c = case
    own_rows = c["lists"] * c["own"]
    if c["mode"] == "whole":
        return own_rows, own_rows, own_rows * (c["prefix"] + (c["own"] + 1) / 2)
    return c["lists"], own_rows, c["lists"] * (c["prefix"] + c["own"])


def work(case):
    c = case
    e = _SIZE[c["dtype"]]
    if c["kind"] == "rope":
        values = c["rows"] * (c["Hq"] + c["Hk"]) * c["d"]
        return {"bytes": 2 * e * values + 4 * (c["rows"] + 2 * c["d"] + c["rot"] // 2), "flops": 8 * values}
    if c["kind"] == "lin":
        states = c["batch"] * c["H"] * c["dk"] * c["dv"] * (2 if c["carry"] else 1)
        return {"bytes": e * c["rows"] * (c["H"] + c["Hkv"]) * (c["dk"] + c["dv"]) + 4 * states, "flops": 4 * c["rows"] * c["H"] * c["dk"] * c["dv"]}
    rows, own_rows, pairs = _lists_of(c)
    keys = own_rows + c["groups"] * c["prefix"]
    return {"bytes": e * c["d"] * 2 * (rows * c["H"] + keys * c["Hkv"]) + 4 * (c["lists"] + 2 * c["groups"]), "flops": int(4 * c["d"] * c["H"] * pairs)}


def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "rope":
        theta = torch.outer(s["positions"].double(), s["freqs"].double())
        turn = torch.polar(torch.ones_like(theta), theta)[:, None]
        out = []
        for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
            if x is None:
                out.append(None)
                continue
            t = x.double()
            if s["norm"]:
                t = t * torch.rsqrt(t.square().mean(2, keepdim=True) + 1e-6) * w.double()
            j = torch.arange(s["rot"] // 2, device="cuda")
            i0, i1 = (2 * j, 2 * j + 1) if s["adjacent"] else (j, j + s["rot"] // 2)
            z = torch.complex(t[..., i0], t[..., i1]) * turn
            t = t.clone()
            t[..., i0], t[..., i1] = z.real, z.imag
            out.append(t)
        return tuple(out)
    if s["kind"] == "lin":
        # position t of every list that has one, one after the other
        starts, lengths = s["offsets"][:-1].long(), s["lengths"].cuda()
        slots = torch.arange(s["batch"], device="cuda") if s["slots"] is None else s["slots"].long()
        shape = (s["batch"], s["H"], s["dk"], s["dv"])
        h = s["h"].double()[slots] if s["h"] is not None else torch.zeros(shape, dtype=torch.float64, device="cuda")
        g = torch.exp(s["log_decay"].double())[:, None, None]
        reads = torch.arange(s["H"], device="cuda") // (s["H"] // s["Hkv"])
        y = torch.zeros((s["rows"], s["H"], s["dv"]), dtype=torch.float64, device="cuda")
        order = torch.argsort(lengths, descending=True)
        longer = (s["batch"] - torch.bincount(s["lengths"], minlength=s["longest"] + 1).cumsum(0)).tolist()
        h = h[order]
        for t in range(s["longest"]):
            n = longer[t]
            r = starts[order[:n]] + t
            h[:n].mul_(g).add_(s["k"][r].double()[:, reads, :, None] * s["v"][r].double()[:, reads, None, :])
            y[r] = (s["q"][r].double()[:, :, None, :] @ h[:n])[:, :, 0] * s["scale"]
        out = torch.zeros(shape, dtype=torch.float64, device="cuda")
        out[slots[order]] = h
        return y, out
    # the own keys of a row side by side, its list's first ones first
    rows = s["q"].shape[0]
    y = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    q = s["q"].double().unflatten(1, (s["Hkv"], -1)) * s["scale"]
    lengths = torch.diff(s["own_off"].long())
    queries = lengths if s["mode"] == "whole" else torch.ones_like(lengths)
    list_of = torch.repeat_interleave(torch.arange(s["lists"], device="cuda"), queries)
    first_row = (queries.cumsum(0) - queries)[list_of]
    begin = s["own_off"].long()[list_of]
    count = torch.arange(rows, device="cuda") - first_row + 1 + (lengths - queries)[list_of]
    group_of = torch.searchsorted(s["members"].long()[1:].contiguous(), list_of, right=True)
    for g in range(s["groups"]):
        mine = (group_of == g).nonzero().flatten()
        if s["pk"] is None:
            pk = pv = s["k"][:0].double()
        else:
            pk, pv = (s[n][s["prefix_at"][g]:s["prefix_at"][g + 1]].double() for n in ("pk", "pv"))
        while len(mine):
            # as many rows as take about 2^27 scores and gathered values together
            most = int(count[mine].max())
            n = max(1, min(len(mine), (1 << 27) // (s["H"] * (len(pk) + most) + 2 * most * s["Hkv"] * s["d"])))
            r, mine = mine[:n], mine[n:]
            far = torch.arange(int(count[r].max()), device="cuda")
            at = (begin[r][:, None] + far).clamp(max=len(s["k"]) - 1)
            k, v = s["k"][at].double(), s["v"][at].double()
            mixed = torch.cat([torch.einsum("rhgd,khd->rhgk", q[r], pk), torch.einsum("rhgd,rkhd->rhgk", q[r], k).masked_fill(
                (far >= count[r][:, None])[:, None, None], -math.inf)], 3).softmax(3)
            y[r] = (torch.einsum("rhgk,khd->rhgd", mixed[..., :len(pk)], pv) + torch.einsum("rhgk,rkhd->rhgd", mixed[..., len(pk):], v)).flatten(1, 2)
    return y
