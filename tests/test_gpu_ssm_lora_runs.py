"""The state-space block's operators together, as a server uses them: whole lists, then one behaviour after the other on kept states,
with the adapters of several scenes; captured and replayed, on streams of their own, several at once."""
import numpy as np
import pytest
import torch

import pkg
import ssm_oracle

pytestmark = pytest.mark.gpu


def _ops():
    pkg.load()
    from x_deeplearning_b200 import capi, ops
    return ops, capi


def _np(t):
    return t.detach().double().cpu().numpy()


class Block:
    """in-projection (adapters) -> convolution -> projections of its result -> scan with the gate -> out-projection (adapters)"""

    def __init__(self, rng, width, D, N, rank, scenes, dtype, K=4, step_rank=8):
        f = lambda *s, std=1.0: torch.from_numpy(rng.normal(0, std, s).astype(np.float32)).cuda()
        h = lambda *s, std=1.0: f(*s, std=std).to(dtype)
        self.width, self.D, self.N, self.step_rank, self.dtype = width, D, N, step_rank, dtype
        self.w_in, self.a_in, self.b_in = h(2 * D, width, std=width ** -0.5), h(scenes, rank, width, std=width ** -0.5), h(scenes, 2 * D, rank, std=0.3 * rank ** -0.5)
        self.conv_w, self.conv_b = h(D, K, std=0.5), h(D, std=0.1)
        self.w_x = h(step_rank + 2 * N, D, std=D ** -0.5)
        self.w_dt = h(D, step_rank, std=step_rank ** -0.5)
        step = np.exp(rng.uniform(np.log(1e-3), np.log(1e-1), D))
        self.dt_bias = torch.from_numpy((step + np.log(-np.expm1(-step))).astype(np.float32)).cuda()
        self.A = -torch.arange(1, N + 1, device="cuda", dtype=torch.float32).repeat(D, 1).contiguous()
        self.skip = torch.ones(D, device="cuda")
        self.w_out, self.a_out, self.b_out = h(width, D, std=D ** -0.5), h(scenes, rank, D, std=D ** -0.5), h(scenes, width, rank, std=0.3 * rank ** -0.5)
        self.scale = torch.from_numpy(rng.uniform(0.5, 1.5, scenes).astype(np.float32)).cuda()

    def __call__(self, ops, x, scene, conv, h, slots=None, longest=0, **lists):
        D, N, r = self.D, self.N, self.step_rank
        xz = ops.lora_gemm(x, self.w_in, self.a_in, self.b_in, scene, scale=self.scale, trans_b=True)
        u = ops.ssm_conv(xz[:, :D], self.conv_w, self.conv_b, state_in=conv, state_out=conv, slots=slots, **lists)
        p = ops.gemm(u, self.w_x, trans_b=True)
        delta = ops.gemm(p[:, :r], self.w_dt, trans_b=True)
        y = ops.ssm_scan(u, delta, self.A, p[:, r:r + N], p[:, r + N:], D=self.skip, z=xz[:, D:], delta_bias=self.dt_bias, h_in=h, h_out=h,
                         slots=slots, longest=longest, **lists)
        return ops.lora_gemm(y, self.w_out, self.a_out, self.b_out, scene, scale=self.scale, trans_b=True)

    def exact(self, x, scene, lists):
        """In 64 bits, every list from zeros; what each operator rounds to its type is not."""
        D, N, r = self.D, self.N, self.step_rank
        n = {k: _np(v) for k, v in self.__dict__.items() if isinstance(v, torch.Tensor)}
        sig = lambda v: 1 / (1 + np.exp(-v))

        def lora(v, w, a, b):
            out = v @ w.T
            for s in range(len(a)):
                m = scene == s
                out[m] += n["scale"][s] * (v[m] @ a[s].T) @ b[s].T
            return out
        xz = lora(x, n["w_in"], n["a_in"], n["b_in"])
        u, y = np.empty((len(x), D)), np.empty((len(x), D))
        for a, b in lists:
            ahead = np.concatenate([np.zeros((3, D)), xz[a:b, :D]])
            v = sum(ahead[j:j + b - a] * n["conv_w"][:, j] for j in range(4)) + n["conv_b"]
            u[a:b] = v * sig(v)
        p = u @ n["w_x"].T
        d = np.logaddexp(0, p[:, :r] @ n["w_dt"].T + n["dt_bias"])
        for a, b in lists:
            h = np.zeros((D, N))
            for t in range(a, b):
                h = np.exp(d[t][:, None] * n["A"]) * h + (d[t] * u[t])[:, None] * p[t, r:r + N]
                y[t] = (h * p[t, r + N:]).sum(1) + n["skip"] * u[t]
        z = xz[:, D:]
        return lora(y * z * sig(z), n["w_out"], n["a_out"], n["b_out"])


def _lists(lengths):
    off = np.concatenate([[0], np.cumsum(lengths)])
    return [(int(off[i]), int(off[i + 1])) for i in range(len(lengths))], torch.from_numpy(off.astype(np.int32)).cuda()


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-5), (torch.float16, 2e-2), (torch.bfloat16, 1.2e-1)], ids=["f32", "f16", "bf16"])
def test_block_whole_and_row_by_row(dtype, tol):
    """fp32: the rounding of sums of at most 72 products and 60 steps, 1e-6 of the magnitudes, through five operators. 16 bits: six roundings of
    half a step each on the way (2^-11, 2^-8), which the gate, the quadratic C h and the projections widen about fivefold."""
    ops, capi = _ops()
    rng = np.random.default_rng(21)
    width, D, N = 36, 72, 16
    block = Block(rng, width, D, N, 8, 5, dtype)
    lengths = [60, 1, 0, 17, 33, 60, 4]
    lists, off = _lists(lengths)
    rows, n = sum(lengths), len(lengths)
    x = torch.from_numpy(rng.normal(0, 1, (rows, width)).astype(np.float32)).cuda().to(dtype)
    per_list = torch.from_numpy(rng.integers(-1, 5, n).astype(np.int32)).cuda()
    scene = torch.repeat_interleave(per_list, torch.tensor(lengths, device="cuda")).to(torch.int32)
    want = block.exact(_np(x), scene.cpu().numpy(), lists)
    zeros = lambda: (torch.zeros(n + 2, 3, D, dtype=dtype, device="cuda"), torch.zeros(n + 2, D, N, device="cuda"))
    slots = torch.from_numpy(rng.permutation(n + 2)[:n].astype(np.int32)).cuda()
    conv, h = zeros()
    got = block(ops, x, scene, conv, h, slots, offsets=off, longest=60)
    rms = np.sqrt((want ** 2).mean())
    assert np.abs(_np(got) - want).max() <= tol * rms * 5 and np.sqrt(((_np(got) - want) ** 2).mean()) <= tol * rms
    # the same lists, all but their last rows at once and those one by one: the lists that are still running are the batch
    c2, h2 = zeros()
    cut = [max(k - 5, 0) for k in lengths]
    head = torch.cat([torch.arange(a, a + c) for (a, _), c in zip(lists, cut)]).cuda()
    _, off2 = _lists(cut)
    out = torch.empty_like(got)
    out[head] = block(ops, x[head].contiguous(), scene[head].contiguous(), c2, h2, slots, offsets=off2)
    for step in range(5):
        run = [i for i in range(n) if cut[i] + step < lengths[i]]
        at = torch.tensor([lists[i][0] + cut[i] + step for i in run], device="cuda")
        out[at] = block(ops, x[at].contiguous(), scene[at].contiguous(), c2, h2, slots[run].contiguous(), T=1)
    assert np.abs(_np(out) - want).max() <= tol * rms * 5
    # kept states agree with those of the whole lists
    used = slots.long()
    assert np.abs(_np(h2[used]) - _np(h[used])).max() <= tol * 5 * max(1.0, np.abs(_np(h[used])).max())


def _calls(rng):
    """One call of each operator and plan on inputs of its own: name -> a function that makes its outputs anew."""
    ops, capi = _ops()
    f = lambda *s, std=1.0: torch.from_numpy(rng.normal(0, std, s).astype(np.float32)).cuda()
    made = {}

    def scan(name, lengths, D, N, dtype, equal=False):
        rows, n = sum(lengths), len(lengths)
        _, off = _lists(lengths)
        x, d, z = (f(rows, D).to(dtype) for _ in range(3))
        B, C = f(rows, N).to(dtype), f(rows, N).to(dtype)
        A, h = -torch.rand(D, N, device="cuda") * 4 - 0.1, f(n, D, N, std=0.3)
        kw = dict(T=lengths[0]) if equal else dict(offsets=off, longest=max(lengths))

        def call():
            state = h.clone()
            return ops.ssm_scan(x, d, A, B, C, z=z, h_in=state, h_out=state, **kw), state
        made[name] = call
    scan("single rows", [1] * 50, 72, 16, torch.float16, True)
    scan("whole lists", [100] * 20, 72, 16, torch.bfloat16, True)
    scan("long ones first", [int(k) for k in rng.integers(0, 41, 900)] + [400], 40, 16, torch.float32)
    scan("chunks", [5000, 3, 0, 2000], 40, 16, torch.float32)
    x, w, st = f(700, 72).half(), f(72, 4).half(), f(9, 3, 72).half()
    off = torch.tensor([0, 0, 5, 300, 301, 302, 600, 640, 699, 700], dtype=torch.int32, device="cuda")

    def conv():
        state = st.clone()
        return ops.ssm_conv(x, w, offsets=off, state_in=state, state_out=state), state
    made["convolution"] = conv

    def lora(name, M, K, N, n, r, dtype, pad=0, out=None):
        X, W = f(M, K + pad).to(dtype)[:, :K], f(N, K + pad, std=K ** -0.5).to(dtype)[:, :K]
        A, B = f(n, r, K + pad, std=K ** -0.5).to(dtype)[:, :, :K], f(n, N, r).to(dtype)
        ad = torch.from_numpy(np.sort(rng.integers(-1, n, M)).astype(np.int32)).cuda()
        made[name] = lambda: (ops.lora_gemm(X, W, A, B, ad, trans_b=True, out_dtype=out),)
    lora("adapters, few rows", 40, 1280, 96, 40, 16, torch.float16)
    lora("adapters, few odd rows", 40, 250, 96, 40, 16, torch.float16, pad=1, out=torch.float32)
    lora("adapters, two steps", 2000, 328, 512, 9, 8, torch.bfloat16)
    lora("adapters, one step", 9600, 328, 200, 9, 8, torch.float16)
    lora("adapters, odd rows", 1000, 250, 131, 5, 12, torch.bfloat16, pad=1)
    lora("adapters, fp32", 300, 250, 131, 5, 12, torch.float32)
    return made


def test_captured_and_replayed():
    """Every plan in a graph of its own, and all in one; replayed while the others' workspaces come and go, and eager calls between."""
    calls = _calls(np.random.default_rng(22))
    want = {k: [t.clone() for t in c()] for k, c in calls.items()}
    torch.cuda.synchronize()
    graphs = {}
    for k, c in calls.items():
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = c()
        graphs[k] = (g, out)
    one = torch.cuda.CUDAGraph()
    with torch.cuda.graph(one):
        outs = {k: c() for k, c in calls.items()}
    for _ in range(3):
        for g, _ in graphs.values():
            g.replay()
        one.replay()
        for c in calls.values():
            c()
    torch.cuda.synchronize()
    for k in calls:
        for w, a, b in zip(want[k], graphs[k][1], outs[k]):
            assert torch.equal(w, a) and torch.equal(w, b), k


def test_on_streams_at_once():
    """The same calls on four streams without order between them: the same bits each time."""
    calls = _calls(np.random.default_rng(23))
    want = {k: [t.clone() for t in c()] for k, c in calls.items()}
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    got = []
    for turn in range(4):
        for i, (k, c) in enumerate(calls.items()):
            with torch.cuda.stream(streams[(i + turn) % 4]):
                got.append((k, c()))
    torch.cuda.synchronize()
    for k, out in got:
        assert all(torch.equal(w, g) for w, g in zip(want[k], out)), k


def test_a_callers_workspace():
    ops, capi = _ops()
    rng = np.random.default_rng(24)
    f = lambda *s: torch.from_numpy(rng.normal(0, 1, s).astype(np.float32)).cuda()
    x, d, B, C, A = f(6000, 24), f(6000, 24), f(6000, 16), f(6000, 16), -torch.rand(24, 16, device="cuda")
    want = ops.ssm_scan(x, d, A, B, C)
    ws = torch.full((1 << 24,), 255, dtype=torch.uint8, device="cuda")            # what it holds does not matter
    assert torch.equal(ops.ssm_scan(x, d, A, B, C, workspace=ws), want)
    with pytest.raises(capi.XbError, match="workspace"):
        ops.ssm_scan(x, d, A, B, C, workspace=ws[:64])
    X, W, a, b = f(1500, 64).half(), f(300, 64).half(), f(3, 8, 64).half(), f(3, 300, 8).half()
    ad = torch.from_numpy(rng.integers(-1, 3, 1500).astype(np.int32)).cuda()
    want = ops.lora_gemm(X, W, a, b, ad, trans_b=True)
    ws.fill_(255)
    assert torch.equal(ops.lora_gemm(X, W, a, b, ad, trans_b=True, workspace=ws), want)


def test_no_wait_ran_out():
    ops, capi = _ops()
    for c in _calls(np.random.default_rng(25)).values():
        c()
    torch.cuda.synchronize()
    assert ops.device_status() == 0
