"""torch-tensor front ends of the C-ABI calls, used by tests and bench.py.

torch is plumbing here (device memory, streams); every computation is a call
into libxdlb200.so. Nothing in this file computes on the CPU or with torch ops.
"""
import ctypes as C

import torch

from . import capi
from .capi import (XB_F16, XB_F32, XB_BF16, XB_I32, XB_I64, PoolGroup, TableDesc, DinAttArgs, binding, check, lib)

_DT = {torch.float32: XB_F32, torch.float16: XB_F16, torch.bfloat16: XB_BF16, torch.int32: XB_I32,
       torch.int64: XB_I64}


def dt(t):
    return _DT[t.dtype]


_raw_stream, _raw_device = getattr(torch._C, "_cuda_getCurrentRawStream", None), getattr(torch._C, "_cuda_getDevice", None)


def raw_stream():
    """The current stream of the current device as a number (torch.cuda.current_stream() makes an object of it: 3.4 us)."""
    if _raw_stream is None or _raw_device is None or not torch.cuda.is_initialized():
        return torch.cuda.current_stream().cuda_stream
    return _raw_stream(_raw_device())


def stream():
    return C.c_void_p(raw_stream())


def ptr(t):
    return C.c_void_p(t.data_ptr()) if t is not None else None


class Table:
    """An embedding table resident in HBM (xb_table_desc over torch-owned memory)."""

    def __init__(self, weights, dtype=torch.float16, keys=None, device="cuda"):
        # weights: CPU float32 [rows, dim]; keys: optional CPU int64 [rows]
        rows, dim = weights.shape
        self.rows, self.dim, self.dtype = rows, dim, dtype
        es = 2 if dtype == torch.float16 else 4
        pitch = int(lib().xb_table_row_pitch(dim, _DT[dtype]))
        self.pitch = pitch
        buf = torch.zeros((rows, pitch // es), dtype=dtype)
        buf[:, :dim] = weights.to(dtype)
        self.buf = buf.to(device)
        self.desc = TableDesc()
        self.desc.weights = self.buf.data_ptr()
        self.desc.rows, self.desc.dim, self.desc.dtype, self.desc.row_pitch_bytes = rows, dim, _DT[dtype], pitch
        self.slot_keys = self.slot_rows = None
        if keys is not None:
            slots = 16
            while slots < 2 * rows:
                slots <<= 1
            sk = torch.empty(slots, dtype=torch.int64)
            sr = torch.empty(slots, dtype=torch.int32)
            k = keys.contiguous().to(torch.int64)
            check(lib().xb_table_build_index_host(ptr(k), rows, slots, ptr(sk), ptr(sr)))
            self.slot_keys, self.slot_rows = sk.to(device), sr.to(device)
            self.desc.slot_keys, self.desc.slot_rows, self.desc.slots = (self.slot_keys.data_ptr(),
                                                                          self.slot_rows.data_ptr(), slots)


def make_group(table, ids, values, segments, items, out_dtype, segments_are_offsets=False, dim=None):
    """items: list of dict(udf, out (2-D tensor), col, trunc_dir, trunc_num, assign_stride)."""
    g = PoolGroup()
    g.table = C.pointer(table.desc) if table is not None else None
    g.ids, g.values, g.segments = ptr(ids), ptr(values), ptr(segments)
    g.n_ids = ids.numel()
    g.batch = segments.numel() - (1 if segments_are_offsets else 0)
    g.dim = table.dim if table is not None else dim
    g.id_dtype = dt(ids)
    g.segments_are_offsets = int(segments_are_offsets)
    g.out_dtype = _DT[out_dtype]
    g.n_items = len(items)
    g.values_dtype = dt(values) if values is not None else 0
    for k, it in enumerate(items):
        o = it["out"]
        assert o.dtype == out_dtype and o.dim() == 2 and o.stride(1) == 1
        g.items[k].udf = it["udf"]
        g.items[k].trunc_dir = it.get("trunc_dir", 1)
        g.items[k].trunc_num = it.get("trunc_num", 0)
        g.items[k].assign_stride = it.get("assign_stride", 0)
        g.items[k].out = o.data_ptr() + it.get("col", 0) * o.element_size()
        g.items[k].stride = o.stride(0)
    g._keep = (table, ids, values, segments, [it["out"] for it in items])
    return g


class PoolPlan:
    """A fixed set of pooling groups with its scratch buffer: one launch per 32 groups."""

    def __init__(self, groups, device="cuda"):
        self.groups = groups
        self.chunks = []
        for i in range(0, len(groups), capi.XB_MAX_POOL_GROUPS):
            part = groups[i:i + capi.XB_MAX_POOL_GROUPS]
            arr = (PoolGroup * len(part))(*part)
            need = int(lib().xb_embedding_pool_scratch_bytes(arr, len(part)))
            scratch = torch.empty(max(need, 16), dtype=torch.uint8, device=device)
            self.chunks.append((arr, len(part), scratch, need))
        # (addresses of what the plan itself owns)
        self._calls = [(C.addressof(arr), n, scratch.data_ptr(), need) for arr, n, scratch, need in self.chunks]
        self._pool = binding().pool

    def run(self):
        s = raw_stream()
        for arr, n, scratch, need in self._calls:
            check(self._pool(arr, n, scratch, need, s))


def embedding_pool(groups):
    PoolPlan(groups).run()


def gemm(A, B, Y=None, bias=None, trans_a=False, trans_b=False, alpha=1.0, beta=1.0, epilogue=0, ep=(None, None, None),
         ep_count=0, nosqrt=False, engine=0, out_dtype=None, batch=1, strides=(0, 0, 0, 0), M=None, N=None, K=None,
         lda=None, ldb=None, ldy=None, bias_kind=None, stride_ep=0, ldbias=None, bias_row_group=0):
    """2-D (or explicitly strided batched) GEMM through xb_gemm. Returns Y."""
    if M is None:
        M, K = (A.shape[-1], A.shape[-2]) if trans_a else (A.shape[-2], A.shape[-1])
        N = B.shape[-2] if trans_b else B.shape[-1]
    if Y is None:
        Y = torch.empty((batch, M, N) if batch > 1 else (M, N), dtype=out_dtype or A.dtype, device=A.device)
    # any indexable will do (a [3, N] tensor of activation parameters, an array of strides); the extension module takes tuples
    if type(ep) is not tuple:
        ep = (ep[0], ep[1], ep[2])
    if type(strides) is not tuple:
        strides = (strides[0], strides[1], strides[2], strides[3])
    global _gemm
    if _gemm is None:
        m = binding()
        m.dtypes(_DT)
        _gemm = m.gemm
    check(_gemm(A, B, Y, bias, trans_a, trans_b, alpha, beta, epilogue, ep, ep_count, nosqrt, engine, batch, strides, M, N, K,
                lda, ldb, ldy, bias_kind, stride_ep, ldbias, bias_row_group, raw_stream()))
    return Y


_gemm = None


def pack_weight_kmajor(W, out_dtype=torch.float16, ldk=None, batch=1):
    """W [K,N] (or [batch,K,N]) -> [N, ldk] K-major, zero padded."""
    K, N = W.shape[-2], W.shape[-1]
    ldk = ldk or (K + 7) // 8 * 8
    out = torch.empty((batch, N, ldk) if batch > 1 else (N, ldk), dtype=out_dtype, device=W.device)
    check(lib().xb_pack_weight_kmajor(ptr(W), dt(W), K, N, W.stride(-2), ptr(out), _DT[out_dtype], ldk, batch,
                                      K * W.stride(-2) if batch > 1 else 0, N * ldk if batch > 1 else 0, stream()))
    return out


class DinAttention:
    """Weights of one attention unit packed for xb_din_attention."""

    def __init__(self, W0, b0, W1, b1, W2, b2, dice0=None, dice1=None, act=capi.XB_ACT_DICE, device="cuda"):
        # W0 [4d,h0], W1 [h0,h1], W2 [h1,1] float32 CPU tensors (Blaze layout [K,N])
        f = lambda t: t.to(device=device, dtype=torch.float32).contiguous()
        self.W0 = W0.t().contiguous().to(device=device, dtype=torch.float16)
        self.W1 = W1.t().contiguous().to(device=device, dtype=torch.float16)
        self.W2 = f(W2.reshape(-1))
        self.b0, self.b1, self.b2 = f(b0), f(b1), float(b2)
        self.dice0 = [f(t) for t in dice0] if dice0 else None
        self.dice1 = [f(t) for t in dice1] if dice1 else None
        self.act = act
        self.h0, self.h1 = W0.shape[1], W1.shape[1]
        self.packed = None
        self.d = W0.shape[0] // 4

    def __call__(self, q, k, requests, n_cand, T, out=None, seq_len=None, use_softmax=False, scores=None, engine=0):
        d = q.shape[1]
        if out is None:
            out = torch.empty((requests * n_cand, d), dtype=torch.float16, device=q.device)
        a = DinAttArgs()
        a.q, a.ldq, a.k, a.ldk = q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0)
        a.seq_len, a.out, a.ldo, a.scores = ptr(seq_len), out.data_ptr(), out.stride(0), ptr(scores)
        a.requests, a.n_cand, a.T, a.d, a.h0, a.h1 = requests, n_cand, T, d, self.h0, self.h1
        a.act, a.use_softmax, a.engine = self.act, int(use_softmax), engine
        w = a.w
        w.W0, w.W1, w.W2, w.b0, w.b1, w.b2 = (self.W0.data_ptr(), self.W1.data_ptr(), self.W2.data_ptr(),
                                               self.b0.data_ptr(), self.b1.data_ptr(), self.b2)
        if self.dice0:
            w.gamma0, w.mean0, w.var0 = [t.data_ptr() for t in self.dice0]
            w.gamma1, w.mean1, w.var1 = [t.data_ptr() for t in self.dice1]
        if self.packed is None:
            # weights are constants: lay the operands out once
            n = int(lib().xb_din_attention_packed_bytes(d, self.h0, self.h1))
            self.packed = False
            if n:
                buf = torch.empty(n, dtype=torch.uint8, device=q.device)
                check(lib().xb_din_attention_pack(C.byref(a), ptr(buf), n, stream()))
                self.packed = buf
        if self.packed is not False:
            w.packed = self.packed.data_ptr()
        check(lib().xb_din_attention(C.byref(a), stream()))
        return out


def device_status():
    s = C.c_int32(0)
    check(lib().xb_device_status(C.byref(s)))
    return s.value


class DinTower:
    """Weights of the DIN tower (du+5d -> n1 -> n2 -> n3, Dice after the first two layers, or PReLU) packed for
    xb_din_tower. W1 [du+5d, n1], W2 [n1, n2], W3 [n2, n3] are float32 CPU tensors in Blaze's [K, N] layout; dice1, dice2:
    (gamma, mean, var), or with act XB_ACT_PRELU (slopes,)."""

    def __init__(self, d, du, W1, b1, dice1, W2, b2, dice2, W3, b3, softmax=True, device="cuda", act=capi.XB_ACT_DICE):
        h = lambda x: x.to(device=device, dtype=torch.float16).contiguous()
        f = lambda x: x.to(device=device, dtype=torch.float32).contiguous()
        self.d, self.du = d, du
        self.n1, self.n2, self.n3 = W1.shape[1], W2.shape[1], W3.shape[1]
        assert W1.shape[0] == du + 5 * d and W2.shape[0] == self.n1 and W3.shape[0] == self.n2
        self.act = act
        if act == capi.XB_ACT_PRELU:
            dice1, dice2 = [dice1[0]] * 3, [dice2[0]] * 3           # only the first of each is read
        self.keep = [h(W1), f(b1), f(dice1[0]), f(dice1[1]), f(dice1[2]), h(W2), f(b2), f(dice2[0]), f(dice2[1]),
                     f(dice2[2]), h(W3), f(b3)]
        self.softmax = softmax
        nbytes = lib().xb_din_tower_packed_bytes(d, self.n1, self.n2, self.n3)
        if nbytes == 0:
            raise capi.XbError("DinTower: shape outside the fused tower kernel")
        self.packed = torch.empty(nbytes, dtype=torch.uint8, device=device)
        a = self._args()
        check(lib().xb_din_tower_pack(C.byref(a), ptr(self.packed), nbytes, stream()))
        self._ws = None

    def _args(self):
        a = capi.DinTowerArgs()
        a.d, a.du, a.n1, a.n2, a.n3, a.softmax = self.d, self.du, self.n1, self.n2, self.n3, int(self.softmax)
        k = self.keep
        a.W1, a.b1, a.gamma1, a.mean1, a.var1 = k[0].data_ptr(), k[1].data_ptr(), k[2].data_ptr(), k[3].data_ptr(), k[4].data_ptr()
        a.W2, a.b2, a.gamma2, a.mean2, a.var2 = k[5].data_ptr(), k[6].data_ptr(), k[7].data_ptr(), k[8].data_ptr(), k[9].data_ptr()
        a.W3, a.b3, a.act = k[10].data_ptr(), k[11].data_ptr(), self.act
        a.packed = self.packed.data_ptr()
        return a

    def workspace(self, requests, device="cuda"):
        """A workspace of its own for callers that keep several launches in flight on different streams."""
        return torch.empty(int(lib().xb_din_tower_workspace_bytes(requests, self.d, self.n1)), dtype=torch.uint8, device=device)

    def __call__(self, user, q, k, att, requests, n_cand, T, out=None, ws=None):
        """user [R, du], q / att [R*n_cand, d], k [R*T, d] fp16 -> probabilities [R*n_cand, n3] fp32.
        `ws`: workspace from workspace(); the default one is shared by all calls of this object (one stream)."""
        if out is None:
            out = torch.empty((requests * n_cand, self.n3), dtype=torch.float32, device=q.device)
        need = lib().xb_din_tower_workspace_bytes(requests, self.d, self.n1)
        if ws is not None:
            assert ws.numel() >= need
            a = self._args()
            a.user, a.ldu, a.q, a.ldq = user.data_ptr(), user.stride(0), q.data_ptr(), q.stride(0)
            a.k, a.ldk, a.att, a.ldatt = k.data_ptr(), k.stride(0), att.data_ptr(), att.stride(0)
            a.prob, a.requests, a.n_cand, a.T = out.data_ptr(), requests, n_cand, T
            check(lib().xb_din_tower(C.byref(a), ptr(ws), ws.numel(), stream()))
            return out
        if self._ws is None or self._ws.numel() < need:
            self._ws = torch.empty(need, dtype=torch.uint8, device=q.device)
        a = self._args()
        a.user, a.ldu, a.q, a.ldq = user.data_ptr(), user.stride(0), q.data_ptr(), q.stride(0)
        a.k, a.ldk, a.att, a.ldatt = k.data_ptr(), k.stride(0), att.data_ptr(), att.stride(0)
        a.prob, a.requests, a.n_cand, a.T = out.data_ptr(), requests, n_cand, T
        check(lib().xb_din_tower(C.byref(a), ptr(self._ws), self._ws.numel(), stream()))
        return out


def _same(what, device, **tensors):
    """The tensors that are given lie on the device the call runs on."""
    for n, t in tensors.items():
        if t is not None and t.device != device:
            raise capi.XbError("%s: %s is on %s, the call on %s" % (what, n, t.device, device))


def _rows(what, name, t, rows, width, dtype):
    if t.dim() != 2 or t.dtype != dtype or t.size(0) != rows or t.size(1) != width or (width > 1 and t.stride(1) != 1):
        raise capi.XbError("%s: %s is [%d, %d] of %s with adjacent columns" % (what, name, rows, width, dtype))


def _dense(what, name, t, shape, dtype):
    if tuple(t.shape) != tuple(shape) or t.dtype != dtype or not t.is_contiguous():
        raise capi.XbError("%s: %s is a contiguous %s of %s" % (what, name, list(shape), dtype))


def _lists(what, a, rows, offsets, T, slots, first, last, inner, dtype):
    """rows, offsets, slots and kept states of the lists of a call into its arguments."""
    if offsets is not None:
        if offsets.dim() != 1 or offsets.dtype != torch.int32 or offsets.numel() < 1 or not offsets.is_contiguous():
            raise capi.XbError("%s: offsets are a contiguous int32 [lists + 1]" % what)
        a.batch = offsets.numel() - 1
    else:
        T = rows if T is None else T
        if T < 0 or (rows and (T < 1 or rows % T)):
            raise capi.XbError("%s: lists of %d rows in %d rows" % (what, T, rows))
        a.batch = rows // T if T else 0
    a.rows, a.offsets = rows, ptr(offsets)
    if slots is not None:
        _dense(what, "slots", slots, (a.batch,), torch.int32)
        a.slots = slots.data_ptr()
    n = None
    for name, t in (("the first states", first), ("the last states", last)):
        if t is None:
            continue
        if t.dim() != 3 or tuple(t.shape[1:]) != inner or t.dtype != dtype or not t.is_contiguous() or (n is not None and t.size(0) != n):
            raise capi.XbError("%s: %s are a contiguous [slots, %d, %d] of %s" % ((what, name) + inner + (dtype,)))
        n = t.size(0)
    a.n_slots = n or 0


def ssm_conv(x, w, bias=None, offsets=None, T=None, state_in=None, state_out=None, slots=None, silu=True, out=None):
    """The short causal convolution ahead of ssm_scan, over lists that lie one after the other in the rows of x [rows, D].

    w [D, K], bias [D]. Lists: `offsets` int32 [lists + 1], or of T rows each (T = 1: one new row a list; None: one list).
    state_in / state_out [slots, K - 1, D]: the inputs before each list and the last ones of it, in row slots[i] for list i (its own
    number without `slots`); they may be one array. Returns [rows, D]; rows behind the last list are not written."""
    rows, D = x.shape
    K = w.size(-1)
    dev = torch.device("cuda", torch.cuda.current_device())
    _same("ssm_conv", dev, x=x, w=w, bias=bias, offsets=offsets, state_in=state_in, state_out=state_out, slots=slots, out=out)
    if out is None:
        out = torch.empty((rows, D), dtype=x.dtype, device=x.device)
    _rows("ssm_conv", "x", x, rows, D, x.dtype)
    _rows("ssm_conv", "out", out, rows, D, x.dtype)
    _dense("ssm_conv", "w", w, (D, K), x.dtype)
    if bias is not None:
        _dense("ssm_conv", "bias", bias, (D,), x.dtype)
    a = capi.SsmConvArgs()
    _lists("ssm_conv", a, rows, offsets, T, slots, state_in, state_out, (K - 1, D), x.dtype)
    a.x, a.ldx, a.y, a.ldy, a.w, a.bias = x.data_ptr(), x.stride(0), out.data_ptr(), out.stride(0), w.data_ptr(), ptr(bias)
    a.state_in, a.state_out, a.D, a.K, a.silu, a.dtype = ptr(state_in), ptr(state_out), D, K, int(silu), dt(x)
    check(lib().xb_ssm_conv(C.byref(a), stream()))
    return out


def ssm_scan(x, delta, A, B, C_, D=None, z=None, delta_bias=None, groups=1, softplus=True, offsets=None, T=None, longest=0, h_in=None,
             h_out=None, slots=None, out=None, workspace=None):
    """The selective state-space scan over lists that lie one after the other in the rows of x [rows, channels].

    delta, z as x; B, C_ [rows, groups * N]; A [channels, N], D and delta_bias [channels], h_in / h_out [slots, channels, N] fp32.
    Lists and slots as in ssm_conv; `longest`: rows of the longest list where the caller knows it (the plan goes by it, no result).
    `workspace`: uint8 scratch for callers that keep one; by default the call takes its own."""
    rows, ch = x.shape
    N = A.size(-1)
    dev = torch.device("cuda", torch.cuda.current_device())
    _same("ssm_scan", dev, x=x, delta=delta, A=A, B=B, C=C_, D=D, z=z, delta_bias=delta_bias, offsets=offsets, h_in=h_in, h_out=h_out,
          slots=slots, out=out, workspace=workspace)
    if out is None:
        out = torch.empty((rows, ch), dtype=x.dtype, device=x.device)
    for n, t, width in (("x", x, ch), ("delta", delta, ch), ("z", z, ch), ("B", B, groups * N), ("C", C_, groups * N), ("out", out, ch)):
        if t is not None:
            _rows("ssm_scan", n, t, rows, width, x.dtype)
    _dense("ssm_scan", "A", A, (ch, N), torch.float32)
    for n, t in (("D", D), ("delta_bias", delta_bias)):
        if t is not None:
            _dense("ssm_scan", n, t, (ch,), torch.float32)
    a = capi.SsmScanArgs()
    _lists("ssm_scan", a, rows, offsets, T, slots, h_in, h_out, (ch, N), torch.float32)
    a.x, a.ldx, a.delta, a.lddelta, a.y, a.ldy = x.data_ptr(), x.stride(0), delta.data_ptr(), delta.stride(0), out.data_ptr(), out.stride(0)
    if z is not None:
        a.z, a.ldz = z.data_ptr(), z.stride(0)
    a.B, a.ldb, a.C, a.ldc = B.data_ptr(), B.stride(0), C_.data_ptr(), C_.stride(0)
    a.A, a.skip, a.delta_bias, a.h_in, a.h_out = A.data_ptr(), ptr(D), ptr(delta_bias), ptr(h_in), ptr(h_out)
    a.D, a.N, a.groups, a.softplus, a.dtype, a.longest = ch, N, groups, int(softplus), dt(x), longest
    need = int(lib().xb_ssm_scan_workspace_bytes(C.byref(a)))
    if need and workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
    check(lib().xb_ssm_scan(C.byref(a), ptr(workspace), workspace.numel() if workspace is not None else 0, stream()))
    return out


def lora_gemm(X, W, A, B, adapter, bias=None, scale=None, trans_b=False, out_dtype=None, Y=None, workspace=None):
    """X W + bias with a low-rank adapter of each row's own beside it: + scale[a] (X[m] A[a]^T) B[a]^T, a = adapter[m].

    X [M, K]; W [K, N], or [N, K] with trans_b; A [adapters, r, K]; B [adapters, N, r]; adapter int32 [M], outside [0, adapters) for a
    row without one; bias [N] and scale [adapters] fp32. Results in X's type or fp32."""
    M, K = X.shape
    N = W.size(0 if trans_b else 1)
    dev = torch.device("cuda", torch.cuda.current_device())
    _same("lora_gemm", dev, X=X, W=W, A=A, B=B, adapter=adapter, bias=bias, scale=scale, Y=Y, workspace=workspace)
    if Y is None:
        Y = torch.empty((M, N), dtype=out_dtype or X.dtype, device=X.device)
    n, r, _ = A.shape
    _rows("lora_gemm", "X", X, M, K, X.dtype)
    _rows("lora_gemm", "W", W, N if trans_b else K, K if trans_b else N, X.dtype)
    _rows("lora_gemm", "Y", Y, M, N, Y.dtype if out_dtype is None else out_dtype)
    _dense("lora_gemm", "adapter", adapter, (M,), torch.int32)
    for name, t, rows, cols in (("A", A, r, K), ("B", B, N, r)):
        if t.dim() != 3 or t.dtype != X.dtype or tuple(t.shape) != (n, rows, cols) or (cols > 1 and t.stride(2) != 1):
            raise capi.XbError("lora_gemm: %s is [%d, %d, %d] of %s with adjacent columns" % (name, n, rows, cols, X.dtype))
    for name, t, size in (("bias", bias, N), ("scale", scale, n)):
        if t is not None:
            _dense("lora_gemm", name, t, (size,), torch.float32)
    a = capi.LoraArgs()
    a.M, a.N, a.K, a.r, a.n_adapters, a.trans_w = M, N, K, r, n, int(trans_b)
    a.X, a.ldx, a.W, a.ldw, a.Y, a.ldy = X.data_ptr(), X.stride(0), W.data_ptr(), W.stride(0), Y.data_ptr(), Y.stride(0)
    a.A, a.lda, a.stride_a, a.B, a.ldb, a.stride_b = A.data_ptr(), A.stride(1), A.stride(0), B.data_ptr(), B.stride(1), B.stride(0)
    a.scale, a.bias, a.adapter, a.dtype, a.y_dtype = ptr(scale), ptr(bias), adapter.data_ptr(), dt(X), dt(Y)
    need = int(lib().xb_lora_workspace_bytes(C.byref(a)))
    if need and workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=X.device)
    check(lib().xb_lora_gemm(C.byref(a), ptr(workspace), workspace.numel() if workspace is not None else 0, stream()))
    return Y
