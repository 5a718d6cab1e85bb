// Selective state-space layer over behaviour lists: the short causal convolution, and what a scan runs as (formulas in xdlb200.h; the scan's
// kernels are in xb_ssm_scan.cuh, compiled for one type each in xb_ssm_scan_*.cu).
#include <algorithm>
#include <cmath>

#include "xb_common.cuh"
#include "xb_ssm.cuh"

namespace xb {
namespace {

constexpr int CONV_THREADS = 128, CONV_AHEAD = 8;
struct ConvParams {
  const void* x; int64_t ldx;
  void* y; int64_t ldy;
  const void* w; const void* bias;
  const void* state_in; void* state_out;
  Lists lists;
  int D, silu, vec, vec_w, vec_state;
  int pieces, n_chunks, rows_a_chunk;     // threads of a row; what a thread walks
  int walk_blocks;                        // the blocks behind these keep the states of lists without rows
};

// The taps and the last K - 1 inputs of V adjacent channels, as pairs of fp32
template <typename T, int V, int K>
struct ConvTaps {
  static constexpr int P = (V + 1) / 2;
  f32x2 w[K][P], bias[P], past[K - 1][P];
  static __device__ __forceinline__ void pairs(const Raw<T, V>& t, f32x2 (&to)[P]) {
#pragma unroll
    for (int q = 0; q < P; ++q) to[q] = pack2(t.get(2 * q), 2 * q + 1 < V ? t.get((2 * q + 1) % V) : 0.f);
  }
  __device__ __forceinline__ void load(const ConvParams& p, int c, int in) {
    const T *pw = static_cast<const T*>(p.w) + (int64_t)c * K, *pb = static_cast<const T*>(p.bias) + c;
    Raw<T, V> t[K];
#pragma unroll
    for (int j = 0; j < K; ++j) t[j].load(pw + j * V, in * K - j * V, p.vec_w);
    auto weight = [&](int e) { return e < V * K ? t[e / V % K].get(e % V) : 0.f; };      // element e of the V channels' K taps
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
      for (int q = 0; q < P; ++q) w[j][q] = pack2(weight(2 * q * K + j), weight((2 * q + 1) * K + j));
    t[0].zero();
    if (p.bias) t[0].load(pb, in, p.vec_w);
    pairs(t[0], bias);
  }
  // the outputs of the row `t`, which becomes the last input
  __device__ __forceinline__ void row(int silu, const Raw<T, V>& t, Raw<T, V>& out) {
    f32x2 x[P], o[P];
    pairs(t, x);
#pragma unroll
    for (int q = 0; q < P; ++q) {
      f32x2 s = bias[q];
#pragma unroll
      for (int j = 0; j < K - 1; ++j) s = fma2(w[j][q], past[j][q], s);
      o[q] = fma2(w[K - 1][q], x[q], s);
#pragma unroll
      for (int j = 0; j + 1 < K - 1; ++j) past[j][q] = past[j + 1][q];
      past[K - 2][q] = x[q];
    }
    if (silu) {
#pragma unroll
      for (int q = 0; q < P; ++q) o[q] = silu2(o[q]);
    }
    float v[2 * P], first[V];
#pragma unroll
    for (int q = 0; q < P; ++q) unpack2(o[q], v[2 * q], v[2 * q + 1]);
#pragma unroll
    for (int i = 0; i < V; ++i) first[i] = v[i];
    out.put_all(first);
  }
};

// One row a list: a thread has V channels of it. All that it reads, states, row and weights, is on its way at once, where the walk reads one
// after the other. 4 taps: 74 rows of 72 in a graph 4.3 us as a walk, 1.95 so; 8192 rows of 256, bf16, 27 and 7.3 (4.6 TB/s).
template <typename T, int V, int K>
__global__ void __launch_bounds__(CONV_THREADS) ssm_conv_step_kernel(const ConvParams p) {
  pdl_begin();
  const uint64_t e = (uint64_t)blockIdx.x * CONV_THREADS + threadIdx.x;
  const int64_t i = e >> 32 ? (int64_t)(e / (uint32_t)p.pieces) : (int64_t)((uint32_t)e / (uint32_t)p.pieces);
  if (i >= p.lists.rows) return;
  const int c = (int)((int64_t)e - i * p.pieces) * V, in = min(V, p.D - c), slot = p.lists.slot((int)i);
  const int64_t state = (int64_t)slot * (K - 1) * p.D + c;
  Raw<T, V> x, kept[K - 1], out;
  x.load(static_cast<const T*>(p.x) + i * p.ldx + c, in, p.vec);
#pragma unroll
  for (int j = 0; j < K - 1; ++j) {
    kept[j].zero();
    if (p.state_in && slot >= 0) kept[j].load_kept(static_cast<const T*>(p.state_in) + state + (int64_t)j * p.D, in, p.vec_state);
  }
  ConvTaps<T, V, K> taps;
  taps.load(p, c, in);
#pragma unroll
  for (int j = 0; j < K - 1; ++j) taps.pairs(kept[j], taps.past[j]);
  taps.row(p.silu, x, out);
  out.store(static_cast<T*>(p.y) + i * p.ldy + c, in, p.vec);
  if (p.state_out && slot >= 0) {
    T* to = static_cast<T*>(p.state_out) + state;
#pragma unroll
    for (int j = 0; j + 1 < K - 1; ++j) kept[j + 1].store(to + (int64_t)j * p.D, in, p.vec_state);
    x.store(to + (int64_t)(K - 2) * p.D, in, p.vec_state);
  }
}

// A thread walks `rows_a_chunk` rows of V channels with the last K - 1 inputs in registers; the threads of a chunk lie side by side, and
// chunks follow one another without a gap, so no lane idles whatever D is. x is read 1 + (K - 1) / rows_a_chunk times.
// The thread that has a list's first row makes its first K - 1 rows (they read the state) and its last state, so that states moved
// on in place are read and written by one thread.
// Pieces of 8 bytes and eight rows ahead: with 16-byte pieces and four rows the registers let half as many warps in, which is what
// the loads in flight are. SiLU is the rest: an exponential and a quotient a value. Bound by the latency of the reads in flight:
// 1024 lists of 262144 rows in all, D = 512, bf16 135 us = 4.0 TB/s, 0.62 of a copy's rate, 24 warps an SM, SFUs 49 % busy. The
// next rows asked for before these are written, and longer or shorter walks, are no faster.
// Blocks of an SM, among which the registers are shared: with fewer the compiler takes more (two taps of fp32 122 of them: 781 lists of 14810 rows, D = 24
// 11.2 us, 8.3 so), with more it spills.
template <typename T, int V, int K>
constexpr int CONV_BLOCKS = K == 2 || (K <= 4 && V * sizeof(T) <= 8) ? 6 : K == 3 ? 5 : 4;
template <typename T, int V, int K>
__global__ void __launch_bounds__(CONV_THREADS, CONV_BLOCKS<T, V, K>) ssm_conv_kernel(const ConvParams p) {
  pdl_begin();
  if ((int)blockIdx.x >= p.walk_blocks) {              // lists without rows: their states go from one array to the other
    const int64_t e = (int64_t)((int)blockIdx.x - p.walk_blocks) * CONV_THREADS + threadIdx.x, i = e / p.pieces;
    if (i >= p.lists.batch || p.lists.begin((int)i + 1) > p.lists.begin((int)i)) return;
    const int slot = p.lists.slot((int)i), c = (int)(e - i * p.pieces) * V, in = min(V, p.D - c);
    if (slot < 0) return;
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
      const int64_t at = ((int64_t)slot * (K - 1) + j) * p.D + c;
      Raw<T, V> t;
      t.zero();
      if (p.state_in) t.load_kept(static_cast<const T*>(p.state_in) + at, in, p.vec_state);
      t.store(static_cast<T*>(p.state_out) + at, in, p.vec_state);
    }
    return;
  }
  __shared__ int s_first[CONV_THREADS];                // the first list that begins in or behind each of the block's chunks
  const int lane = threadIdx.x & 31;
  const int64_t at = (int64_t)blockIdx.x * CONV_THREADS, at_me = at + threadIdx.x;
  const int64_t c_first = at / p.pieces;
  const int chunks = (int)((at + CONV_THREADS - 1) / p.pieces - c_first) + 1;
  for (int i = threadIdx.x / 32; i < chunks; i += CONV_THREADS / 32) {
    const int f = p.lists.first_from((c_first + i) * p.rows_a_chunk, lane);
    if (lane == 0) s_first[i] = f;
  }
  __syncthreads();
  const int64_t chunk = at_me / p.pieces;
  if (chunk >= p.n_chunks) return;
  const int c = (int)(at_me - chunk * p.pieces) * V, in = min(V, p.D - c);
  const int64_t r0 = chunk * p.rows_a_chunk, r1 = r0 + p.rows_a_chunk;
  const T* px = static_cast<const T*>(p.x) + c;
  T* py = static_cast<T*>(p.y) + c;
  constexpr int CONV_FEW = V == 1 ? CONV_AHEAD : 4;
  ConvTaps<T, V, K> taps;
  taps.load(p, c, in);
  auto& past = taps.past;
  auto row_of = [&](const Raw<T, V>& t, Raw<T, V>& out) { taps.row(p.silu, t, out); };
  const bool whole_piece = Raw<T, V>::PIECE && p.vec && in == V;
  int nxt = s_first[(int)(chunk - c_first)];
  int64_t r = r0, stop = r0;
  if (nxt > 0 && p.lists.begin(nxt) > r0) {            // a list from before: its rows from the K-th on
    const int64_t b = p.lists.begin(nxt - 1);
    r = max(r0, b + K - 1);
    stop = min(r1, p.lists.begin(nxt));
    if (r < stop) {
#pragma unroll
      for (int j = 0; j < K - 1; ++j) {
        Raw<T, V> t;
        t.load(px + (r - (K - 1) + j) * p.ldx, in, p.vec);
        taps.pairs(t, past[j]);
      }
    }
  }
  for (;;) {
    const T* from = px + r * p.ldx;
    T* to = py + r * p.ldy;
    if (whole_piece) {
      for (; r + CONV_AHEAD <= stop; r += CONV_AHEAD, from += CONV_AHEAD * p.ldx, to += CONV_AHEAD * p.ldy) {
        Raw<T, V> t[CONV_AHEAD];
#pragma unroll
        for (int i = 0; i < CONV_AHEAD; ++i) t[i].load_piece(from + i * p.ldx);
#pragma unroll
        for (int i = 0; i < CONV_AHEAD; ++i) {
          Raw<T, V> out;
          row_of(t[i], out);
          out.store_piece(to + i * p.ldy);
        }
      }
    }
    for (; r < stop; r += CONV_FEW, from += CONV_FEW * p.ldx, to += CONV_FEW * p.ldy) {
      Raw<T, V> t[CONV_FEW], out;
#pragma unroll
      for (int i = 0; i < CONV_FEW; ++i) t[i].load(from + i * p.ldx, r + i < stop ? in : 0, p.vec);
#pragma unroll
      for (int i = 0; i < CONV_FEW; ++i) {
        if (r + i >= stop) break;
        row_of(t[i], out);
        out.store(to + i * p.ldy, in, p.vec);
      }
    }
    r = stop;
    if (nxt >= p.lists.batch) return;
    const int64_t b = p.lists.begin(nxt);
    if (b >= r1) return;
    int64_t e = p.lists.begin(nxt + 1);
    if (e <= b) {                                      // past all lists without rows: up to the last that begins at b
      int lo = nxt + 1, hi = p.lists.batch;            // the first that begins behind b is in [lo, hi], or there is none
      while (lo < hi) {
        const int mid = lo + (hi - lo) / 2;
        if (p.lists.begin(mid) > b) hi = mid;
        else lo = mid + 1;
      }
      e = p.lists.begin(hi);
      if (e <= b) return;
      nxt = hi - 1;
    }
    const int slot = p.lists.slot(nxt);
    const int64_t state = ((int64_t)slot * (K - 1)) * p.D + c;
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
      Raw<T, V> t;
      t.zero();
      if (p.state_in && slot >= 0) t.load_kept(static_cast<const T*>(p.state_in) + state + (int64_t)j * p.D, in, p.vec_state);
      taps.pairs(t, past[j]);
    }
    if (p.state_out && slot >= 0) {
#pragma unroll
      for (int j = 0; j < K - 1; ++j) {                // place len - (K - 1) + j of the list, before its first row in the state
        const int64_t place = e - b - (K - 1) + j;
        Raw<T, V> t;
        if (place >= 0) {
          t.load(px + (b + place) * p.ldx, in, p.vec);
        } else {
#pragma unroll
          for (int q = 0; q < taps.P; ++q) {
            f32x2 was = 0;
#pragma unroll
            for (int k = 0; k < K - 1; ++k) was = k == (int)place + K - 1 ? past[k][q] : was;
            float lo, hi;
            unpack2(was, lo, hi);
            t.put(2 * q, lo);
            if (2 * q + 1 < V) t.put((2 * q + 1) % V, hi);
          }
        }
        t.store(static_cast<T*>(p.state_out) + state + (int64_t)j * p.D, in, p.vec_state);
      }
    }
    ++nxt;
    r = b;
    stop = min(e, max(r1, b + K - 1));
  }
}

constexpr int32_t MOST = INT32_MAX - 1023;             // of channels and lists: rounded up to whole blocks they are counted in 32 bits
int check_lists(const char* what, const int32_t* offsets, const int32_t* slots, bool states, int64_t rows, int32_t batch, int32_t n_slots, int32_t D) {
  XB_REQUIRE(rows >= 0 && batch >= 0, XB_ERR_ARG, "%s: %lld rows, %d lists", what, (long long)rows, batch);
  XB_REQUIRE(batch <= MOST && D <= MOST, XB_ERR_LIMIT, "%s: %d lists, %d channels, at most 2^31 - 1024", what, batch, D);
  XB_REQUIRE(rows < ((int64_t)1 << 31), XB_ERR_LIMIT, "%s: %lld rows, fewer than 2^31", what, (long long)rows);
  XB_REQUIRE(offsets || batch == 0 || rows % batch == 0, XB_ERR_ARG, "%s: without offsets %d lists divide %lld rows", what, batch, (long long)rows);
  XB_REQUIRE(!states || n_slots >= 0, XB_ERR_ARG, "%s: n_slots %d", what, n_slots);
  XB_REQUIRE(!states || slots || n_slots >= batch, XB_ERR_ARG, "%s: %d states for %d lists without slots", what, n_slots, batch);
  return 0;
}
// the arrays of kept states: one, or two that share nothing
bool states_apart(const void* first, const void* last, int64_t bytes) {
  const uintptr_t p = reinterpret_cast<uintptr_t>(first), q = reinterpret_cast<uintptr_t>(last);
  return !first || !last || p == q || p + (uintptr_t)bytes <= q || q + (uintptr_t)bytes <= p;
}
Lists lists_of(const int32_t* offsets, const int32_t* slots, int64_t rows, int32_t batch, int32_t n_slots) {
  return {offsets, slots, rows, batch > 0 ? rows / batch : 0, batch, n_slots};
}
bool ssm_dtype(int dtype) { return dtype == XB_F32 || dtype == XB_F16 || dtype == XB_BF16; }

template <typename T, int V, int K>
int launch_conv_taps(ConvParams p, cudaStream_t s) {
  auto blocks_of = [&](int64_t n) { return (n * p.pieces + CONV_THREADS - 1) / CONV_THREADS; };
  if (!p.lists.offsets && p.lists.per == 1) {
    const int64_t blocks = blocks_of(p.lists.rows);
    XB_REQUIRE(blocks < ((int64_t)1 << 31), XB_ERR_LIMIT, "xb_ssm_conv: too many rows and channels");
    launch_dependent(ssm_conv_step_kernel<T, V, K>, (unsigned)blocks, CONV_THREADS, 0, s, p);
    return check_launch("ssm_conv_step_kernel");
  }
  int64_t blocks = blocks_of(p.n_chunks);
  p.walk_blocks = (int)std::min<int64_t>(blocks, INT32_MAX);
  // states moved on in place stay as they are
  if (p.state_out && p.state_out != p.state_in && (p.lists.offsets || p.lists.rows == 0)) blocks += blocks_of(p.lists.batch);
  XB_REQUIRE(blocks < ((int64_t)1 << 31), XB_ERR_LIMIT, "xb_ssm_conv: too many rows and channels");
  launch_dependent(ssm_conv_kernel<T, V, K>, (unsigned)blocks, CONV_THREADS, 0, s, p);
  return check_launch("ssm_conv_kernel");
}
template <typename T, int V>
int launch_conv_pieces(ConvParams p, int K, cudaStream_t s) {
  p.pieces = (p.D + V - 1) / V;
  if (V == 1) p.vec = p.vec_w = p.vec_state = 1;       // (pieces of one element lie aligned)
  // Longer walks read less twice, shorter ones keep more threads in flight.
  const int64_t threads = p.lists.rows * p.pieces, fill = (int64_t)sm_count() * 1024;
  p.rows_a_chunk = (int)std::min<int64_t>(std::max<int64_t>(threads / fill, 1), 32);
  p.n_chunks = (int)std::max<int64_t>((p.lists.rows + p.rows_a_chunk - 1) / p.rows_a_chunk, 1);
  switch (K) {
    case 2: return launch_conv_taps<T, V, 2>(p, s);
    case 3: return launch_conv_taps<T, V, 3>(p, s);
    case 4: return launch_conv_taps<T, V, 4>(p, s);
    case 5: return launch_conv_taps<T, V, 5>(p, s);
    case 6: return launch_conv_taps<T, V, 6>(p, s);
    case 7: return launch_conv_taps<T, V, 7>(p, s);
    default: return launch_conv_taps<T, V, 8>(p, s);
  }
}
bool whole(const void* q, int64_t ld_bytes, int64_t unit) { return reinterpret_cast<uintptr_t>(q) % unit == 0 && ld_bytes % unit == 0; }
template <typename T>
int launch_conv(const xb_ssm_conv_args& a, cudaStream_t s) {
  constexpr int SIZE = sizeof(T);
  ConvParams p = {};
  p.x = a.x; p.ldx = a.ldx; p.y = a.y; p.ldy = a.ldy; p.w = a.w; p.bias = a.bias; p.state_in = a.state_in; p.state_out = a.state_out;
  p.lists = lists_of(a.offsets, a.slots, a.rows, a.batch, a.n_slots);
  p.D = a.D; p.silu = a.silu;
  constexpr int unit = 4 * SIZE;
  p.vec = whole(a.x, a.ldx * SIZE, unit) && whole(a.y, a.ldy * SIZE, unit);
  p.vec_w = whole(a.w, 0, unit) && whole(a.bias, 0, unit);
  p.vec_state = whole(a.state_in, (int64_t)a.D * SIZE, unit) && whole(a.state_out, 0, unit);
  // rows that do not start on whole pieces: a channel a thread, adjacent lanes adjacent channels
  return p.vec ? launch_conv_pieces<T, 4>(p, a.K, s) : launch_conv_pieces<T, 1>(p, a.K, s);
}

int scan_blocks(const xb_ssm_scan_args& a, int lanes, int K) {
  const int per = a.D / a.groups, ch = SCAN_THREADS / lanes * K;
  return a.groups * ((per + ch - 1) / ch);
}
ScanPlan scan_plan(const xb_ssm_scan_args& a) {
  ScanPlan p = {};
  p.lanes = a.N <= 4 ? 1 : a.N <= 8 ? 2 : a.N <= 16 ? 4 : a.N <= 32 ? 8 : 16;
  p.step = !a.offsets && a.rows == a.batch;
  if (p.step) return p;
  const double sms = std::max(sm_count(), 1), mean = (double)a.rows / a.batch;
  const double longest = !a.offsets ? mean : (double)(a.longest > 0 ? std::min(a.longest, a.rows) : a.rows);
  // Cycles: a row of a block takes `work` of a full SM and `alone` where its SM has little else, which is what the longest list (or
  // chunk) ends with; a block begins with 600 of them, one of the two walks of a chunk with 2000. Lists that are split are walked nearly
  // twice; of lists of all lengths the share in ones above `chunk` rows is that of an exponential distribution.
  // us, whole lists as they come, long ones first, the best split: 256 lists of up to 1860 rows in 70000, D = 256 229, 193, 226; 1000 in
  // 20000, D = 256 68, 54; 16 of up to 3640 in 16384, D = 512 246 and 125 split; one of 4096, D = 1024 302 and 68; 300 of 100, D = 256
  // 65 and 124.
  double best = 0;
  for (int K : {1, 2}) {
    if (K == 1 && p.lanes > 4) continue;  // (a block would have 16 channels or fewer)
    const double work = K == 2 ? 155 : 80, alone = K == 1 ? 130 : p.lanes <= 4 ? 260 : 32 * p.lanes;
    const int blocks = scan_blocks(a, p.lanes, K);
    const double full = (double)a.rows * blocks * work / sms;
    // lists of unlike lengths in more than a wave of blocks: long ones first (one block puts them in order: up to 64 rounds of its threads)
    const bool order = a.offsets && longest > 1.5 * mean && a.batch <= 65536 && (double)a.batch * blocks > 5 * sms;
    const double whole = (order ? std::max(full + 6000, alone * longest) : full + 0.6 * alone * longest) + 600.0 * a.batch * blocks / sms;
    if (best == 0 || whole < best) { best = whole; p.K = K; p.chunk = 0; p.order = order; }
    for (int64_t chunk = 64; chunk < longest; chunk += chunk & (chunk - 1) ? chunk / 3 : chunk / 2) {      // 64, 96, 128, 192, ...
      const double twice = longest > 1.5 * mean ? (1 + chunk / mean) * std::exp(-chunk / mean) : 1;
      const double split = full * (1 + 0.8 * twice) + 1.2 * alone * chunk + 4000 * (a.rows / (double)chunk + a.batch) * blocks / sms + 15000;
      if (split < best) { best = split; p.K = K; p.chunk = chunk; p.order = false; }
    }
  }
  return p;
}
constexpr size_t align256(size_t n) { return (n + 255) / 256 * 256; }
struct ScanScratch { size_t end, first, steps, kind, bytes; };      // (a plan has chunks or an order, whose place is the first)
ScanScratch scan_scratch(const xb_ssm_scan_args& a, const ScanPlan& p) {
  ScanScratch w = {};
  if (p.order) w.bytes = align256((size_t)a.batch * 4);
  if (p.chunk == 0 || a.rows / p.chunk == 0) return w;
  const size_t n = (size_t)(a.rows / p.chunk), states = align256(n * a.D * a.N * 4);
  w.first = w.end + states;
  w.steps = w.first + (a.h_in ? states : 0);
  w.kind = w.steps + align256(n * a.D * 4);
  w.bytes = w.kind + align256(n * 4);
  return w;
}

ScanParams scan_params(const xb_ssm_scan_args& a, const ScanPlan& plan, uint8_t* ws) {
  ScanParams p = {};
  p.x = a.x; p.ldx = a.ldx; p.delta = a.delta; p.lddelta = a.lddelta; p.z = a.z; p.ldz = a.ldz;
  p.B = a.B; p.ldb = a.ldb; p.C = a.C; p.ldc = a.ldc; p.y = a.y; p.ldy = a.ldy;
  p.A = a.A; p.skip = a.skip; p.delta_bias = a.delta_bias; p.h_in = a.h_in; p.h_out = a.h_out;
  p.lists = lists_of(a.offsets, a.slots, a.rows, a.batch, a.n_slots);
  p.D = a.D; p.N = a.N; p.per_group = a.D / a.groups; p.groups = a.groups; p.softplus = a.softplus;
  const int64_t size = (int64_t)dtype_size(a.dtype);
  p.vec = whole(a.x, a.ldx * size, 4 * size) && whole(a.delta, a.lddelta * size, 4 * size) && whole(a.y, a.ldy * size, 4 * size) &&
          (!a.z || whole(a.z, a.ldz * size, 4 * size)) && (a.groups == 1 || p.per_group % 4 == 0);
  p.vec_bc = a.N % 4 == 0 && whole(a.B, a.ldb * size, 4 * size) && whole(a.C, a.ldc * size, 4 * size);
  p.vec_h = a.N % 4 == 0 && whole(a.A, 0, 16) && whole(a.h_in, 0, 16) && whole(a.h_out, 0, 16);
  const ScanScratch w = scan_scratch(a, plan);
  if (plan.order) p.order = reinterpret_cast<int*>(ws);
  if (plan.chunk > 0 && w.bytes) {
    p.chunk = plan.chunk; p.n_ends = (int)(a.rows / plan.chunk);
    p.end = reinterpret_cast<float*>(ws + w.end); p.first = reinterpret_cast<float*>(ws + w.first);
    p.steps = reinterpret_cast<float*>(ws + w.steps); p.kind = reinterpret_cast<int*>(ws + w.kind);
  }
  return p;
}

}  // namespace
}  // namespace xb

using namespace xb;

extern "C" int xb_ssm_conv(const xb_ssm_conv_args* a, xb_stream_t s) {
  XB_REQUIRE(a, XB_ERR_ARG, "xb_ssm_conv: null arguments");
  XB_REQUIRE(ssm_dtype(a->dtype), XB_ERR_UNSUPPORTED, "xb_ssm_conv: dtype %d", a->dtype);
  XB_REQUIRE(a->D >= 1, XB_ERR_ARG, "xb_ssm_conv: %d channels", a->D);
  XB_REQUIRE(a->K >= 2 && a->K <= 8, XB_ERR_LIMIT, "xb_ssm_conv: %d taps, from 2 to 8", a->K);
  if (int rc = check_lists("xb_ssm_conv", a->offsets, a->slots, a->state_in || a->state_out, a->rows, a->batch, a->n_slots, a->D)) return rc;
  if (a->batch == 0) return 0;
  XB_REQUIRE(a->w && (a->rows == 0 || (a->x && a->y)), XB_ERR_ARG, "xb_ssm_conv: null tensor");
  XB_REQUIRE(a->rows == 0 || (a->ldx >= a->D && a->ldy >= a->D), XB_ERR_ARG, "xb_ssm_conv: row strides %lld, %lld of %d channels",
             (long long)a->ldx, (long long)a->ldy, a->D);
  const int64_t size = (int64_t)dtype_size(a->dtype), states = (int64_t)a->n_slots * (a->K - 1) * a->D * size;
  XB_REQUIRE(!rows_meet(a->x, a->ldx * size, a->D * size, a->y, a->ldy * size, a->D * size, a->rows), XB_ERR_ARG, "xb_ssm_conv: y overlaps x");
  XB_REQUIRE(states_apart(a->state_in, a->state_out, states), XB_ERR_ARG, "xb_ssm_conv: the two arrays of states overlap and are not one");
  if (a->dtype == XB_F32) return launch_conv<float>(*a, (cudaStream_t)s);
  if (a->dtype == XB_F16) return launch_conv<__half>(*a, (cudaStream_t)s);
  return launch_conv<__nv_bfloat16>(*a, (cudaStream_t)s);
}

namespace {
int check_scan(const xb_ssm_scan_args* a) {
  XB_REQUIRE(a, XB_ERR_ARG, "xb_ssm_scan: null arguments");
  XB_REQUIRE(ssm_dtype(a->dtype), XB_ERR_UNSUPPORTED, "xb_ssm_scan: dtype %d", a->dtype);
  XB_REQUIRE(a->D >= 1 && a->N >= 1 && a->groups >= 1 && a->D % a->groups == 0, XB_ERR_ARG, "xb_ssm_scan: %d channels in %d groups, %d states",
             a->D, a->groups, a->N);
  XB_REQUIRE(a->N <= 64, XB_ERR_LIMIT, "xb_ssm_scan: %d states, at most 64", a->N);
  XB_REQUIRE(a->longest >= 0, XB_ERR_ARG, "xb_ssm_scan: longest %lld", (long long)a->longest);
  if (int rc = check_lists("xb_ssm_scan", a->offsets, a->slots, a->h_in || a->h_out, a->rows, a->batch, a->n_slots, a->D)) return rc;
  if (a->batch == 0) return 0;
  XB_REQUIRE(a->A && (a->rows == 0 || (a->x && a->delta && a->B && a->C && a->y)), XB_ERR_ARG, "xb_ssm_scan: null tensor");
  XB_REQUIRE(a->rows == 0 || (a->ldx >= a->D && a->lddelta >= a->D && a->ldy >= a->D && (!a->z || a->ldz >= a->D)), XB_ERR_ARG,
             "xb_ssm_scan: a row stride below %d channels", a->D);
  XB_REQUIRE(a->rows == 0 || (a->ldb >= (int64_t)a->groups * a->N && a->ldc >= (int64_t)a->groups * a->N), XB_ERR_ARG,
             "xb_ssm_scan: a row stride of B or C below %d x %d", a->groups, a->N);
  return 0;
}
}  // namespace

extern "C" size_t xb_ssm_scan_workspace_bytes(const xb_ssm_scan_args* a) {
  if (check_scan(a) != 0 || a->batch == 0) return 0;
  return scan_scratch(*a, scan_plan(*a)).bytes;
}

extern "C" int xb_ssm_scan(const xb_ssm_scan_args* a, void* workspace, size_t workspace_bytes, xb_stream_t s) {
  if (int rc = check_scan(a)) return rc;
  if (a->batch == 0) return 0;
  const ScanPlan plan = scan_plan(*a);
  const size_t need = scan_scratch(*a, plan).bytes;
  XB_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), XB_ERR_SCRATCH, "xb_ssm_scan: workspace of %zu bytes, %zu needed",
             workspace_bytes, need);
  XB_REQUIRE(need == 0 || (reinterpret_cast<uintptr_t>(workspace) & 15) == 0, XB_ERR_ARG, "xb_ssm_scan: the workspace is not on 16 bytes");
  const int64_t size = (int64_t)dtype_size(a->dtype), row = a->D * size, bc = (int64_t)a->groups * a->N * size;
  auto over = [&](const void* in, int64_t ld, int64_t width) { return in && rows_meet(in, ld * size, width, a->y, a->ldy * size, row, a->rows); };
  XB_REQUIRE(!over(a->x, a->ldx, row) && !over(a->delta, a->lddelta, row) && !over(a->z, a->ldz, row) && !over(a->B, a->ldb, bc) && !over(a->C, a->ldc, bc),
             XB_ERR_ARG, "xb_ssm_scan: y overlaps an input");
  XB_REQUIRE(states_apart(a->h_in, a->h_out, (int64_t)a->n_slots * a->D * a->N * 4), XB_ERR_ARG, "xb_ssm_scan: the two arrays of states overlap and are not one");
  const ScanParams p = scan_params(*a, plan, static_cast<uint8_t*>(workspace));
  if (a->dtype == XB_F32) return ssm_scan_f32(p, plan, (cudaStream_t)s);
  if (a->dtype == XB_F16) return ssm_scan_f16(p, plan, (cudaStream_t)s);
  return ssm_scan_bf16(p, plan, (cudaStream_t)s);
}
