// Linear attention over lists: arguments, and what a call runs as (formulas in xdlb200.h; the kernels are in xb_linear.cuh, compiled for one type
// each in xb_linear_*.cu).
#include "xb_linear.cuh"

namespace xb {
namespace {

constexpr int32_t MOST = INT32_MAX - 1023;
constexpr size_t align256(size_t n) { return (n + 255) / 256 * 256; }

LinearPlan linear_plan(const xb_linear_attention_args& a) {
  LinearPlan p = {};
  const int64_t mean = a.batch > 0 ? a.rows / a.batch : 0;
  p.step = !a.offsets && a.rows == a.batch && a.dv % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.h_in) | reinterpret_cast<uintptr_t>(a.h_out)) & 15) == 0;
  if (p.step) return p;
  // A list of a few rows is a chunk of 64 all the same. us by rows and by chunks, bf16, 4096 lists, 4 heads of 64: of 8 rows 209 and 209, of 12 272 and
  // 211; 64 lists of 12 13 and 11.
  p.tiles = a.dtype != XB_F32 && mean >= 8;
  const int64_t longest = !a.offsets ? mean : a.longest > 0 ? std::min(a.longest, a.rows) : a.rows;
  // Lists are cut where some are so long that whole ones would leave SMs idle: into segments of what a block has of the rows where all are busy, 256
  // rows at least (both ways of a segment, and its state in memory, cost about half as much again).
  const int64_t slots = (int64_t)std::max(sm_count(), 1) * (p.tiles ? a.dv <= 64 ? (a.dk <= 64 ? 4 : 2) : (a.dk <= 64 ? 2 : 1) : 4);
  const int64_t share = (a.rows * a.H + slots - 1) / slots, chunk = std::max<int64_t>((share + 63) / 64 * 64, 256);
  if (longest > 3 * chunk) p.chunk = chunk;
  // whole lists of unlike lengths in more than a wave of blocks: long ones first
  p.order = p.chunk == 0 && a.offsets && longest > mean + mean / 2 && a.batch <= 65536 && (int64_t)a.batch * a.H > slots;
  return p;
}
struct LinearScratch { size_t first, bytes; };      // (the ends lie first; a plan has chunks or an order)
LinearScratch linear_scratch(const xb_linear_attention_args& a, const LinearPlan& p) {
  LinearScratch w = {};
  if (p.order) w.bytes = align256((size_t)a.batch * 4);
  if (p.chunk == 0 || a.rows / p.chunk == 0) return w;
  const size_t states = align256((size_t)(a.rows / p.chunk) * a.H * a.dk * a.dv * 4);
  w.first = states;
  w.bytes = states + (a.h_in ? states : 0);
  return w;
}

int check_linear(const xb_linear_attention_args* a) {
  XB_REQUIRE(a, XB_ERR_ARG, "xb_linear_attention: null arguments");
  XB_REQUIRE(a->dtype == XB_F32 || a->dtype == XB_F16 || a->dtype == XB_BF16, XB_ERR_UNSUPPORTED, "xb_linear_attention: dtype %d", a->dtype);
  XB_REQUIRE(a->H >= 1 && a->Hkv >= 1 && a->H % a->Hkv == 0 && a->dk >= 1 && a->dv >= 1, XB_ERR_ARG, "xb_linear_attention: %d heads on %d, of %d and %d",
             a->H, a->Hkv, a->dk, a->dv);
  XB_REQUIRE(a->dk <= LIN_MAX && a->dv <= LIN_MAX, XB_ERR_LIMIT, "xb_linear_attention: heads of %d and %d, at most %d", a->dk, a->dv, LIN_MAX);
  XB_REQUIRE(a->H <= 65535, XB_ERR_LIMIT, "xb_linear_attention: %d heads, at most 65535", a->H);
  XB_REQUIRE(a->rows >= 0 && a->batch >= 0 && a->longest >= 0, XB_ERR_ARG, "xb_linear_attention: %lld rows, %d lists, longest %lld", (long long)a->rows,
             a->batch, (long long)a->longest);
  XB_REQUIRE(a->batch <= MOST, XB_ERR_LIMIT, "xb_linear_attention: %d lists, at most 2^31 - 1024", a->batch);
  XB_REQUIRE(a->rows < ((int64_t)1 << 31), XB_ERR_LIMIT, "xb_linear_attention: %lld rows, fewer than 2^31", (long long)a->rows);
  XB_REQUIRE(a->offsets || a->batch == 0 || a->rows % a->batch == 0, XB_ERR_ARG, "xb_linear_attention: without offsets %d lists divide %lld rows", a->batch,
             (long long)a->rows);
  const bool states = a->h_in || a->h_out;
  XB_REQUIRE(!states || a->n_slots >= 0, XB_ERR_ARG, "xb_linear_attention: n_slots %d", a->n_slots);
  XB_REQUIRE(!states || a->slots || a->n_slots >= a->batch, XB_ERR_ARG, "xb_linear_attention: %d states for %d lists without slots", a->n_slots, a->batch);
  if (a->batch == 0) return 0;
  XB_REQUIRE(a->log_decay && (a->rows == 0 || (a->q && a->k && a->v && a->y)), XB_ERR_ARG, "xb_linear_attention: null tensor");
  XB_REQUIRE(a->q_row >= 0 && a->q_head >= 0 && a->k_row >= 0 && a->k_head >= 0 && a->v_row >= 0 && a->v_head >= 0 && a->y_row >= 0 && a->y_head >= 0,
             XB_ERR_ARG, "xb_linear_attention: a negative stride");
  return 0;
}

}  // namespace
}  // namespace xb

using namespace xb;

extern "C" size_t xb_linear_attention_workspace_bytes(const xb_linear_attention_args* a) {
  if (check_linear(a) != 0 || a->batch == 0) return 0;
  return linear_scratch(*a, linear_plan(*a)).bytes;
}

extern "C" int xb_linear_attention(const xb_linear_attention_args* a, void* workspace, size_t workspace_bytes, xb_stream_t s) {
  if (int rc = check_linear(a)) return rc;
  if (a->batch == 0) return 0;
  const LinearPlan plan = linear_plan(*a);
  const LinearScratch w = linear_scratch(*a, plan);
  XB_REQUIRE(w.bytes == 0 || (workspace && workspace_bytes >= w.bytes), XB_ERR_SCRATCH, "xb_linear_attention: workspace of %zu bytes, %zu needed",
             workspace_bytes, w.bytes);
  XB_REQUIRE(w.bytes == 0 || (reinterpret_cast<uintptr_t>(workspace) & 15) == 0, XB_ERR_ARG, "xb_linear_attention: the workspace is not on 16 bytes");
  const int64_t size = (int64_t)dtype_size(a->dtype);
  const Heads q = {a->q, a->q_row, a->q_head}, k = {a->k, a->k_row, a->k_head}, v = {a->v, a->v_row, a->v_head}, y = {a->y, a->y_row, a->y_head};
  XB_REQUIRE(heads_apart(y, a->H, a->dv, a->rows), XB_ERR_ARG, "xb_linear_attention: rows of y overlap one another");
  XB_REQUIRE(!heads_meet(q, a->H, a->dk, y, a->H, a->dv, a->rows, size) && !heads_meet(k, a->Hkv, a->dk, y, a->H, a->dv, a->rows, size) &&
                 !heads_meet(v, a->Hkv, a->dv, y, a->H, a->dv, a->rows, size), XB_ERR_ARG, "xb_linear_attention: y overlaps an input");
  const uintptr_t hi = reinterpret_cast<uintptr_t>(a->h_in), ho = reinterpret_cast<uintptr_t>(a->h_out);
  const uintptr_t states = (uintptr_t)a->n_slots * a->H * a->dk * a->dv * 4;
  XB_REQUIRE(!hi || !ho || hi == ho || hi + states <= ho || ho + states <= hi, XB_ERR_ARG, "xb_linear_attention: the two arrays of states overlap and are not one");
  LinearParams p = {};
  p.q = q; p.k = k; p.v = v; p.y = y;
  p.log_decay = a->log_decay; p.h_in = a->h_in; p.h_out = a->h_out;
  p.lists = {a->offsets, a->slots, a->rows, a->rows / a->batch, a->batch, a->n_slots};
  p.H = a->H; p.share = a->H / a->Hkv; p.dk = a->dk; p.dv = a->dv; p.scale = a->scale;
  p.vec_y = heads_whole(y, size, 2 * size) && a->dv % 2 == 0;
  auto unit = [&](const Heads& x) { return heads_whole(x, size, 16) ? 16 : heads_whole(x, size, 8) ? 8 : heads_whole(x, size, 4) ? 4 : 2; };
  p.unit_q = unit(q); p.unit_k = unit(k); p.unit_v = unit(v);
  p.vec_h = a->dv % 2 == 0 && (hi | ho) % 8 == 0;
  p.vec_e = a->dk * a->dv % 4 == 0;
  if (plan.order) p.order = static_cast<int*>(workspace);
  if (plan.chunk && w.bytes) {
    p.chunk = plan.chunk;
    p.n_ends = (int)(a->rows / plan.chunk);
    p.end = static_cast<float*>(workspace);
    p.first = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + w.first);
  }
  if (a->dtype == XB_F32) return linear_f32(p, plan, (cudaStream_t)s);
  if (a->dtype == XB_F16) return linear_f16(p, plan, (cudaStream_t)s);
  return linear_bf16(p, plan, (cudaStream_t)s);
}
