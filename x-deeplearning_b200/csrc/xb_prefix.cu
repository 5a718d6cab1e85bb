// Softmax attention of lists that share a prefix: arguments and launches (formulas in xdlb200.h, kernels in xb_prefix.cuh).
#include "xb_prefix.cuh"

#include "xb_gemm_tile.cuh"

namespace xb {
namespace {

constexpr int32_t MOST = INT32_MAX - 1023;
constexpr int PFX_MAX_D = 128;
constexpr float LOG2_E = 1.4426950408889634f;

struct PrefixScratch {
  size_t own_weight, groups, begins, records, part, part_ml, kept, bytes;      // (the items lie first)
  int max_items, ctas, part_rows, n_groups;
};
// items that a call may have: two tiles each, and one more for every prefix
int64_t most_items(const xb_prefix_attention_args& a) {
  return a.rows / (2 * (PFX_ROWS / (a.H / a.Hkv))) + std::min<int64_t>(a.rows, a.prefixes == 0 ? 1 : (int64_t)a.prefixes + 2);
}
PrefixScratch prefix_scratch(const xb_prefix_attention_args& a) {
  auto align256 = [](size_t n) { return (n + 255) / 256 * 256; };
  PrefixScratch w;
  const int64_t share = a.H / a.Hkv, R = PFX_ROWS / share;
  w.ctas = std::min(std::max(sm_count(), 1), JOIN_MOST / PFX_SLOTS);
  w.n_groups = a.prefixes == 0 ? 1 : a.prefixes + 2;
  w.max_items = (int)most_items(a);
  w.part_rows = (int)std::min<int64_t>(2 * R, a.rows) * (int)share;
  const size_t slots = (size_t)w.ctas * PFX_SLOTS;
  w.own_weight = align256((size_t)w.max_items * sizeof(PrefixItem));
  w.groups = w.own_weight + align256(((size_t)w.max_items + 1) * 8);
  w.begins = w.groups + align256(((size_t)w.n_groups + 1) * sizeof(PrefixGroup));
  w.records = w.begins + align256(((size_t)w.ctas + 1) * sizeof(PrefixAt));
  w.part = w.records + align256(slots * sizeof(PrefixRecord));
  w.part_ml = w.part + align256(slots * w.part_rows * a.d * 4);
  w.kept = w.part_ml + align256(slots * w.part_rows * 8);
  // (an item has no more blocks than this)
  const bool long_items = (a.prefix_rows + PFX_KEYS - 1) / PFX_KEYS + (a.own_rows + PFX_KEYS - 1) / PFX_KEYS > PFX_KEPT;
  w.bytes = w.kept + (long_items ? (size_t)w.ctas * 2 * PFX_ROWS * a.d * 4 : 0);
  return w;
}

int check_prefix(const xb_prefix_attention_args* a) {
  XB_REQUIRE(a, XB_ERR_ARG, "xb_prefix_attention: null arguments");
  XB_REQUIRE(a->dtype == XB_F16 || a->dtype == XB_BF16, XB_ERR_UNSUPPORTED, "xb_prefix_attention: dtype %d, fp16 or bf16", a->dtype);
  XB_REQUIRE(a->H >= 1 && a->Hkv >= 1 && a->H % a->Hkv == 0 && a->d >= 1, XB_ERR_ARG, "xb_prefix_attention: %d heads on %d, of %d", a->H, a->Hkv, a->d);
  XB_REQUIRE(a->d % 8 == 0, XB_ERR_UNSUPPORTED, "xb_prefix_attention: heads of %d, whole pieces of 8", a->d);
  XB_REQUIRE(a->d <= PFX_MAX_D && a->H / a->Hkv <= PFX_ROWS && a->H <= 65535, XB_ERR_LIMIT, "xb_prefix_attention: %d heads on %d of %d, at most 65535, 128 on one, of 128",
             a->H, a->Hkv, a->d);
  XB_REQUIRE(a->rows >= 0 && a->own_rows >= 0 && a->prefix_rows >= 0 && a->batch >= 0 && a->prefixes >= 0, XB_ERR_ARG, "xb_prefix_attention: a negative size");
  // (groups and items are counted in 32 bits, a block of 1024 threads at a time)
  XB_REQUIRE(a->batch <= MOST && a->prefixes <= MOST - 1024, XB_ERR_LIMIT, "xb_prefix_attention: %d lists, at most 2^31 - 1024, %d prefixes, at most 2^31 - 2048", a->batch,
             a->prefixes);
  constexpr int64_t ROWS = ((int64_t)1 << 31) - 1024;      // (blocks of 128 rows are counted in 32 bits)
  XB_REQUIRE(a->rows <= ROWS && a->own_rows <= ROWS && a->prefix_rows <= ROWS, XB_ERR_LIMIT, "xb_prefix_attention: %lld, %lld and %lld rows, at most 2^31 - 1024",
             (long long)a->rows, (long long)a->own_rows, (long long)a->prefix_rows);
  XB_REQUIRE(most_items(*a) <= MOST, XB_ERR_LIMIT, "xb_prefix_attention: %lld rows and %d prefixes are too many for one call", (long long)a->rows, a->prefixes);
  XB_REQUIRE(a->scale > 0 && a->scale <= 3.0e38f, XB_ERR_ARG, "xb_prefix_attention: scale %g", (double)a->scale);
  if (a->batch == 0 || a->rows == 0) return 0;
  XB_REQUIRE(a->offsets || a->rows % a->batch == 0, XB_ERR_ARG, "xb_prefix_attention: without offsets %d lists divide %lld rows", a->batch, (long long)a->rows);
  XB_REQUIRE(!a->k == !a->v && !a->prefix_k == !a->prefix_v, XB_ERR_ARG, "xb_prefix_attention: keys without values");
  XB_REQUIRE(a->q && a->y && (a->own_rows == 0 || a->k) && (a->prefix_rows == 0 || a->prefix_k), XB_ERR_ARG, "xb_prefix_attention: null tensor");
  XB_REQUIRE(a->own_rows == 0 || a->own_offsets || a->own_rows == a->rows, XB_ERR_ARG, "xb_prefix_attention: without offsets of their own %lld own rows beside %lld",
             (long long)a->own_rows, (long long)a->rows);
  XB_REQUIRE(a->prefix_rows == 0 || a->prefixes > 0, XB_ERR_ARG, "xb_prefix_attention: rows of no prefix");
  XB_REQUIRE(a->prefixes == 0 || a->members || a->batch % a->prefixes == 0, XB_ERR_ARG, "xb_prefix_attention: without members %d prefixes divide %d lists", a->prefixes, a->batch);
  XB_REQUIRE(a->prefixes == 0 || a->prefix_offsets || a->prefix_rows % a->prefixes == 0, XB_ERR_ARG,
             "xb_prefix_attention: without offsets %d prefixes divide %lld rows", a->prefixes, (long long)a->prefix_rows);
  const struct { const char* name; const void* at; int64_t row, head, rows; int n; } in[] = {
      {"q", a->q, a->q_row, a->q_head, a->rows, a->H}, {"k", a->k, a->k_row, a->k_head, a->own_rows, a->Hkv}, {"v", a->v, a->v_row, a->v_head, a->own_rows, a->Hkv},
      {"prefix_k", a->prefix_k, a->prefix_k_row, a->prefix_k_head, a->prefix_rows, a->Hkv}, {"prefix_v", a->prefix_v, a->prefix_v_row, a->prefix_v_head, a->prefix_rows, a->Hkv}};
  for (const auto& t : in) {
    if (t.rows == 0) continue;
    const bool rows = t.rows == 1 || (t.row >= a->d && t.row % 8 == 0), heads = t.n == 1 || (t.head >= a->d && t.head % 8 == 0);
    XB_REQUIRE(rows && heads && (reinterpret_cast<uintptr_t>(t.at) & 15) == 0, XB_ERR_UNSUPPORTED,
               "xb_prefix_attention: rows of %s start on 16 bytes, with strides of at least %d in whole pieces of 8 (%lld, %lld)", t.name, a->d, (long long)t.row, (long long)t.head);
    XB_REQUIRE(t.row < ((int64_t)1 << 38) && t.head < ((int64_t)1 << 38), XB_ERR_LIMIT, "xb_prefix_attention: strides of %s of %lld and %lld", t.name, (long long)t.row,
               (long long)t.head);
  }
  XB_REQUIRE(a->y_row >= 0 && a->y_head >= 0, XB_ERR_ARG, "xb_prefix_attention: a negative stride");
  return 0;
}

// rows of heads as a tensor map: boxes of 64 elements, `share` heads that read one head of keys, and `box_rows` rows
int make_heads_map(CUtensorMap* map, int dtype, const void* at, int64_t row, int64_t head, int64_t rows, int heads, int share, int d, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  XB_REQUIRE(fn, XB_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  // (a stride over one row or head says nothing)
  const cuuint64_t by_head = (cuuint64_t)(heads > 1 ? head : d) * 2, by_row = (cuuint64_t)(rows > 1 ? row : (int64_t)d * heads) * 2;
  const bool shared = share > 0;
  const cuuint64_t dims_q[4] = {(cuuint64_t)d, (cuuint64_t)share, (cuuint64_t)(shared ? heads / share : 1), (cuuint64_t)rows}, strides_q[3] = {by_head, by_head * share, by_row};
  const cuuint64_t dims_k[3] = {(cuuint64_t)d, (cuuint64_t)heads, (cuuint64_t)rows}, strides_k[2] = {by_head, by_row};
  const cuuint32_t box_q[4] = {64, (cuuint32_t)share, 1, (cuuint32_t)box_rows}, box_k[3] = {64, 1, (cuuint32_t)box_rows}, ones[4] = {1, 1, 1, 1};
  const CUresult r = fn(map, dtype == XB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, shared ? 4 : 3, const_cast<void*>(at),
                        shared ? dims_q : dims_k, shared ? strides_q : strides_k, shared ? box_q : box_k, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  XB_REQUIRE(r == CUDA_SUCCESS, XB_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d", (int)r);
  return 0;
}

template <bool BF16, int DP>
int launch_prefix(const CUtensorMap (&m)[5], const PrefixParams& p, cudaStream_t s) {
  static PerDeviceOnce once;
  XB_SET_MAX_SMEM_ONCE(once, PrefixShape<DP>::SMEM, (const void*)prefix_attention_kernel<BF16, DP>);
  // (a thread a group, an item and a CTA, while there are threads)
  const int want = std::max({p.n_groups, p.max_items, p.ctas + 1});
  launch_dependent(prefix_plan_kernel, 1, (unsigned)std::min((want + 31) / 32 * 32, PLAN_THREADS), 0, s, p);
  if (int rc = check_launch("prefix_plan_kernel")) return rc;
  launch_dependent(prefix_attention_kernel<BF16, DP>, (unsigned)p.ctas, PFX_THREADS, PrefixShape<DP>::SMEM, s, m[0], m[1], m[2], m[3], m[4], p);
  if (int rc = check_launch("prefix_attention_kernel")) return rc;
  launch_dependent(prefix_join_kernel<BF16>, (unsigned)p.ctas * 4, JOIN_THREADS, 0, s, p);
  return check_launch("prefix_join_kernel");
}

}  // namespace

int prefix_status(int* out) { return umma::read_status_word(out); }
int prefix_clear_status() { return umma::clear_status_word(); }
int prefix_set_status_mirror(int* p) { return umma::set_status_mirror(p); }
}  // namespace xb

using namespace xb;

extern "C" size_t xb_prefix_attention_workspace_bytes(const xb_prefix_attention_args* a) {
  if (check_prefix(a) != 0 || a->batch == 0 || a->rows == 0) return 0;
  return prefix_scratch(*a).bytes;
}

extern "C" int xb_prefix_attention(const xb_prefix_attention_args* a, void* workspace, size_t workspace_bytes, xb_stream_t s) {
  if (int rc = check_prefix(a)) return rc;
  if (a->batch == 0 || a->rows == 0) return 0;
  const PrefixScratch w = prefix_scratch(*a);
  XB_REQUIRE(workspace && workspace_bytes >= w.bytes, XB_ERR_SCRATCH, "xb_prefix_attention: workspace of %zu bytes, %zu needed", workspace_bytes, w.bytes);
  XB_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, XB_ERR_ARG, "xb_prefix_attention: the workspace is not on 16 bytes");
  const Heads q = {a->q, a->q_row, a->q_head}, k = {a->k, a->k_row, a->k_head}, v = {a->v, a->v_row, a->v_head}, y = {a->y, a->y_row, a->y_head};
  const Heads pk = {a->prefix_k, a->prefix_k_row, a->prefix_k_head}, pv = {a->prefix_v, a->prefix_v_row, a->prefix_v_head};
  XB_REQUIRE(heads_apart(y, a->H, a->d, a->rows), XB_ERR_ARG, "xb_prefix_attention: rows of y overlap one another");
  auto over = [&](const Heads& x, int n, int64_t rows) {
    if (rows == a->rows) return heads_meet(x, n, a->d, y, a->H, a->d, rows, 2);
    return heads_meet_ends(x, n, a->d, rows, y, a->H, a->d, a->rows, 2);
  };
  XB_REQUIRE(!over(q, a->H, a->rows) && !over(k, a->Hkv, a->own_rows) && !over(v, a->Hkv, a->own_rows) && !over(pk, a->Hkv, a->prefix_rows) &&
                 !over(pv, a->Hkv, a->prefix_rows), XB_ERR_ARG, "xb_prefix_attention: y overlaps an input");
  PrefixParams p = {};
  p.lists = {a->offsets, nullptr, a->rows, a->rows / a->batch, a->batch, 0};
  p.own = a->own_offsets ? Lists{a->own_offsets, nullptr, a->own_rows, 0, a->batch, 0} : p.lists;
  if (a->own_rows == 0) p.own.rows = 0;
  p.members = a->members; p.prefix_offsets = a->prefix_offsets; p.prefix_rows = a->prefix_rows; p.prefixes = a->prefixes;
  p.H = a->H; p.Hkv = a->Hkv; p.share = a->H / a->Hkv; p.R = PFX_ROWS / p.share; p.d = a->d;
  p.scale = a->scale * LOG2_E;
  p.y = y; p.v = v;
  p.vec_y = heads_whole(y, 2, 16);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.items = reinterpret_cast<PrefixItem*>(ws);
  p.own_weight = reinterpret_cast<int64_t*>(ws + w.own_weight);
  p.groups = reinterpret_cast<PrefixGroup*>(ws + w.groups);
  p.begins = reinterpret_cast<PrefixAt*>(ws + w.begins);
  p.records = reinterpret_cast<PrefixRecord*>(ws + w.records);
  p.part = reinterpret_cast<float4*>(ws + w.part);
  p.part_ml = reinterpret_cast<float2*>(ws + w.part_ml);
  p.kept = w.bytes > w.kept ? reinterpret_cast<float4*>(ws + w.kept) : nullptr;
  p.max_items = w.max_items; p.ctas = w.ctas; p.n_groups = w.n_groups; p.part_rows = w.part_rows;
  CUtensorMap m[5];
  if (int rc = make_heads_map(&m[0], a->dtype, a->q, a->q_row, a->q_head, a->rows, a->H, p.share, a->d, p.R)) return rc;
  // (a map that no block of keys is read by is that of the queries)
  const struct { const Heads* t; int64_t rows; } in[4] = {{&k, a->own_rows}, {&v, a->own_rows}, {&pk, a->prefix_rows}, {&pv, a->prefix_rows}};
  for (int i = 0; i < 4; ++i) {
    m[1 + i] = m[0];
    if (in[i].rows == 0) continue;
    if (int rc = make_heads_map(&m[1 + i], a->dtype, in[i].t->at, in[i].t->row, in[i].t->head, in[i].rows, a->Hkv, 0, a->d, PFX_KEYS)) return rc;
  }
  const bool wide = a->d > 64;
  if (a->dtype == XB_BF16) return wide ? launch_prefix<true, 128>(m, p, (cudaStream_t)s) : launch_prefix<true, 64>(m, p, (cudaStream_t)s);
  return wide ? launch_prefix<false, 128>(m, p, (cudaStream_t)s) : launch_prefix<false, 64>(m, p, (cudaStream_t)s);
}
