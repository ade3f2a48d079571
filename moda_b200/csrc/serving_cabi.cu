// C ABI of the operators that serve token by token: rotary positions, the paged KV cache's append, and the
// attention of one new token.  Declarations are in include/moda_b200.h.
#include "../../include/moda_b200.h"

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "cabi_common.cuh"
#include "profiler.cuh"
#include "rotary_kernels.cuh"
#include "paged_decode_kernel.cuh"

namespace {

using namespace moda;

// The sizes that the three operators share.
int check_sizes(const moda_problem* pr) {
  if (pr == nullptr) return MODA_ERR_NULL;
  if (pr->B < 1 || pr->T_kv < 1 || pr->H < 1 || pr->G < 1 || pr->L < 0) return MODA_ERR_SHAPE;
  if (pr->B > 65535 || pr->H > 65535 || pr->G > 65535) return MODA_ERR_SHAPE;
  if ((int64_t)pr->B * pr->T_kv > 0x7fffffff || (int64_t)pr->T_kv * pr->G > (int64_t)1 << 30) return MODA_ERR_SHAPE;
  if ((int64_t)pr->H * (pr->G + 1) > 1 << 24) return MODA_ERR_SHAPE;
  if (pr->D != 64 && pr->D != 128) return MODA_ERR_HEAD_DIM;
  if (pr->dtype != MODA_BF16 && pr->dtype != MODA_FP16) return MODA_ERR_DTYPE;
  return MODA_OK;
}
// rot may be NULL (no rotation) unless `required`.
int check_rotary(const moda_rotary* rot, bool required, int D, rotary::Args* out) {
  *out = rotary::Args{nullptr, 0, 0, 0, 1.f};
  if (rot == nullptr) return required ? MODA_ERR_NULL : MODA_OK;
  if (rot->inv_freq == nullptr) return MODA_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(rot->inv_freq) & 7u) return MODA_ERR_ALIGNMENT;
  if (rot->rotary_dim < 16 || rot->rotary_dim > D || rot->rotary_dim % 16 != 0) return MODA_ERR_SHAPE;
  *out = rotary::Args{rot->inv_freq, rot->rotary_dim, rot->interleaved != 0, 0, rot->scale};
  return MODA_OK;
}
int check_pages(const moda_problem* pr, const moda_paged_cache* c, paged::Pages* out) {
  if (c == nullptr || c->block_table == nullptr || c->seq_lens == nullptr) return MODA_ERR_NULL;
  if (c->num_pages < 1 || c->page_size < 1 || c->max_pages < 1 || c->table_stride < 0) return MODA_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(c->block_table) | reinterpret_cast<uintptr_t>(c->seq_lens)) & 3u) return MODA_ERR_ALIGNMENT;
  if (int rc = check_tensor(&c->k, true, c->num_pages, c->page_size, pr->H)) return rc;
  if (int rc = check_tensor(&c->v, true, c->num_pages, c->page_size, pr->H)) return rc;
  out->k = to_view(&c->k, c->num_pages, c->page_size, pr->H); out->v = to_view(&c->v, c->num_pages, c->page_size, pr->H);
  out->table = c->block_table; out->table_stride = c->table_stride; out->seq_lens = c->seq_lens;
  out->num_pages = c->num_pages; out->page_size = c->page_size; out->max_pages = c->max_pages;
  out->room = (int)std::min<int64_t>((int64_t)c->max_pages * c->page_size, 0x7fffffff);
  out->by_page = rotary::FastDiv((uint32_t)c->page_size);
  return MODA_OK;
}

// How the kernels that turn a token's vectors are divided: tokens a warp, vectors of a token that a warp takes, grid (tokens, shares of a
// token's vectors).  A warp has 32 / (D / 16) vectors of a token side by side, or where there are so few of them as many tokens; more than
// fill it at once where there would be more warps than run at once, since a warp that ends early costs more than one that takes
// steps.  65536 tokens of 5 vectors of 64: 19.9 us, 28.9 without; of 9 of 128 53.4 and 57.9; 4096 of 4 of 128 would be 3.5 for 3.3.
// A token that one warp can walk in a few steps stays whole (the sines are computed once); few tokens are shared by more warps, down to
// one step of kBatch vectors a lane, until there are some 16 warps for each SM.
struct TokenGrid { int tokens_a_warp, per_warp; dim3 grid; };
TokenGrid token_grid(int64_t tokens, int vectors, int D, int n_sm) {
  TokenGrid r{1, 0, dim3()};
  int lanes = 32 / (D / 16);
  while (r.tokens_a_warp < (D == 128 ? 2 : 4) && (vectors * 2 <= lanes || (vectors <= lanes * 3 && tokens > (int64_t)n_sm * 32 * r.tokens_a_warp))) {
    r.tokens_a_warp *= 2;
    lanes /= 2;
  }
  const int step = lanes * rotary::kBatch, most = (vectors + step - 1) / step;
  const int64_t a_block = (int64_t)(rotary::kThreads / 32) * r.tokens_a_warp;
  const int64_t shares = std::min<int64_t>(most, std::max<int64_t>(1, (int64_t)n_sm * 16 / std::max<int64_t>(tokens, 1)));
  r.per_warp = (int)((most + shares - 1) / shares) * step;
  r.grid = dim3((unsigned)((tokens + a_block - 1) / a_block), (unsigned)((vectors + r.per_warp - 1) / r.per_warp));
  return r;
}

// A launch that may begin when the grid before it has ended but not flushed what it wrote: the kernels here wait for that themselves, before
// anything else.  A cluster of `cluster` CTAs.
template <typename P>
cudaError_t launch(void (*kern)(P), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t st, const P& p) {
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, p);
}
template <typename T, int D> cudaError_t launch_rotary(const rotary::RotaryParams& p, const TokenGrid& g, cudaStream_t st) {
  auto kern = rotary::rotary_kernel<T, D, 1>;
  if (g.tokens_a_warp == 2) kern = rotary::rotary_kernel<T, D, 2>;
  if constexpr (D == 64) if (g.tokens_a_warp == 4) kern = rotary::rotary_kernel<T, D, 4>;
  return launch(kern, g.grid, rotary::kThreads, 0, 1, st, p);
}
template <typename T, int D> cudaError_t launch_append(const paged::AppendParams& p, const TokenGrid& g, cudaStream_t st) {
  auto kern = paged::append_kernel<T, D, 1>;
  if (g.tokens_a_warp == 2) kern = paged::append_kernel<T, D, 2>;
  if constexpr (D == 64) if (g.tokens_a_warp == 4) kern = paged::append_kernel<T, D, 4>;
  return launch(kern, g.grid, rotary::kThreads, 0, 1, st, p);
}

int append(const moda_problem* pr, const moda_tensor4* k, const moda_tensor4* v, const paged::Pages& pages, const int32_t* lengths,
           const rotary::Args& rot, int n_sm, cudaStream_t st) {
  paged::AppendParams p{};
  p.k = to_view(k, pr->B, pr->T_kv, pr->H); p.v = to_view(v, pr->B, pr->T_kv, pr->H); p.pages = pages; p.lengths = lengths; p.rot = rot;
  p.B = pr->B; p.T = pr->T_kv; p.H = pr->H; p.by_t = rotary::FastDiv((uint32_t)pr->T_kv);
  const TokenGrid grid = token_grid((int64_t)pr->B * pr->T_kv, 2 * pr->H, pr->D, n_sm);
  p.per_warp = grid.per_warp;
  cudaError_t e;
  {
    prof::Scope ps(prof::kPagedAppend, st);
    const bool bf = pr->dtype == MODA_BF16;
    if (pr->D == 128) e = bf ? launch_append<__nv_bfloat16, 128>(p, grid, st) : launch_append<__half, 128>(p, grid, st);
    else e = bf ? launch_append<__nv_bfloat16, 64>(p, grid, st) : launch_append<__half, 64>(p, grid, st);
  }
  MODA_CUDA(e);
  g_last_launches += 1;
  return MODA_OK;
}

// The decoding kernel, made ready once a device (the calls cost the host 0.4 us each).
template <typename T, int D> int ready_decode(int device) {
  static std::atomic<uint64_t> done{0};
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if ((done.load(std::memory_order_relaxed) & bit) != 0) return MODA_OK;
  if (int rc = opt_in_smem(paged::decode_kernel<T, D>, paged::smem_bytes<D>())) return rc;
  MODA_CUDA(cudaFuncSetAttribute(paged::decode_kernel<T, D>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  done.fetch_or(bit, std::memory_order_relaxed);
  return MODA_OK;
}

// How many clusters of 2^log_size CTAs the device, which is current, runs at once: fewer than its CTAs make, as a cluster lies in one
// group of SMs and the groups differ in size (2 CTAs an SM: 14 clusters of 16, 33 of 8, 71 of 4).  Asked once a device.
constexpr int kMostClusterLog = 4;
template <int D> int clusters_at_once(int device, int log_size, int* out) {
  static std::atomic<int> known[64][kMostClusterLog + 1];       // and one more; 0: not asked yet
  if (device < 64) {
    const int k = known[device][log_size].load(std::memory_order_relaxed);
    if (k != 0) { *out = k - 1; return MODA_OK; }
  }
  if (int rc = ready_decode<__nv_bfloat16, D>(device)) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(1u << log_size);
  cfg.blockDim = dim3(paged::kThreads);
  cfg.dynamicSmemBytes = paged::smem_bytes<D>();
  cudaLaunchAttribute size{};
  size.id = cudaLaunchAttributeClusterDimension;
  size.val.clusterDim.x = 1u << log_size;
  size.val.clusterDim.y = size.val.clusterDim.z = 1;
  cfg.attrs = &size;
  cfg.numAttrs = 1;
  MODA_CUDA(cudaOccupancyMaxActiveClusters(out, paged::decode_kernel<__nv_bfloat16, D>, &cfg));
  if (device < 64) known[device][log_size].store(*out + 1, std::memory_order_relaxed);
  return MODA_OK;
}

// The decoding kernels count keys, and the tiles of one head of all sequences, in 31 bits.
bool too_many_keys(int64_t B, int64_t most_keys) {
  return most_keys > 0x7fffffff - 64 || B * (most_keys / paged::kTile + 2 + paged::unit_cost(paged::kWarps)) > 0x7fffffff;
}

// How a decoding call is divided.  The lengths are known on the device alone; what is known here is how long a sequence may be, by
// the width of its table (and L depth rows).  A table wider than its sequences costs the one-launch forms: one step over 4095 rows
// of 8 heads 12.0 us, 14.6 where the table has 131072 positions, 60 sequences of 60 rows 8.2 and 12.5.  Depth rows of several positions count as
// those of one here: a choice of fewer CTAs for them than they could use, not of a wrong result.
struct Division { int ctas, cluster; };
int divide(const moda_problem* pr, int64_t most_rows, Division* out) {
  const int n_sm = sm_count(pr->device);
  if (n_sm <= 0) return cuda_fail(cudaErrorInvalidDevice);
  const int64_t heads = (int64_t)pr->H * ((pr->G + paged::kQ - 1) / paged::kQ), units = pr->B * heads;
  const int64_t tiles = std::max<int64_t>(1, (most_rows + paged::kTile - 1) / paged::kTile + (pr->L + paged::kTile - 1) / paged::kTile), slots = (int64_t)n_sm * (pr->D == 128 ? paged::ctas_per_sm<128>() : paged::ctas_per_sm<64>());
  // clusters that have to wait for others cost a round: 16 sequences' heads of 2000 rows 14.4 us by 16, 9.5 by 8
  int log_size = 0;
  for (int next = 1; next <= kMostClusterLog && ((int64_t)paged::kWarps << next) <= tiles; ++next) {
    int most = 0;
    if (int rc = pr->D == 128 ? clusters_at_once<128>(pr->device, next, &most) : clusters_at_once<64>(pr->device, next, &most)) return rc;
    if (units > most) break;
    log_size = next;
  }
  // A cluster's CTAs may have up to 32 tiles of cached and one position's depth rows each, or 52 times the part of the device that they fill if that is more: an even division
  // fills all of it, but takes a second launch.  Rows as long as the table allows, and half of that on average, D = 128, 8 heads (128 CTAs of 296), 28 tiles:
  // 13.2 and 11.4 us against 13.8 and 12.6, 44 tiles: 17.7 and 14.7 against 15.3 and 14.2; 32 heads (256 CTAs), 44 tiles: 19.3 and 16.5
  // against 24.3 and 15.4; 296 heads, 49 tiles: 22.6 and 17.5 against 26.4 and 20.5
  const int cluster = 1 << log_size;
  const int64_t ctas = units * cluster;
  if (ctas <= slots && tiles * slots <= cluster * std::max(32 * slots, 52 * ctas)) {
    *out = {(int)ctas, cluster};
    return MODA_OK;
  }
  // more units than CTAs, and none long: whole ones to warps, without a division by lengths and without parts to join.  1000 units of up
  // to 128 rows, D = 128: 14.0 us against 22.4; 480 of up to 384, too long for it: 25.6 against 19.7
  if (units > slots && tiles <= paged::kShort) {
    *out = {(int)std::min<int64_t>(slots, (units + paged::kWarps - 1) / paged::kWarps), paged::kByWarps};
    return MODA_OK;
  }
  const int cost = paged::unit_cost(paged::kWarps), least = paged::least_places(paged::kWarps);
  *out = {(int)std::min<int64_t>(slots, std::max<int64_t>(1, (units * (tiles + cost) + least - 1) / least)), 0};
  return MODA_OK;
}
// Scratch of an evenly divided call: which units are shared, their parts' maxima and sums, their parts.
size_t parts_bytes(int n) { return ((size_t)n * paged::kWarps * sizeof(int2) + 255) & ~(size_t)255; }
size_t rows_of_teams(int n, int G) { return (size_t)n * paged::kWarps * 2 * std::min(G, paged::kQ); }
size_t ml_bytes(int n, int G) { return rows_of_teams(n, G) * sizeof(float2); }      // a multiple of 64, so that the parts are aligned
size_t decode_scratch(int n, int G, int D) { return parts_bytes(n) + ml_bytes(n, G) + rows_of_teams(n, G) * D * sizeof(float); }

template <typename T, int D> int decode(const paged::DecodeParams& p, int n_cta, int device, cudaStream_t st) {
  auto kern = paged::decode_kernel<T, D>;
  constexpr size_t smem = paged::smem_bytes<D>();
  if (int rc = ready_decode<T, D>(device)) return rc;
  cudaError_t e;
  {
    prof::Scope ps(prof::kPagedDecode, st);
    e = launch(kern, dim3(n_cta), paged::kThreads, smem, std::max(p.cluster, 1), st, p);
  }
  MODA_CUDA(e);
  g_last_launches += 1;
  if (p.cluster != 0) return MODA_OK;
  {
    prof::Scope ps(prof::kPagedJoin, st);
    e = launch(paged::join_kernel<T, D>, dim3(n_cta, std::min(p.G, paged::kQ)), paged::kJoinWarps * 32, 0, 1, st, p);
  }
  MODA_CUDA(e);
  g_last_launches += 1;
  return MODA_OK;
}

}  // namespace

namespace moda {
// The word of the paged kernels (paged::g_wrong) of the current device: read, and cleared when set.
int read_paged_status(int* out) {
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, paged::g_wrong, sizeof(int));
  if (e == cudaSuccess && v != 0) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(paged::g_wrong, &zero, sizeof(int));
  }
  *out = v;
  return (int)e;
}
}  // namespace moda

extern "C" {

int moda_b200_rotary(const moda_problem* prob, const moda_rotary* rot, const moda_positions* positions, int inverse,
                     const moda_tensor4* q, const moda_tensor4* k, const moda_tensor4* q_out, const moda_tensor4* k_out, void* stream) {
  if (int rc = check_sizes(prob)) return rc;
  const int64_t B = prob->B, T = prob->T_kv, H = prob->H;
  const bool has_k = k != nullptr && k->data != nullptr;
  if (int rc = check_tensor(q, true, B, T * prob->G, H)) return rc;
  if (int rc = check_tensor(k, false, B, T, H)) return rc;
  if (int rc = check_tensor(q_out, true, B, T * prob->G, H)) return rc;
  if (int rc = check_tensor(k_out, has_k, B, T, H)) return rc;
  rotary::RotaryParams p{};
  if (int rc = check_rotary(rot, true, prob->D, &p.rot)) return rc;
  p.rot.inverse = inverse != 0;
  if (positions != nullptr) {
    if (reinterpret_cast<uintptr_t>(positions->data) & (positions->is_int64 ? 7u : 3u)) return MODA_ERR_ALIGNMENT;
    p.pos = rotary::Positions{positions->data, positions->stride_b, positions->stride_t, positions->offset, positions->is_int64 != 0};
  }
  p.q = to_view(q, B, T * prob->G, H); p.k = to_view(has_k ? k : nullptr, B, T, H);
  p.q_out = to_view(q_out, B, T * prob->G, H); p.k_out = to_view(has_k ? k_out : nullptr, B, T, H);
  p.B = prob->B; p.T = prob->T_kv; p.H = prob->H; p.G = prob->G;
  p.vectors = prob->H * (prob->G + (has_k ? 1 : 0));
  p.by_h = rotary::FastDiv((uint32_t)prob->H); p.by_t = rotary::FastDiv((uint32_t)prob->T_kv);
  DeviceGuard guard(prob->device);
  if (!guard.ok) return cuda_fail(guard.err);
  g_last_launches = 0;
  const int n_sm = sm_count(prob->device);
  if (n_sm <= 0) return cuda_fail(cudaErrorInvalidDevice);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const TokenGrid grid = token_grid(B * T, p.vectors, prob->D, n_sm);
  p.per_warp = grid.per_warp;
  cudaError_t e;
  {
    prof::Scope ps(prof::kRotary, st);
    const bool bf = prob->dtype == MODA_BF16;
    if (prob->D == 128) e = bf ? launch_rotary<__nv_bfloat16, 128>(p, grid, st) : launch_rotary<__half, 128>(p, grid, st);
    else e = bf ? launch_rotary<__nv_bfloat16, 64>(p, grid, st) : launch_rotary<__half, 64>(p, grid, st);
  }
  MODA_CUDA(e);
  g_last_launches += 1;
  return MODA_OK;
}

int moda_b200_paged_append(const moda_problem* prob, const moda_tensor4* k, const moda_tensor4* v, const moda_paged_cache* cache,
                           const int32_t* lengths, const moda_rotary* rot, void* stream) {
  if (int rc = check_sizes(prob)) return rc;
  if (int rc = check_tensor(k, true, prob->B, prob->T_kv, prob->H)) return rc;
  if (int rc = check_tensor(v, true, prob->B, prob->T_kv, prob->H)) return rc;
  if (reinterpret_cast<uintptr_t>(lengths) & 3u) return MODA_ERR_ALIGNMENT;
  paged::Pages pages;
  rotary::Args turn;
  if (int rc = check_pages(prob, cache, &pages)) return rc;
  if (int rc = check_rotary(rot, false, prob->D, &turn)) return rc;
  DeviceGuard guard(prob->device);
  if (!guard.ok) return cuda_fail(guard.err);
  g_last_launches = 0;
  const int n_sm = sm_count(prob->device);
  if (n_sm <= 0) return cuda_fail(cudaErrorInvalidDevice);
  return append(prob, k, v, pages, lengths, turn, n_sm, reinterpret_cast<cudaStream_t>(stream));
}

int moda_b200_paged_decode_workspace_bytes(const moda_problem* prob, const moda_paged_cache* cache, size_t* bytes) {
  if (bytes == nullptr || cache == nullptr) return MODA_ERR_NULL;
  if (int rc = check_sizes(prob)) return rc;
  if (cache->max_pages < 1 || cache->page_size < 1) return MODA_ERR_SHAPE;
  if (too_many_keys(prob->B, (int64_t)cache->max_pages * cache->page_size)) return MODA_ERR_TOO_LARGE;
  DeviceGuard guard(prob->device);
  if (!guard.ok) return cuda_fail(guard.err);
  Division div;
  if (int rc = divide(prob, (int64_t)cache->max_pages * cache->page_size, &div)) return rc;
  *bytes = div.cluster != 0 ? 0 : decode_scratch(div.ctas, prob->G, prob->D);
  return MODA_OK;
}

int moda_b200_paged_decode(const moda_problem* prob, const moda_tensor4* q, const moda_paged_cache* cache, const moda_tensor4* k,
                           const moda_tensor4* v, const moda_tensor4* k_copy, const moda_tensor4* v_copy, const moda_depth_rows* depth,
                           const moda_rotary* rot, const moda_tensor4* o, float* lse, void* workspace, size_t workspace_bytes,
                           void* stream) {
  if (int rc = check_sizes(prob)) return rc;
  if (prob->T_kv != 1 || !(prob->scale == prob->scale)) return MODA_ERR_SHAPE;
  const int64_t B = prob->B, H = prob->H, query_blocks = (prob->G + paged::kQ - 1) / paged::kQ;
  if (B * H * query_blocks > 0x7fffffff) return MODA_ERR_SHAPE;
  if (int rc = check_tensor(q, true, B, prob->G, H)) return rc;
  if (int rc = check_tensor(o, true, B, prob->G, H)) return rc;
  const bool own_key = k != nullptr && k->data != nullptr;
  if (int rc = check_tensor(k, false, B, 1, H)) return rc;
  if (int rc = check_tensor(v, own_key, B, 1, H)) return rc;
  if (k_copy != nullptr && !own_key) return MODA_ERR_NULL;
  if (int rc = check_tensor(k_copy, false, B, 1, H)) return rc;
  if (int rc = check_tensor(v_copy, k_copy != nullptr && k_copy->data != nullptr, B, 1, H)) return rc;
  if (lse == nullptr) return MODA_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(lse) & 3u) return MODA_ERR_ALIGNMENT;
  paged::DecodeParams p{};
  if (int rc = check_pages(prob, cache, &p.pages)) return rc;
  if (int rc = check_rotary(rot, false, prob->D, &p.rot)) return rc;
  if (depth != nullptr && prob->L > 0) {
    const int64_t P = depth->positions_per_sequence;
    if (P < 1 || P * prob->L > (int64_t)1 << 30) return MODA_ERR_SHAPE;
    if (int rc = check_tensor(&depth->k, true, B, prob->L, H)) return rc;
    if (int rc = check_tensor(&depth->v, true, B, prob->L, H)) return rc;
    if (P > 1 && (depth->k_stride_position <= 0 || depth->k_stride_position % 8 || depth->v_stride_position <= 0 || depth->v_stride_position % 8))
      return MODA_ERR_ALIGNMENT;
    if (reinterpret_cast<uintptr_t>(depth->positions_seen) & 3u) return MODA_ERR_ALIGNMENT;
    p.kd = to_view(&depth->k, B, prob->L, H); p.vd = to_view(&depth->v, B, prob->L, H);
    p.kd_sp = P > 1 ? depth->k_stride_position : 0; p.vd_sp = P > 1 ? depth->v_stride_position : 0;
    p.depth_positions = depth->positions_seen; p.P = (int)P; p.L = prob->L;
    p.by_L = rotary::FastDiv((uint32_t)prob->L);
  } else if (prob->L > 0) {
    return MODA_ERR_NULL;
  } else {
    p.kd = p.vd = View{p.pages.k.ptr, 0, 0, 0};      // no row of it is read
  }
  if (too_many_keys(B, (int64_t)p.pages.max_pages * p.pages.page_size + own_key + (int64_t)p.P * p.L)) return MODA_ERR_TOO_LARGE;
  DeviceGuard guard(prob->device);
  if (!guard.ok) return cuda_fail(guard.err);
  Division div;
  if (int rc = divide(prob, (int64_t)p.pages.max_pages * p.pages.page_size, &div)) return rc;
  // depth rows of several positions may make units long after all: one to a CTA then, which needs no scratch either
  if (div.cluster == paged::kByWarps && p.P > 1 && (int64_t)p.P * p.L > (int64_t)paged::kShort * paged::kTile - (int64_t)p.pages.max_pages * p.pages.page_size)
    div = {(int)(B * H * query_blocks), 1};
  const int n_cta = div.ctas;
  p.cluster = div.cluster;
  if (p.cluster == 0) {
    if (workspace == nullptr || workspace_bytes < decode_scratch(n_cta, prob->G, prob->D)) return MODA_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(workspace) & 255u) return MODA_ERR_ALIGNMENT;
  }
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  p.q = to_view(q, B, prob->G, H); p.o = to_view(o, B, prob->G, H); p.lse = lse;
  p.B = prob->B; p.H = prob->H; p.G = prob->G; p.rows = std::min(prob->G, paged::kQ);
  p.k = to_view(own_key ? k : nullptr, B, 1, H); p.v = to_view(own_key ? v : nullptr, B, 1, H);
  p.k_copy = to_view(own_key ? k_copy : nullptr, B, 1, H); p.v_copy = to_view(own_key ? v_copy : nullptr, B, 1, H);
  p.copy_all = p.k_copy.ptr != nullptr && cache->copy_all != 0;
  p.scale_log2 = prob->scale * 1.4426950408889634f;
  p.parts = reinterpret_cast<int2*>(ws);
  p.ml = reinterpret_cast<float2*>(ws + parts_bytes(n_cta));
  p.acc = reinterpret_cast<float*>(ws + parts_bytes(n_cta) + ml_bytes(n_cta, prob->G));
  g_last_launches = 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool bf = prob->dtype == MODA_BF16;
  if (prob->D == 128) return bf ? decode<__nv_bfloat16, 128>(p, n_cta, prob->device, st) : decode<__half, 128>(p, n_cta, prob->device, st);
  return bf ? decode<__nv_bfloat16, 64>(p, n_cta, prob->device, st) : decode<__half, 64>(p, n_cta, prob->device, st);
}

}  // extern "C"
