// Attention over a paged K / V cache: ragged batches of query tokens, 16- or 32-bit pages or pages
// of 4-bit codes (the rows kv_append.cu writes).
//
// Sequence z has lengths[z] keys and query tokens cu_seqlens_q[z] .. cu_seqlens_q[z+1] (without
// cu_seqlens_q: T / Z each).  Token i of n sees keys j <= lengths[z] - n + i (causal, aligned to
// the last key) or all of them; query head h reads K / V head h / (H / H_KV).  Key j of sequence z
// is row j % block of physical page page_table[z][j / block].  out = softmax(scale q k^T) v, lse =
// the natural log of the sum of exponentials; a row that sees no key gets zeros and lse = +inf,
// as in the other attention entry points.
#include "attn_paged.cuh"

#include <time.h>
#include <unistd.h>

#include <atomic>

namespace b200 {
namespace paged {

// ------------------------------------------------------------------ any head size, any layout
// One CTA per (query token, head): its warps take keys in turn, every warp keeps a running
// maximum, sum and weighted row, and the states are merged in shared memory.
constexpr int WARPS = 4;
constexpr int PER_LANE = kMaxDim / 32;

template <typename T, bool FOUR>
__global__ void __launch_bounds__(WARPS * 32) attn_paged_rows_kernel(const Params p) {
  __shared__ float row[kMaxDim];
  __shared__ float acc_all[WARPS][kMaxDim];
  __shared__ float m_all[WARPS], l_all[WARPS];
  __shared__ int found;
  const int t = (int)blockIdx.x, h = (int)blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) found = -1;
  __syncthreads();
  for (int z = threadIdx.x; z < p.Z; z += WARPS * 32) {
    int begin, end;
    query_span(p, z, begin, end);
    if (t >= begin && t < end) atomicMax(&found, z);
  }
  __syncthreads();
  const int z = found;
  if (z < 0) return;  // a token behind the last sequence: left as it is
  int begin, end;
  query_span(p, z, begin, end);
  const int n = key_count(p, z);
  const int64_t seen64 = p.causal ? (int64_t)n - (end - begin) + (t - begin) + 1 : n;
  const int seen = (int)max((int64_t)0, min((int64_t)n, seen64));
  const int kv = h / (p.H / p.HK);
  for (int i = threadIdx.x; i < p.D; i += WARPS * 32)
    row[i] = io<T>::load(((const T *)p.q)[t * p.q_t + h * p.q_h + i]) * p.scale;
  __syncthreads();

  float m = -INFINITY, l = 0.f, acc[PER_LANE];
#pragma unroll
  for (int i = 0; i < PER_LANE; ++i) acc[i] = 0.f;
  for (int j = warp; j < seen; j += WARPS) {
    const int page = p.table[z * p.table_row + j / p.block], r = j % p.block;
    if (page < 0 || page >= p.pages) {
      if (lane == 0) report_rejected(p.status, kSitePage);
      continue;  // keys of a page that does not exist are left out
    }
    const int64_t ks = page * p.kc_p + kv * p.kc_h + r * p.kc_r;
    const int64_t vs = page * p.vc_p + kv * p.vc_h + r * p.vc_r;
    float k_scale = 0.f, k_low = 0.f, v_scale = 0.f, v_low = 0.f;
    if constexpr (FOUR) {
      const T *kp = (const T *)p.k_params + page * p.kp_p + kv * p.kp_h + r * p.kp_r;
      const T *vp = (const T *)p.v_params + page * p.vp_p + kv * p.vp_h + r * p.vp_r;
      k_scale = io<T>::load(kp[0]); k_low = io<T>::load(kp[1]);
      v_scale = io<T>::load(vp[0]); v_low = io<T>::load(vp[1]);
    }
    auto value = [&](const void *base, int64_t at, int i, float scale, float low) {
      if constexpr (FOUR) {
        const uint32_t b = ((const uint8_t *)base)[at + i / 2];
        return fmaf((float)((i & 1) ? b >> 4 : b & 15u), scale, low);
      } else {
        return io<T>::load(((const T *)base)[at + i]);
      }
    };
    float dot = 0.f;
    for (int i = lane; i < p.D; i += 32) dot = fmaf(row[i], value(p.k_cache, ks, i, k_scale, k_low), dot);
    dot = warp_sum(dot);
    const float m_n = fmaxf(m, dot);
    const float keep = m == -INFINITY ? 0.f : expf(m - m_n);
    const float w = dot == -INFINITY ? 0.f : expf(dot - m_n);
    l = l * keep + w;
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) {
      const int d = lane + 32 * i;
      if (d < p.D) acc[i] = acc[i] * keep + w * value(p.v_cache, vs, d, v_scale, v_low);
    }
    m = m_n;
  }
#pragma unroll
  for (int i = 0; i < PER_LANE; ++i) acc_all[warp][lane + 32 * i] = acc[i];
  if (lane == 0) {
    m_all[warp] = m;
    l_all[warp] = l;
  }
  __syncthreads();
  float top = m_all[0];
  for (int w = 1; w < WARPS; ++w) top = fmaxf(top, m_all[w]);
  float total = 0.f, part[WARPS];
  for (int w = 0; w < WARPS; ++w) {
    part[w] = m_all[w] == -INFINITY ? 0.f : expf(m_all[w] - top);
    total += part[w] * l_all[w];
  }
  // no key seen: zeros and +inf.  (A NaN score makes the sum NaN, and stays one.)
  const bool empty = total == 0.f;
  T *o = (T *)p.out + t * p.o_t + h * p.o_h;
  for (int i = threadIdx.x; i < p.D; i += WARPS * 32) {
    float sum = 0.f;
    for (int w = 0; w < WARPS; ++w) sum += part[w] * acc_all[w][i];
    o[i] = io<T>::store(empty ? 0.f : sum / total);
  }
  if (threadIdx.x == 0 && p.lse != nullptr)
    p.lse[t * p.l_t + h * p.l_h] = empty ? INFINITY : top + logf(total);
}

template <typename T, bool FOUR> static int launch_rows(const Params &p, cudaStream_t stream) {
  attn_paged_rows_kernel<T, FOUR><<<dim3((unsigned)p.T, (unsigned)p.H), WARPS * 32, 0, stream>>>(p);
  B200_CUDA_OK(cudaGetLastError());
  return B200_OK;
}


unsigned long long next_launch() {
  // from a start that differs from process to process, so that what an earlier one left in memory is
  // no launch of this one
  static std::atomic<unsigned long long> number{[] {
    timespec now = {};
    (void)clock_gettime(CLOCK_REALTIME, &now);
    return ((unsigned long long)now.tv_sec * 1000000000ull + (unsigned long long)now.tv_nsec) * 0x9e3779b97f4a7c15ull +
           ((unsigned long long)getpid() << 20);
  }()};
  unsigned long long n;
  do n = number.fetch_add(1, std::memory_order_relaxed); while (n == 0);
  return n;
}

// What the tensor-core kernel takes: see its head.  K and V pages with the same strides (one offset
// serves both), rows of q and out on 4-byte boundaries.
static bool takes_tiles(const Params &p, bool four) {
  if (p.D != 64 && p.D != 128) return false;
  if (p.block % 16 != 0) return false;
  const int64_t es = four ? 1 : 2;
  const int64_t cache[] = {p.kc_p, p.kc_h, p.kc_r, p.vc_h};
  if (p.vc_p != p.kc_p || p.vc_r != p.kc_r || p.kc_p < 0 || p.kc_r < 0) return false;
  for (int64_t s : cache)
    if ((s * es) % 16 != 0) return false;
  if (((uintptr_t)p.k_cache | (uintptr_t)p.v_cache) % 16 != 0) return false;
  if (four) {
    const int64_t par[] = {p.kp_p, p.kp_h, p.kp_r, p.vp_h};
    if (p.vp_p != p.kp_p || p.vp_r != p.kp_r || p.kp_p < 0 || p.kp_r < 0) return false;
    for (int64_t s : par)
      if (s % 2 != 0) return false;
    if (((uintptr_t)p.k_params | (uintptr_t)p.v_params) % 4 != 0) return false;
  }
  const int64_t rows[] = {p.q_t, p.q_h, p.o_t, p.o_h};
  for (int64_t s : rows)
    if (s % 2 != 0) return false;
  return ((uintptr_t)p.q | (uintptr_t)p.out) % 4 == 0;
}

template <typename T> static int launch(const Params &p, bool four, void *workspace, cudaStream_t stream) {
  if constexpr (!std::is_same<T, float>::value) {
    if (takes_tiles(p, four)) return launch_tensor_core<T>(p, four, workspace, stream);
  }
  return four ? launch_rows<T, true>(p, stream) : launch_rows<T, false>(p, stream);
}

}  // namespace paged
}  // namespace b200

// Room for the states of rows that are cut between CTAs: two per CTA of one wave.
static size_t paged_workspace_bytes(int64_t head_dim) {
  using namespace b200::paged;
  return (size_t)kMaxCtas * 2 * (sizeof(unsigned long long) + kMaxRows * (size_t)(head_dim + 2) * sizeof(float));
}

extern "C" int b200_attn_paged_workspace(int64_t tokens, int64_t heads, int64_t kv_heads,
                                         int64_t head_dim, size_t *bytes) {
  using namespace b200;
  if (bytes == nullptr) return fail(B200_USAGE, "null out pointer");
  B200_REQUIRE(tokens >= 0 && heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0,
               "heads must be a multiple of kv_heads");
  B200_REQUIRE(head_dim >= 1 && head_dim <= paged::kMaxDim, "head size out of range 1..%d", paged::kMaxDim);
  *bytes = paged_workspace_bytes(head_dim);
  return B200_OK;
}

extern "C" int b200_attn_paged(const b200_tensor *q, const b200_tensor *k_cache,
                               const b200_tensor *v_cache, const b200_tensor *k_params,
                               const b200_tensor *v_params, const b200_tensor *page_table,
                               const b200_tensor *lengths, const b200_tensor *cu_seqlens_q,
                               b200_tensor *out, b200_tensor *lse, float scale, int causal,
                               void *workspace, size_t workspace_bytes, void *stream) {
  using namespace b200;
  int st;
  if ((st = check_tensor(q, "q", 3)) || (st = check_tensor(k_cache, "k_cache", 4)) ||
      (st = check_tensor(v_cache, "v_cache", 4)) || (st = check_tensor(page_table, "page_table", 2)) ||
      (st = check_tensor(lengths, "lengths", 1)) || (st = check_tensor(out, "out", 3)))
    return st;
  const int64_t T = q->shape[0], H = q->shape[1], D = q->shape[2], Z = page_table->shape[0];
  const int64_t pages = k_cache->shape[0], HK = k_cache->shape[1], block = k_cache->shape[2];
  const uint32_t dt = q->dtype;
  B200_REQUIRE(is_float_io(dt), "q: dtype %u is not f16/bf16/f32", dt);
  B200_REQUIRE(out->dtype == dt && out->shape[0] == T && out->shape[1] == H && out->shape[2] == D,
               "out must be [T, H, D] like q");
  B200_REQUIRE(q->stride[2] == 1 && out->stride[2] == 1, "q and out need a unit last stride");
  B200_REQUIRE(D >= 1 && D <= paged::kMaxDim, "head size %lld out of range 1..%d", (long long)D, paged::kMaxDim);
  B200_REQUIRE(HK >= 1 && H >= 1 && H % HK == 0, "%lld query heads are not a multiple of %lld K / V heads",
               (long long)H, (long long)HK);
  const bool four = k_cache->dtype == B200_DTYPE_UINT8;
  B200_REQUIRE(k_cache->dtype == v_cache->dtype && (four || k_cache->dtype == dt),
               "the caches must both be of q's dtype, or uint8 (4-bit codes)");
  B200_REQUIRE(!four || D % 2 == 0, "a 4-bit cache needs an even head size");
  for (const b200_tensor *c : {k_cache, v_cache}) {
    B200_REQUIRE(c->shape[0] == pages && c->shape[1] == HK && c->shape[2] == block &&
                     c->shape[3] == (four ? D / 2 : D),
                 "both caches must be [pages, H_KV, block, %lld]", (long long)(four ? D / 2 : D));
    B200_REQUIRE(c->stride[3] == 1, "the caches need a unit last stride");
  }
  B200_REQUIRE(block >= 1 && pages < (1ll << 31) && block < (1ll << 31), "block size or pages out of range");
  B200_REQUIRE((k_params != nullptr) == four && (v_params != nullptr) == four,
               "k_params and v_params belong to a 4-bit cache, and only to it");
  if (four) {
    if ((st = check_tensor(k_params, "k_params", 4)) || (st = check_tensor(v_params, "v_params", 4))) return st;
    for (const b200_tensor *c : {k_params, v_params}) {
      B200_REQUIRE(c->dtype == dt, "the params must have q's dtype");
      B200_REQUIRE(c->shape[0] == pages && c->shape[1] == HK && c->shape[2] == block && c->shape[3] == 2,
                   "the params must be [pages, H_KV, block, 2]");
      B200_REQUIRE(c->stride[3] == 1, "the params need a unit last stride");
    }
  }
  B200_REQUIRE(page_table->dtype == B200_DTYPE_INT32 && lengths->dtype == B200_DTYPE_INT32,
               "page_table and lengths must be int32");
  B200_REQUIRE(page_table->stride[1] == 1, "page_table needs a unit last stride");
  B200_REQUIRE(lengths->shape[0] == Z && lengths->stride[0] == 1, "lengths needs one entry per row of page_table");
  B200_REQUIRE(Z < (1 << 20) && page_table->shape[1] * block < (1ll << 30), "sequences or keys out of range");
  if (cu_seqlens_q != nullptr) {
    if ((st = check_tensor(cu_seqlens_q, "cu_seqlens_q", 1))) return st;
    B200_REQUIRE(cu_seqlens_q->dtype == B200_DTYPE_INT32 && cu_seqlens_q->shape[0] == Z + 1 &&
                     cu_seqlens_q->stride[0] == 1, "cu_seqlens_q must be int32 [Z + 1]");
  } else {
    B200_REQUIRE(Z > 0 ? T % Z == 0 : T == 0, "without cu_seqlens_q the %lld tokens must divide into %lld sequences",
                 (long long)T, (long long)Z);
  }
  if (lse != nullptr) {
    if ((st = check_tensor(lse, "lse", 2))) return st;
    B200_REQUIRE(lse->dtype == B200_DTYPE_FLOAT32 && lse->shape[0] == T && lse->shape[1] == H, "lse must be f32 [T, H]");
  }
  B200_REQUIRE(scale == scale && scale > 0.f && scale < INFINITY, "scale must be positive and finite");
  B200_REQUIRE(T < (1ll << 31) && H < 65536 && T * H < (1ll << 31), "query rows out of range");
  B200_REQUIRE(workspace != nullptr && workspace_bytes >= paged_workspace_bytes(D) && (uintptr_t)workspace % 16 == 0,
               "the workspace must be 16-byte aligned and hold %zu bytes (b200_attn_paged_workspace)",
               paged_workspace_bytes(D));
  if (T == 0 || Z == 0) return B200_OK;

  const b200_tensor *all[] = {q, k_cache, v_cache, k_params, v_params, page_table, lengths, cu_seqlens_q, out, lse};
  static const char *const names[] = {"q", "k_cache", "v_cache", "k_params", "v_params", "page_table", "lengths",
                                      "cu_seqlens_q", "out", "lse"};
  for (int i = 0; i < 10; ++i)
    if (all[i] != nullptr && (st = check_reachable(all[i]->data, names[i], i >= 1 && i <= 4))) return st;
  if ((st = check_reachable(workspace, "workspace", true))) return st;

  paged::Params p = {};
  p.q = q->data; p.k_cache = k_cache->data; p.v_cache = v_cache->data; p.out = out->data;
  p.q_t = q->stride[0]; p.q_h = q->stride[1]; p.o_t = out->stride[0]; p.o_h = out->stride[1];
  p.kc_p = k_cache->stride[0]; p.kc_h = k_cache->stride[1]; p.kc_r = k_cache->stride[2];
  p.vc_p = v_cache->stride[0]; p.vc_h = v_cache->stride[1]; p.vc_r = v_cache->stride[2];
  if (four) {
    p.k_params = k_params->data; p.v_params = v_params->data;
    p.kp_p = k_params->stride[0]; p.kp_h = k_params->stride[1]; p.kp_r = k_params->stride[2];
    p.vp_p = v_params->stride[0]; p.vp_h = v_params->stride[1]; p.vp_r = v_params->stride[2];
  }
  if (lse != nullptr) { p.lse = (float *)lse->data; p.l_t = lse->stride[0]; p.l_h = lse->stride[1]; }
  p.table = (const int *)page_table->data; p.lengths = (const int *)lengths->data;
  p.cu = cu_seqlens_q != nullptr ? (const int *)cu_seqlens_q->data : nullptr;
  p.table_row = page_table->stride[0];
  p.T = (int)T; p.Z = (int)Z; p.H = (int)H; p.HK = (int)HK; p.D = (int)D;
  p.pages = (int)pages; p.width = (int)page_table->shape[1]; p.block = (int)block;
  p.causal = causal != 0;
  p.scale = scale;
  p.status = device_status_word();
  if (p.status == nullptr) return fail(B200_RESOURCE, "no status word on this device");
  cudaStream_t s = (cudaStream_t)stream;
  if (dt == B200_DTYPE_FLOAT32) return paged::launch<float>(p, four, workspace, s);
  if (dt == B200_DTYPE_FLOAT16) return paged::launch<__half>(p, four, workspace, s);
  return paged::launch<__nv_bfloat16>(p, four, workspace, s);
}
