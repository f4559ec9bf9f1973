// A linear layer in 8-bit integers: y[m,n] = act(x_scale[m] w_scale[n] sum_k x[m,k] w[n,k] + bias[n])
// with one scale per token and one per output channel, and the operator that makes x: rows divided
// by their largest magnitude / 127 and rounded to the nearest whole number, ties to even.
//
// The sums are exact (32-bit integers, K <= 131071 keeps |sum| below 2^31); scales, bias and the
// activation are 32-bit floats, rounded once at the store.
//
// Measured with the quantiser: 8 tokens x 14336 x 4096 13.2 us (59 MB of weights, 4.5 TB/s; the copy rate
// would give 9.0), 4097 x 11008 x 4096 159 us (2.33 Pop/s), 8192 x 8192 x 8192 355 us (3.10 Pop/s).  Few
// tokens are bound by the ring's fill and the set-up of a launch that streams its weights once, the
// large ones by the tensor pipe under the power cap and by the last wave's and last rows' rounding up.
#include "sm100.cuh"

namespace b200 {
namespace int8 {

constexpr int64_t kMaxK = 131071;  // 128 * 128 * K < 2^31

// ------------------------------------------------------------------------- rows to 8 bits
// One CTA per row.  The magnitudes are compared as integers, which order like the floats and put
// a NaN above infinity: a row that holds either gets a scale that is not finite and zero codes.
struct QuantParams {
  const void *x;
  int8_t *out;
  float *scale;
  int64_t x_row, o_row;
  int M, K;
};

__device__ __forceinline__ int round_code(float x, float scale, float inv) {
  const float y = x * inv;  // |y| <= 127: within 3e-5 of the quotient while 1 / scale is normal
  float r = rintf(y);
  if (!(fabsf(fabsf(y - r) - 0.5f) > 1e-4f) || scale < 1e-30f)
    r = (float)rint((double)x / (double)scale);
  return (int)fminf(fmaxf(r, -127.f), 127.f);
}

constexpr int QTHREADS = 256;

template <typename T>
__global__ void __launch_bounds__(QTHREADS) quantize_rows_kernel(const QuantParams p) {
  __shared__ unsigned int tops[QTHREADS / 32];
  const int64_t m = blockIdx.x;
  const T *x = (const T *)p.x + m * p.x_row;
  unsigned int top = 0;
  for (int i = threadIdx.x; i < p.K; i += QTHREADS)
    top = max(top, __float_as_uint(io<T>::load(x[i])) & 0x7fffffffu);
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
  for (int w = 0; w < QTHREADS / 32; ++w) top = max(top, tops[w]);
  const float scale = __fdiv_rn(__uint_as_float(top), 127.f);
  const bool usable = scale > 0.f && scale < INFINITY;
  const float inv = 1.f / scale;
  int8_t *out = p.out + m * p.o_row;
  for (int i = threadIdx.x; i < p.K; i += QTHREADS)
    out[i] = usable ? (int8_t)round_code(io<T>::load(x[i]), scale, inv) : (int8_t)0;
  if (threadIdx.x == 0) p.scale[m] = scale;
}

// Rows of whole 16-byte vectors that fit in the registers of one CTA (four vectors per thread, up to 1024
// threads): read once, reduced, divided and stored.  Bound by HBM (three bytes per 16-bit element);
// the codes come from adding 1.5 * 2^23, whose sum's low byte is the nearest whole number, and only
// vectors with an element next to a border are decided by 64-bit quotients.
constexpr int kVectors = 4;

template <typename T>
__global__ void __launch_bounds__(1024) quantize_rows_vector_kernel(const QuantParams p) {
  constexpr int N = vec16<T>::N;
  __shared__ unsigned int tops[32];
  // a product launched behind this kernel may set itself up meanwhile; it waits for the end before it
  // reads anything
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t m = blockIdx.x;
  const int vectors = p.K / N;
  const T *x = (const T *)p.x + m * p.x_row;
  vec16<T> v[kVectors];
  unsigned int top = 0;
#pragma unroll
  for (int j = 0; j < kVectors; ++j) {
    const int i = threadIdx.x + j * blockDim.x;
    v[j].raw = i < vectors ? ld_stream16(x + (int64_t)i * N) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int j = 0; j < kVectors; ++j)
#pragma unroll
    for (int e = 0; e < N; ++e) top = max(top, __float_as_uint(io<T>::load(v[j].e[e])) & 0x7fffffffu);
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
  top = __reduce_max_sync(0xffffffffu, threadIdx.x % 32 < blockDim.x / 32 ? tops[threadIdx.x % 32] : 0u);
  const float scale = __fdiv_rn(__uint_as_float(top), 127.f);
  const bool usable = scale > 0.f && scale < INFINITY;
  const float inv = 1.f / scale;
  if (threadIdx.x == 0) p.scale[m] = scale;
  int8_t *out = p.out + m * p.o_row;
#pragma unroll
  for (int j = 0; j < kVectors; ++j) {
    const int i = threadIdx.x + j * blockDim.x;
    if (i >= vectors) break;
    constexpr float kMove = 12582912.f;
    uint32_t word[N / 4];
    float far = 0.f;
#pragma unroll
    for (int w = 0; w < N / 4; ++w) {
      uint32_t b[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float y = io<T>::load(v[j].e[4 * w + e]) * inv;
        const float moved = y + kMove;
        far = fmaxf(far, fabsf(y - (moved - kMove)));
        b[e] = __float_as_uint(moved);
      }
      word[w] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    }
    if (!(far < 0.4999f) || !(scale >= 1e-30f) || !usable) {
#pragma unroll
      for (int w = 0; w < N / 4; ++w) {
        word[w] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (usable)
            word[w] |= ((uint32_t)round_code(io<T>::load(v[j].e[4 * w + e]), scale, inv) & 255u) << (8 * e);
      }
    }
    if constexpr (N == 8) *reinterpret_cast<uint2 *>(out + (int64_t)i * N) = make_uint2(word[0], word[1]);
    else *reinterpret_cast<uint32_t *>(out + (int64_t)i * N) = word[0];
  }
}

template <typename T> static int launch_quantize(const QuantParams &p, cudaStream_t stream) {
  constexpr int N = vec16<T>::N;
  const int threads = (p.K / N + kVectors * 32 - 1) / (kVectors * 32) * 32;
  if (p.K % N == 0 && p.K > 0 && threads <= 1024 && (uintptr_t)p.x % 16 == 0 && p.x_row % N == 0 &&
      (uintptr_t)p.out % N == 0 && p.o_row % N == 0)
    quantize_rows_vector_kernel<T><<<(unsigned)p.M, threads, 0, stream>>>(p);
  else
    quantize_rows_kernel<T><<<(unsigned)p.M, QTHREADS, 0, stream>>>(p);
  B200_CUDA_OK(cudaGetLastError());
  return B200_OK;
}

// ------------------------------------------------------------------------- the product
struct Params {
  const int8_t *x, *w;
  const float *x_scale, *w_scale;
  const void *bias;
  void *y;
  int64_t x_row, w_row, y_row;
  int M, N, K;
  int act, bias_kind;
};

__device__ __forceinline__ float load_bias(const void *bias, int kind, int col) {
  if (kind == 0) return 0.f;
  if (kind == B200_DTYPE_FLOAT32) return ((const float *)bias)[col];
  if (kind == B200_DTYPE_BFLOAT16) return __bfloat162float(((const __nv_bfloat16 *)bias)[col]);
  return __half2float(((const __half *)bias)[col]);
}

// gelu_tanh(z) = z (1 + tanh u) / 2 = z / (1 + exp(-2 u)): the quotient keeps its relative precision
// where 1 + tanh u cancels.  16-bit results take the approximate exponential and division (2^-21).
template <typename T, int ACT> __device__ __forceinline__ float activate(float z) {
  if constexpr (ACT == B200_ACT_GELU_ERF) return z * normcdff(z);  // z (1 + erf(z / sqrt 2)) / 2
  if constexpr (ACT == B200_ACT_GELU_TANH) {
    const float u = -1.5957691216057308f * (z + 0.044715f * z * z * z);
    return sizeof(T) == 2 ? __fdividef(z, 1.0f + __expf(u)) : z / (1.0f + expf(u));
  }
  if constexpr (ACT == B200_ACT_LEAKY_RELU) return z >= 0.f ? z : 0.01f * z;
  return z;
}
template <typename T> __device__ __forceinline__ float activate(float z, int act) {
  switch (act) {
    case B200_ACT_GELU_ERF: return activate<T, B200_ACT_GELU_ERF>(z);
    case B200_ACT_GELU_TANH: return activate<T, B200_ACT_GELU_TANH>(z);
    case B200_ACT_LEAKY_RELU: return activate<T, B200_ACT_LEAKY_RELU>(z);
    default: return z;
  }
}

// Any sizes and alignment: 32 x 32 outputs per CTA, operands staged in shared memory.
constexpr int TILE = 32;

template <typename T>
__global__ void __launch_bounds__(256) linear_int8_tile_kernel(const Params p) {
  __shared__ int8_t xs[TILE][TILE + 4], ws[TILE][TILE + 4];
  const int m0 = (int)blockIdx.y * TILE, n0 = (int)blockIdx.x * TILE;
  const int col = threadIdx.x & 31, group = threadIdx.x >> 5;  // 8 groups of 4 rows
  int acc[4] = {0, 0, 0, 0};
  for (int k0 = 0; k0 < p.K; k0 += TILE) {
    for (int i = group; i < TILE; i += 8) {
      const int k = k0 + col;
      xs[i][col] = (m0 + i < p.M && k < p.K) ? p.x[(int64_t)(m0 + i) * p.x_row + k] : (int8_t)0;
      ws[i][col] = (n0 + i < p.N && k < p.K) ? p.w[(int64_t)(n0 + i) * p.w_row + k] : (int8_t)0;
    }
    __syncthreads();
#pragma unroll 8
    for (int k = 0; k < TILE; ++k) {
      const int b = ws[col][k];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] += b * (int)xs[group * 4 + i][k];
    }
    __syncthreads();
  }
  const int n = n0 + col;
  if (n >= p.N) return;
  const float sw = p.w_scale[n], b = load_bias(p.bias, p.bias_kind, n);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = m0 + group * 4 + i;
    if (m < p.M)
      ((T *)p.y)[(int64_t)m * p.y_row + n] =
          io<T>::store(activate<T>(fmaf((float)acc[i], p.x_scale[m] * sw, b), p.act));
  }
}

// ------------------------------------------------------------------------- tensor cores
// Both operands are rows of K bytes, so a k-block is one 128-byte swizzle span (128 values) and
// the shared-memory tiles, descriptors and pipeline are those of the 16-bit products
// (gemm_sm100.cu); an MMA takes 32 values of K in the time kind::f16 takes 16.
using namespace sm100;

constexpr int BK = 128;                  // bytes of K per k-block
constexpr int MMA_K = 32;
constexpr int A_BYTES = 128 * BK;        // 128 rows: 16 KiB
constexpr int THREADS = 192;             // warps 0-3 epilogue, 4 producer, 5 MMA issuer
constexpr uint32_t kHi = desc_hi_sw128(1024);

__device__ __forceinline__ bool wait_all(uint32_t bar, uint32_t parity, const WaitCtx &ctx, uint32_t site) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, ctx, site)) != 0;
}

// Many tokens: a cluster of two CTAs per 256 x 256 tile of y, cta_group::2 MMAs (256 x 256 x 32);
// each CTA loads its 128 rows of x and its 128 of the tile's rows of w and finishes the 256
// columns of its own 128 rows while the next tile's MMAs run (two 256-column accumulators).
constexpr int PAIR_STAGES = 6;
constexpr int PAIR_STAGE_BYTES = 2 * A_BYTES;
constexpr int PAIR_SMEM_BYTES = PAIR_STAGES * PAIR_STAGE_BYTES + 1024 + 256;

struct TcParams {
  Params p;
  int group_m;     // pair kernel: row pairs per raster group
  int vector_store;
  int vector_cols; // w_scale and bias are 16-byte aligned
  unsigned int *status;
};

__device__ __forceinline__ void load_floats32(const float *src, int col0, int n, bool vec, float (&v)[32]) {
  if (vec && col0 + 32 <= n) {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const float4 t = __ldg(reinterpret_cast<const float4 *>(src + col0) + q);
      v[4 * q] = t.x; v[4 * q + 1] = t.y; v[4 * q + 2] = t.z; v[4 * q + 3] = t.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = col0 + j < n ? __ldg(src + col0 + j) : 0.f;
  }
}
__device__ __forceinline__ void load_bias32(const Params &p, int col0, bool vec, float (&b)[32]) {
  if (p.bias_kind == 0) {
#pragma unroll
    for (int j = 0; j < 32; ++j) b[j] = 0.f;
  } else if (p.bias_kind == B200_DTYPE_FLOAT32) {
    load_floats32((const float *)p.bias, col0, p.N, vec, b);
  } else if (vec && col0 + 32 <= p.N) {
    const bool bf = p.bias_kind == B200_DTYPE_BFLOAT16;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint4 t = __ldg(reinterpret_cast<const uint4 *>((const uint16_t *)p.bias + col0) + q);
      const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 h = bf ? make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u))
                            : __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        b[8 * q + 2 * i] = h.x;
        b[8 * q + 2 * i + 1] = h.y;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j) b[j] = col0 + j < p.N ? load_bias(p.bias, p.bias_kind, col0 + j) : 0.f;
  }
}

// 32 accumulator columns of one row: scale, bias, activation, one rounding, store
template <typename T, int ACT>
__device__ __forceinline__ void finish32(const uint32_t (&r)[32], const TcParams &t, T *row, int col0,
                                         bool row_ok, float sx) {
  const Params &p = t.p;
  if (col0 >= p.N) return;  // warp-uniform
  float s[32], b[32];
  load_floats32(p.w_scale, col0, p.N, t.vector_cols != 0, s);
  load_bias32(p, col0, t.vector_cols != 0, b);
#pragma unroll
  for (int j = 0; j < 32; ++j) s[j] = activate<T, ACT>(fmaf((float)(int)r[j], sx * s[j], b[j]));
  if (!row_ok) return;
  if (t.vector_store && col0 + 32 <= p.N) {
    constexpr int PER = 16 / (int)sizeof(T);
#pragma unroll
    for (int q = 0; q < 32 / PER; ++q) {
      vec16<T> o;
#pragma unroll
      for (int j = 0; j < PER; ++j) o.e[j] = io<T>::store(s[q * PER + j]);
      *reinterpret_cast<uint4 *>(row + col0 + q * PER) = o.raw;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (col0 + j < p.N) row[col0 + j] = io<T>::store(s[j]);
  }
}

template <typename T, int ACT>
__device__ __forceinline__ void finish_tile(uint32_t t_row, const TcParams &t, T *row, int col_base,
                                            bool row_ok, float sx) {
  uint32_t ra[32], rb[32];
  tmem_ld_32x32b_x32(t_row, ra);
#pragma unroll 1
  for (int c = 0; c < 8; c += 2) {
    tmem_ld_wait();
    tmem_ld_32x32b_x32(t_row + (uint32_t)(c + 1) * 32u, rb);
    finish32<T, ACT>(ra, t, row, col_base + c * 32, row_ok, sx);
    tmem_ld_wait();
    if (c + 2 < 8) tmem_ld_32x32b_x32(t_row + (uint32_t)(c + 2) * 32u, ra);
    finish32<T, ACT>(rb, t, row, col_base + (c + 1) * 32, row_ok, sx);
  }
}

// raster order: groups of group_m row pairs, column blocks inside a group, so the CTAs that run
// at one time share rows of x and of w in L2
__device__ __forceinline__ void tile_coords(int tile, int m_pairs, int n_blocks, int group_m, int &mp, int &nb) {
  const int per_group = group_m * n_blocks;
  const int group = tile / per_group, first = group * group_m;
  const int rows = min(group_m, m_pairs - first);
  const int in_group = tile - group * per_group;
  mp = first + in_group % rows;
  nb = in_group / rows;
}

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
linear_int8_pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                        const TcParams t) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t *smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t x_smem = smem_base, w_smem = smem_base + PAIR_STAGES * A_BYTES;
  const uint32_t bar0 = smem_base + PAIR_STAGES * PAIR_STAGE_BYTES;
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (PAIR_STAGES + s); };
  auto acc_full_bar = [&](int a) { return bar0 + 8u * (2 * PAIR_STAGES + a); };
  auto acc_empty_bar = [&](int a) { return bar0 + 8u * (2 * PAIR_STAGES + 2 + a); };
  const uint32_t drain_bar = bar0 + 8u * (2 * PAIR_STAGES + 4);
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem_gen + PAIR_STAGES * PAIR_STAGE_BYTES +
                                                     8 * (2 * PAIR_STAGES + 5));
  volatile uint32_t *abort_flag = tmem_slot + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_cta_rank();
  const WaitCtx ctx{abort_flag, t.status};
  const Params &p = t.p;
  const int m_pairs = (p.M + 255) / 256, n_blocks = (p.N + 255) / 256;
  const int num_tiles = m_pairs * n_blocks, num_kb = (p.K + BK - 1) / BK;
  const int first = (int)(blockIdx.x >> 1), step = (int)(gridDim.x >> 1);

  if (threadIdx.x == 0) {
    for (int s = 0; s < PAIR_STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(acc_full_bar(a), 1);
      mbar_init(acc_empty_bar(a), 8);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0u;
    mbar_init_fence();
  }
  if (warp == 4 && lane == 0) {
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_w);
  }
  if (warp == 5) tmem_alloc_pair(smem_u32(tmem_slot), 512);
  tc_fence_before_sync();
  __syncthreads();
  cluster_arrive();  // the peer's barriers exist before anything of this CTA reaches them
  cluster_wait();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 4) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, issued = 0, parity = 0;
      bool ok = true;
      for (int tile = first; ok && tile < num_tiles; tile += step) {
        int mp, nb;
        tile_coords(tile, m_pairs, n_blocks, t.group_m, mp, nb);
        const int row0 = (mp * 2 + (int)rank) * 128, col0 = nb * 256 + (int)rank * 128;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1u, ctx, 54)) { ok = false; break; }
          if (rank == 0) mbar_arrive_expect_tx(full_bar(stage), 2 * PAIR_STAGE_BYTES);
          const uint32_t full0 = map_to_cta(full_bar(stage), 0);
          tma_load_2d_pair(x_smem + stage * A_BYTES, &tm_x, full0, kb * BK, row0);
          tma_load_2d_pair(w_smem + stage * A_BYTES, &tm_w, full0, kb * BK, col0);
          issued |= 1u << stage;
          parity = (parity & ~(1u << stage)) | (phase << stage);
          if (++stage == PAIR_STAGES) { stage = 0; phase ^= 1u; }
        }
      }
      if (!ok && rank == 0)  // copies in flight still target shared memory of the pair
        for (int s = 0; s < PAIR_STAGES; ++s)
          if (issued & (1u << s)) mbar_wait_drain(full_bar(s), (parity >> s) & 1u);
    }
  } else if (warp == 5) {
    if (rank == 0) {
      const bool leader = elect_one();
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      const uint32_t x_lo0 = desc_lo_sw128(x_smem, 16), w_lo0 = desc_lo_sw128(w_smem, 16);
      const uint32_t peer_bar0 = map_to_cta(bar0, 1);
      constexpr uint32_t idesc = make_idesc_s8(256, 256);
      for (int tile = first; ok && tile < num_tiles; tile += step) {
        if (!wait_all(acc_empty_bar(acc), acc_phase ^ 1u, ctx, 55)) { ok = false; break; }
        tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + (uint32_t)(acc * 256);
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!wait_all(full_bar(stage), phase, ctx, 56)) { ok = false; break; }
          tc_fence_after_sync();
          const uint32_t x_lo = x_lo0 + (uint32_t)stage * (A_BYTES >> 4);
          const uint32_t w_lo = w_lo0 + (uint32_t)stage * (A_BYTES >> 4);
          if (leader) {
#pragma unroll
            for (int k = 0; k < BK / MMA_K; ++k)
              mma_i8_ss_pair(d_tmem, x_lo + (uint32_t)(k * (MMA_K >> 4)), kHi,
                             w_lo + (uint32_t)(k * (MMA_K >> 4)), kHi, idesc, (kb > 0 || k > 0) ? 1u : 0u);
            tc_commit_pair(empty_bar(stage));
            tc_commit_pair(peer_bar0 + (empty_bar(stage) - bar0));
          }
          if (++stage == PAIR_STAGES) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        if (leader) {
          tc_commit_pair(acc_full_bar(acc));
          tc_commit_pair(peer_bar0 + (acc_full_bar(acc) - bar0));
        }
        if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
      }
      if (leader) {
        tc_commit_pair(drain_bar);
        mbar_wait_drain(drain_bar, 0);
      }
      __syncwarp();
    }
  } else {
    int acc = 0;
    uint32_t acc_phase = 0;
    const uint32_t acc_empty0 = map_to_cta(acc_empty_bar(0), 0);
    for (int tile = first; tile < num_tiles; tile += step) {
      int mp, nb;
      tile_coords(tile, m_pairs, n_blocks, t.group_m, mp, nb);
      if (!wait_all(acc_full_bar(acc), acc_phase, ctx, 57)) break;
      tc_fence_after_sync();
      const int row = (mp * 2 + (int)rank) * 128 + warp * 32 + lane;
      const bool row_ok = row < p.M;
      const float sx = row_ok ? p.x_scale[row] : 0.f;
      const uint32_t t_row = tmem_base + ((uint32_t)(warp * 32) << 16) + (uint32_t)(acc * 256);
      T *y = (T *)p.y + (int64_t)row * p.y_row;
      switch (p.act) {
        case B200_ACT_GELU_ERF: finish_tile<T, B200_ACT_GELU_ERF>(t_row, t, y, nb * 256, row_ok, sx); break;
        case B200_ACT_GELU_TANH: finish_tile<T, B200_ACT_GELU_TANH>(t_row, t, y, nb * 256, row_ok, sx); break;
        case B200_ACT_LEAKY_RELU: finish_tile<T, B200_ACT_LEAKY_RELU>(t_row, t, y, nb * 256, row_ok, sx); break;
        default: finish_tile<T, B200_ACT_NONE>(t_row, t, y, nb * 256, row_ok, sx);
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(acc_empty0 + 8u * (uint32_t)acc);
      if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
    }
  }
  // neither CTA leaves while the pair's MMAs can touch its memory: the even CTA has drained them
  tc_fence_before_sync();
  __syncthreads();
  cluster_arrive();
  cluster_wait();
  if (warp == 5) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// Fewer tokens than fill the pairs: the roles are swapped -- 128 rows of w are the MMA's rows and
// TN tokens its columns -- so a decode step multiplies a few columns instead of 128 rows of
// padding, and K is cut between the CTAs of a cluster when the row blocks alone do not fill the
// SMs.  The CTAs of a cluster then exchange their integer sums through distributed shared memory
// (exact, so their order does not matter), every CTA finishing every S-th token.
template <int TN> constexpr int skinny_stage_bytes() { return A_BYTES + TN * BK; }
template <int TN> constexpr int skinny_stages() { return TN == 32 ? 5 : (TN == 64 ? 4 : (TN == 128 ? 6 : 4)); }
template <int TN> constexpr int skinny_smem() { return skinny_stages<TN>() * skinny_stage_bytes<TN>() + 1024 + 256; }
template <int TN> constexpr int skinny_ctas_per_sm() { return TN <= 64 ? 2 : 1; }

__device__ __forceinline__ int ld_cluster_s32(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// The end of the swapped kernel: warps 0-3 have row n0 + 32 warp + lane of w each, the tokens are the
// accumulator's columns; a token's 32 outputs of a warp are consecutive in y.  All warps come here.
template <typename T, int ACT>
__device__ __forceinline__ void skinny_epilogue(const Params &p, uint32_t smem_base, uint8_t *smem_gen, uint32_t tmem_base,
                                                int n0, int m0, int tokens, int rank, int slices, bool summed) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = n0 + (warp & 3) * 32 + lane;
  const bool n_ok = warp < 4 && n < p.N;
  const float sw = n_ok ? p.w_scale[n] : 0.f, b = n_ok ? load_bias(p.bias, p.bias_kind, n) : 0.f;
  T *y = (T *)p.y + (int64_t)m0 * p.y_row + n;
  const uint32_t t_row = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
  if (slices == 1) {
    if (!summed) return;
#pragma unroll 1
    for (int c0 = 0; c0 < tokens; c0 += 32) {
      uint32_t r[32];
      tmem_ld_32x32b_x32(t_row + (uint32_t)c0, r);
      const float mine = c0 + lane < tokens ? __ldg(p.x_scale + m0 + c0 + lane) : 0.f;
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        const float sx = __shfl_sync(0xffffffffu, mine, j);
        const float v = activate<T, ACT>(fmaf((float)(int)r[j], sx * sw, b));
        if (n_ok && c0 + j < tokens) *y = io<T>::store(v);
        y += p.y_row;
      }
    }
    return;
  }
  // the ring is empty (every load was consumed before the accumulator was complete): it takes the
  // sums as [token][128 rows]
  int *sums = reinterpret_cast<int *>(smem_gen);
  if (summed) {
#pragma unroll 1
    for (int c0 = 0; c0 < tokens; c0 += 32) {
      uint32_t r[32];
      tmem_ld_32x32b_x32(t_row + (uint32_t)c0, r);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 32; ++j) sums[(c0 + j) * 128 + warp * 32 + lane] = (int)r[j];
    }
  }
  __syncwarp();
  cluster_arrive();
  cluster_wait();
  if (n_ok && summed) {
    constexpr int kAt = 8;  // tokens in flight
    const uint32_t mine = smem_base + (uint32_t)(warp * 32 + lane) * 4u;
    for (int c0 = rank; c0 < tokens; c0 += kAt * slices) {
      int total[kAt];
#pragma unroll
      for (int j = 0; j < kAt; ++j) total[j] = 0;
      for (int s = 0; s < slices; ++s) {
        const uint32_t from = map_to_cta(mine, (uint32_t)s);
#pragma unroll
        for (int j = 0; j < kAt; ++j)
          if (c0 + j * slices < tokens) total[j] += ld_cluster_s32(from + (uint32_t)(c0 + j * slices) * 512u);
      }
#pragma unroll
      for (int j = 0; j < kAt; ++j) {
        const int c = c0 + j * slices;
        if (c < tokens)
          y[(int64_t)c * p.y_row] =
              io<T>::store(activate<T, ACT>(fmaf((float)total[j], __ldg(p.x_scale + m0 + c) * sw, b)));
      }
    }
  }
  __syncwarp();
  cluster_arrive();  // the peers read this CTA's sums until they arrive
  cluster_wait();
}

template <typename T, int TN>
__global__ void __launch_bounds__(THREADS, skinny_ctas_per_sm<TN>())
linear_int8_skinny_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                          const TcParams t, int slices) {
  constexpr int STAGES = skinny_stages<TN>(), X_BYTES = TN * BK, STAGE_BYTES = skinny_stage_bytes<TN>();
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t *smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t w_smem = smem_base, x_smem = smem_base + STAGES * A_BYTES;
  const uint32_t bar0 = smem_base + STAGES * STAGE_BYTES;
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (STAGES + s); };
  const uint32_t acc_bar = bar0 + 8u * (2 * STAGES), drain_bar = acc_bar + 8u;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem_gen + STAGES * STAGE_BYTES + 8 * (2 * STAGES + 2));
  volatile uint32_t *abort_flag = tmem_slot + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const WaitCtx ctx{abort_flag, t.status};
  const Params &p = t.p;
  const int rank = (int)blockIdx.x % slices, tile = (int)blockIdx.x / slices;
  const int n_blocks = (p.N + 127) / 128, num_kb = (p.K + BK - 1) / BK;
  const int n0 = (tile % n_blocks) * 128, m0 = (tile / n_blocks) * TN;
  const int kb0 = num_kb * rank / slices, kb1 = num_kb * (rank + 1) / slices;
  const int tokens = min(TN, p.M - m0);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(acc_bar, 1);
    mbar_init(drain_bar, 1);
    *abort_flag = 0u;
    mbar_init_fence();
  }
  if (warp == 4 && lane == 0) {
    tma_prefetch_desc(&tm_w);
    tma_prefetch_desc(&tm_x);
  }
  if (warp == 5) tmem_alloc(smem_u32(tmem_slot), TN);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  bool summed = false;
  // The set-up above overlaps the end of the kernel before this one in the stream (the row quantiser);
  // nothing that a kernel wrote is read, and nothing written, before all of it is done.
  asm volatile("griddepcontrol.wait;" ::: "memory");

  if (warp == 4) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, issued = 0, parity = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(empty_bar(stage), phase ^ 1u, ctx, 54)) { ok = false; break; }
        mbar_arrive_expect_tx(full_bar(stage), STAGE_BYTES);
        tma_load_2d(w_smem + stage * A_BYTES, &tm_w, full_bar(stage), kb * BK, n0);
        tma_load_2d(x_smem + stage * X_BYTES, &tm_x, full_bar(stage), kb * BK, m0);
        issued |= 1u << stage;
        parity = (parity & ~(1u << stage)) | (phase << stage);
        if (++stage == STAGES) { stage = 0; phase ^= 1u; }
      }
      if (!ok)
        for (int s = 0; s < STAGES; ++s)
          if (issued & (1u << s)) mbar_wait_drain(full_bar(s), (parity >> s) & 1u);
    }
  } else if (warp == 5) {
    const bool leader = elect_one();
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint32_t w_lo0 = desc_lo_sw128(w_smem, 16), x_lo0 = desc_lo_sw128(x_smem, 16);
    constexpr uint32_t idesc = make_idesc_s8(128, TN);
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!wait_all(full_bar(stage), phase, ctx, 56)) { ok = false; break; }
      tc_fence_after_sync();
      const uint32_t w_lo = w_lo0 + (uint32_t)stage * (A_BYTES >> 4);
      const uint32_t x_lo = x_lo0 + (uint32_t)stage * (X_BYTES >> 4);
      if (leader) {
#pragma unroll
        for (int k = 0; k < BK / MMA_K; ++k)
          mma_i8_ss(tmem_base, w_lo + (uint32_t)(k * (MMA_K >> 4)), kHi, x_lo + (uint32_t)(k * (MMA_K >> 4)), kHi,
                    idesc, (kb > kb0 || k > 0) ? 1u : 0u);
        tc_commit(empty_bar(stage));
      }
      if (++stage == STAGES) { stage = 0; phase ^= 1u; }
    }
    if (leader) {
      if (ok) tc_commit(acc_bar);
      tc_commit(drain_bar);
      mbar_wait_drain(drain_bar, 0);
    }
    __syncwarp();
  } else {
    summed = wait_all(acc_bar, 0, ctx, 57);
    tc_fence_after_sync();
  }

  switch (p.act) {
    case B200_ACT_GELU_ERF: skinny_epilogue<T, B200_ACT_GELU_ERF>(p, smem_base, smem_gen, tmem_base, n0, m0, tokens, rank, slices, summed); break;
    case B200_ACT_GELU_TANH: skinny_epilogue<T, B200_ACT_GELU_TANH>(p, smem_base, smem_gen, tmem_base, n0, m0, tokens, rank, slices, summed); break;
    case B200_ACT_LEAKY_RELU: skinny_epilogue<T, B200_ACT_LEAKY_RELU>(p, smem_base, smem_gen, tmem_base, n0, m0, tokens, rank, slices, summed); break;
    default: skinny_epilogue<T, B200_ACT_NONE>(p, smem_base, smem_gen, tmem_base, n0, m0, tokens, rank, slices, summed);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, TN);
  }
}

template <typename T, int TN>
static int launch_skinny(const CUtensorMap &tm_w, const CUtensorMap &tm_x, const TcParams &t, cudaStream_t stream) {
  auto kernel = linear_int8_skinny_kernel<T, TN>;
  static bool configured[64] = {false};
  int dev = 0;
  B200_CUDA_OK(cudaGetDevice(&dev));
  if (dev >= 64) return fail(B200_RESOURCE, "device index %d out of range", dev);
  if (!configured[dev]) {
    B200_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, skinny_smem<TN>()));
    configured[dev] = true;
  }
  const int64_t tiles = (int64_t)((t.p.N + 127) / 128) * ((t.p.M + TN - 1) / TN);
  if (tiles >= (1ll << 28)) return fail(B200_REJECTED, "%lld tiles out of range", (long long)tiles);
  // Cut K while the CTAs fit beside one another and a slice keeps four k-blocks, four times at most and
  // not for 128 tokens or more: what the slices exchange grows with the tokens (4096 x 4096 weights:
  // 8 tokens in 4 / 8 slices 9.2 / 9.6 us, 64 tokens in 2 / 4 / 8 17.3 / 15.4 / 16.8, 128 tokens in
  // 1 / 2 / 4 17.2 / 22.1 / 18.8).
  const int num_kb = (t.p.K + BK - 1) / BK;
  int slices = 1;
  while (slices < (TN >= 128 ? 1 : 4) && tiles * slices * 2 <= (int64_t)sm_count() * skinny_ctas_per_sm<TN>() && num_kb / (slices * 2) >= 4)
    slices *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * slices));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = skinny_smem<TN>();
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)slices;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = slices > 1 ? 2 : 1;
  B200_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, tm_w, tm_x, t, slices));
  return B200_OK;
}

template <typename T>
static int launch_pair(const CUtensorMap &tm_x, const CUtensorMap &tm_w, const TcParams &t, cudaStream_t stream) {
  auto kernel = linear_int8_pair_kernel<T>;
  static int max_clusters[64] = {0};
  int dev = 0;
  B200_CUDA_OK(cudaGetDevice(&dev));
  if (dev >= 64) return fail(B200_RESOURCE, "device index %d out of range", dev);
  if (max_clusters[dev] == 0) {
    B200_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PAIR_SMEM_BYTES));
    cudaLaunchConfig_t probe = {};
    probe.gridDim = dim3((unsigned)sm_count());
    probe.blockDim = dim3(THREADS);
    probe.dynamicSmemBytes = PAIR_SMEM_BYTES;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    probe.attrs = &attr;
    probe.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &probe) != cudaSuccess) {
      (void)cudaGetLastError();
      n = 0;
    }
    max_clusters[dev] = n > 0 ? n : sm_count() / 2;
  }
  const int64_t tiles = (int64_t)((t.p.M + 255) / 256) * ((t.p.N + 255) / 256);
  if (tiles >= (1ll << 30)) return fail(B200_REJECTED, "%lld tiles out of range", (long long)tiles);
  const int clusters = (int)(tiles < max_clusters[dev] ? tiles : max_clusters[dev]);
  kernel<<<2 * clusters, THREADS, PAIR_SMEM_BYTES, stream>>>(tm_x, tm_w, t);
  B200_CUDA_OK(cudaGetLastError());
  return B200_OK;
}

static int byte_map(CUtensorMap *map, const int8_t *base, int rows, int cols, int64_t pitch, int box_rows) {
  const uint64_t dims[2] = {(uint64_t)cols, (uint64_t)rows};
  const uint64_t strides[2] = {1, (uint64_t)pitch};
  const uint32_t box[2] = {BK, (uint32_t)box_rows};
  return encode_tensor_map(map, B200_DTYPE_INT8, base, 2, dims, strides, box);
}

// 256 x 256 tiles on CTA pairs from 256 tokens on (and outputs wider than half a tile); below that the
// swapped kernel with the narrowest token tile that takes the tokens.  Pairs / swapped, 4096 x 4096
// weights: 256 tokens 23.6 / 27.3 us, 512 24.3 / 34.1, 1024 26.3 / 25.8.
template <typename T> static int launch_tc(const Params &p, cudaStream_t stream) {
  TcParams t;
  t.p = p;
  t.status = device_status_word();
  if (t.status == nullptr) return fail(B200_RESOURCE, "no status word on this device");
  t.vector_store = (p.y_row * (int64_t)sizeof(T)) % 16 == 0 && (uintptr_t)p.y % 16 == 0;
  t.vector_cols = (uintptr_t)p.w_scale % 16 == 0 && (uintptr_t)p.bias % 16 == 0;
  CUtensorMap tm_x, tm_w;
  int st;
  if (p.M >= 256 && p.N > 128) {
    if ((st = byte_map(&tm_x, p.x, p.M, p.K, p.x_row, 128)) || (st = byte_map(&tm_w, p.w, p.N, p.K, p.w_row, 128)))
      return st;
    // rows of x per raster group that stay within 40 MiB of L2 while w streams past them
    const int m_pairs = (p.M + 255) / 256;
    int most = (int)(((int64_t)40 << 20) / ((int64_t)256 * p.K));
    if (most < 2) most = 2;
    const int groups = (m_pairs + most - 1) / most;
    t.group_m = (m_pairs + groups - 1) / groups;
    return launch_pair<T>(tm_x, tm_w, t, stream);
  }
  const int tn = p.M <= 32 ? 32 : (p.M <= 64 ? 64 : (p.M <= 128 ? 128 : 256));
  t.group_m = 1;
  if ((st = byte_map(&tm_w, p.w, p.N, p.K, p.w_row, 128)) || (st = byte_map(&tm_x, p.x, p.M, p.K, p.x_row, tn)))
    return st;
  switch (tn) {
    case 32: return launch_skinny<T, 32>(tm_w, tm_x, t, stream);
    case 64: return launch_skinny<T, 64>(tm_w, tm_x, t, stream);
    case 128: return launch_skinny<T, 128>(tm_w, tm_x, t, stream);
    default: return launch_skinny<T, 256>(tm_w, tm_x, t, stream);
  }
}

template <typename T> static int launch(const Params &p, cudaStream_t stream) {
  // tensor maps want rows 16-byte aligned and apart
  if (p.x_row > 0 && p.w_row > 0 && p.x_row % 16 == 0 && p.w_row % 16 == 0 && ((uintptr_t)p.x | (uintptr_t)p.w) % 16 == 0)
    return launch_tc<T>(p, stream);
  const dim3 grid((unsigned)((p.N + TILE - 1) / TILE), (unsigned)((p.M + TILE - 1) / TILE));
  if (grid.y > 65535u) return fail(B200_REJECTED, "%d rows exceed the limit of the unaligned path", p.M);
  linear_int8_tile_kernel<T><<<grid, 256, 0, stream>>>(p);
  B200_CUDA_OK(cudaGetLastError());
  return B200_OK;
}

}  // namespace int8
}  // namespace b200

extern "C" int b200_quantize_rows(const b200_tensor *x, b200_tensor *out, b200_tensor *scale, void *stream) {
  using namespace b200;
  int st;
  if ((st = check_tensor(x, "x", 2)) || (st = check_tensor(out, "out", 2)) || (st = check_tensor(scale, "scale", 1)))
    return st;
  const int64_t M = x->shape[0], K = x->shape[1];
  B200_REQUIRE(is_float_io(x->dtype), "x: dtype %u is not f16/bf16/f32", x->dtype);
  B200_REQUIRE(out->dtype == B200_DTYPE_INT8 && out->shape[0] == M && out->shape[1] == K, "out must be int8 [M, K]");
  B200_REQUIRE(scale->dtype == B200_DTYPE_FLOAT32 && scale->shape[0] == M && scale->stride[0] == 1,
               "scale must be contiguous f32 [M]");
  B200_REQUIRE(x->stride[1] == 1 && out->stride[1] == 1, "x and out need a unit column stride");
  B200_REQUIRE(M < (1ll << 31) && K < (1ll << 31), "rows or columns out of range");
  if (M == 0) return B200_OK;
  if ((st = check_reachable(x->data, "x")) || (st = check_reachable(out->data, "out")) ||
      (st = check_reachable(scale->data, "scale")))
    return st;
  int8::QuantParams p;
  p.x = x->data; p.out = (int8_t *)out->data; p.scale = (float *)scale->data;
  p.x_row = x->stride[0]; p.o_row = out->stride[0]; p.M = (int)M; p.K = (int)K;
  cudaStream_t s = (cudaStream_t)stream;
  if (x->dtype == B200_DTYPE_FLOAT32) return int8::launch_quantize<float>(p, s);
  if (x->dtype == B200_DTYPE_FLOAT16) return int8::launch_quantize<__half>(p, s);
  return int8::launch_quantize<__nv_bfloat16>(p, s);
}

extern "C" int b200_linear_int8(const b200_tensor *x, const b200_tensor *x_scale, const b200_tensor *w,
                                const b200_tensor *w_scale, const b200_tensor *bias, b200_tensor *y, int act,
                                void *stream) {
  using namespace b200;
  int st;
  if ((st = check_tensor(x, "x", 2)) || (st = check_tensor(x_scale, "x_scale", 1)) || (st = check_tensor(w, "w", 2)) ||
      (st = check_tensor(w_scale, "w_scale", 1)) || (st = check_tensor(y, "y", 2)))
    return st;
  const int64_t M = x->shape[0], K = x->shape[1], N = w->shape[0];
  B200_REQUIRE(x->dtype == B200_DTYPE_INT8 && w->dtype == B200_DTYPE_INT8, "x and w must be int8");
  B200_REQUIRE(w->shape[1] == K, "x has %lld columns, w has %lld", (long long)K, (long long)w->shape[1]);
  B200_REQUIRE(K >= 1 && K <= int8::kMaxK, "K %lld out of range 1..%lld (32-bit sums)", (long long)K,
               (long long)int8::kMaxK);
  B200_REQUIRE(is_float_io(y->dtype) && y->shape[0] == M && y->shape[1] == N, "y must be f16/bf16/f32 [M, N]");
  B200_REQUIRE(x_scale->dtype == B200_DTYPE_FLOAT32 && x_scale->shape[0] == M && x_scale->stride[0] == 1,
               "x_scale must be contiguous f32 [M]");
  B200_REQUIRE(w_scale->dtype == B200_DTYPE_FLOAT32 && w_scale->shape[0] == N && w_scale->stride[0] == 1,
               "w_scale must be contiguous f32 [N]");
  B200_REQUIRE(x->stride[1] == 1 && w->stride[1] == 1 && y->stride[1] == 1, "x, w and y need a unit column stride");
  if (bias != nullptr) {
    if ((st = check_tensor(bias, "bias", 1))) return st;
    B200_REQUIRE(bias->shape[0] == N && bias->stride[0] == 1 && is_float_io(bias->dtype),
                 "bias must be contiguous f16/bf16/f32 [N]");
  }
  if (act != B200_ACT_NONE && act != B200_ACT_GELU_ERF && act != B200_ACT_GELU_TANH && act != B200_ACT_LEAKY_RELU)
    return fail(B200_USAGE, "activation %d is not available here", act);
  B200_REQUIRE(M < (1ll << 31) && N < (1ll << 31), "rows or columns out of range");
  if (M == 0 || N == 0) return B200_OK;
  if ((st = check_reachable(x->data, "x", true)) || (st = check_reachable(x_scale->data, "x_scale")) ||
      (st = check_reachable(w->data, "w", true)) || (st = check_reachable(w_scale->data, "w_scale")) ||
      (st = check_reachable(bias ? bias->data : nullptr, "bias")) || (st = check_reachable(y->data, "y")))
    return st;
  int8::Params p;
  p.x = (const int8_t *)x->data; p.w = (const int8_t *)w->data;
  p.x_scale = (const float *)x_scale->data; p.w_scale = (const float *)w_scale->data;
  p.bias = bias ? bias->data : nullptr;
  p.bias_kind = bias ? (int)bias->dtype : 0;
  p.y = y->data;
  p.x_row = x->stride[0]; p.w_row = w->stride[0]; p.y_row = y->stride[0];
  p.M = (int)M; p.N = (int)N; p.K = (int)K; p.act = act;
  cudaStream_t s = (cudaStream_t)stream;
  if (y->dtype == B200_DTYPE_FLOAT32) return int8::launch<float>(p, s);
  if (y->dtype == B200_DTYPE_FLOAT16) return int8::launch<__half>(p, s);
  return int8::launch<__nv_bfloat16>(p, s);
}
