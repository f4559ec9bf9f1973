// Appending keys and values to a paged cache, with the position rotation applied on the way.
//
// Token t of a call belongs to sequence seq[t] (a row of the page table; negative: padding) and
// stands at position pos[t]: its key and value rows go to row pos % block of physical page
// page_table[seq][pos / block].  Keys -- and, on the way, the query rows of the same tokens --
// are rotated by the angles of their position first: a pair (a, b) becomes
// (a cos - b sin, b cos + a sin), the pairs being elements (i, i + R/2) or (2i, 2i + 1) of the
// first R of a row.
//
// A cache of 8-bit words holds a row in 4-bit codes: the row stands for low + code * scale with
// low = min(row), scale = (max(row) - low) / 15 rounded to the row's type and code =
// (x - low) / scale rounded to the nearest whole number, ties to even.  What is quantised is the
// rotated row rounded to its type, so the codes are the ones a 16-bit cache would have given.
//
// Which code a value next to a border gets must not depend on the order of roundings, so the
// rotation keeps the rounding errors of both products and of their sum (error-free
// transformations: a product's error by one fused multiply-add, a sum's by Knuth's two-sum) and
// is rounded ONCE to the row's type; the scale is a 64-bit quotient rounded once; and a code whose
// 32-bit quotient is within 1e-5 of a border is decided by the 64-bit quotient.
//
// Measured, heads of 128: 16385 fp16 tokens of 32 + 32 heads into a 16-bit cache 153 us (5.3 TB/s of the 809
// MB that go in and out; the copy rate would give 123), 32768 tokens of 32 + 8 heads into 4 bits 234 us
// (3.7 TB/s; 131): the arithmetic of the exact rounding and of the codes takes the issue slots.  64
// tokens into 16 bits 3.1 us, 256 into 4 bits 6.3: the latency of token, page, row and store in turn.
#include "common.cuh"

#include <type_traits>

namespace b200 {
namespace append {

constexpr int kMaxDim = 512;
constexpr unsigned kSiteToken = 50, kSitePage = 51;

struct Params {
  const void *q, *k, *v;            // [T, heads, D]
  void *q_out, *k_out, *v_out;      // q_out iff q; k_out / v_out may be null
  void *k_cache, *v_cache;          // [pages, HK, block, D] in T, or [pages, HK, block, D / 2] codes
  void *k_params, *v_params;        // 4 bits: [pages, HK, block, 2] (scale, low) in T
  const int *table, *seq, *pos;
  const float *cos_t, *sin_t;       // [angles, R / 2]
  int64_t q_t, q_h, k_t, k_h, v_t, v_h;              // element strides of the inputs
  int64_t qo_t, qo_h, ko_t, ko_h, vo_t, vo_h;        // and of the outputs
  int64_t kc_p, kc_h, kc_r, vc_p, vc_h, vc_r;        // cache: page, head, row
  int64_t kp_p, kp_h, kp_r, vp_p, vp_h, vp_r;        // params
  int64_t table_row, cos_row, sin_row;
  int T, H, HK, D, R, pages, width, seqs, block, angles;
  int interleaved;
  unsigned int *status;
};

// x + y = s + e exactly
__device__ __forceinline__ void two_sum(float x, float y, float &s, float &e) {
  s = __fadd_rn(x, y);
  const float t = __fsub_rn(s, x);
  e = __fadd_rn(__fsub_rn(x, __fsub_rn(s, t)), __fsub_rn(y, t));
}

// a c + b s, rounded once to T (returned as a float that T holds)
template <typename T>
__device__ __forceinline__ float turn(float a, float c, float b, float s) {
  const float p = __fmul_rn(a, c), q = __fmul_rn(b, s);
  const float ep = __fmaf_rn(a, c, -p), eq = __fmaf_rn(b, s, -q);
  float sum, es, hi, lo;
  two_sum(p, q, sum, es);
  if (!(fabsf(sum) < INFINITY)) return io<T>::load(io<T>::store(sum));
  two_sum(sum, __fadd_rn(es, __fadd_rn(ep, eq)), hi, lo);
  if constexpr (std::is_same<T, float>::value) {
    return hi;
  } else {
    // round to odd: a neighbour of `hi` stands for "not exactly hi", so the second rounding
    // decides as the exact value would
    uint32_t u = __float_as_uint(hi);
    if (lo != 0.f && (u & 1u) == 0u) u += ((lo > 0.f) == (hi > 0.f)) ? 1u : 0xffffffffu;
    return io<T>::load(io<T>::store(__uint_as_float(u)));
  }
}

// the non-negative 64-bit value rounded once to T
template <typename T> __device__ __forceinline__ float round_once(double x) {
  if constexpr (std::is_same<T, float>::value) return __double2float_rn(x);
  float f = __double2float_rz(x);
  if ((double)f != x) f = __uint_as_float(__float_as_uint(f) | 1u);
  return io<T>::load(io<T>::store(f));
}

template <typename T> __device__ __forceinline__ float scale_of(float low, float high) {
  return round_once<T>(((double)high - (double)low) / 15.0);
}

// code of x in a row with (scale, low); inv = 1 / scale
__device__ __forceinline__ uint32_t code_of(float x, float scale, float low, float inv) {
  if (!(scale > 0.f)) return 0u;
  const float y = (x - low) * inv;  // within 3e-6 of the quotient while 1 / scale is a normal number
  float r = rintf(y);
  if (!(fabsf(fabsf(y - r) - 0.5f) > 1e-5f) || scale < 1e-30f)
    r = (float)rint(((double)x - (double)low) / (double)scale);
  return (uint32_t)fminf(fmaxf(r, 0.f), 15.f);
}

// Where token t's rows go: false when they go nowhere (padding, or an index outside its table).
struct Place {
  int page, row, pos;
};
// raw: a token's seq, pos and the page the table gave for them, if they are in it
template <typename Raw> __device__ __forceinline__ bool place_of(const Params &p, const Raw &raw, Place &at) {
  if (raw.seq < 0) return false;
  if (raw.seq >= p.seqs || raw.pos < 0 || raw.pos / p.block >= p.width || (p.R > 0 && raw.pos >= p.angles)) {
    report_rejected(p.status, kSiteToken);
    return false;
  }
  if (raw.page < 0 || raw.page >= p.pages) {
    report_rejected(p.status, kSitePage);
    return false;
  }
  at.page = raw.page;
  at.row = raw.pos % p.block;
  at.pos = raw.pos;
  return true;
}
struct Raw {
  int seq, pos, page;
};
__device__ __forceinline__ Raw read_token(const Params &p, int64_t t) {
  return Raw{__ldg(p.seq + t), __ldg(p.pos + t), -1};
}
__device__ __forceinline__ void read_page(const Params &p, Raw &r) {
  if (r.seq >= 0 && r.seq < p.seqs && r.pos >= 0 && r.pos / p.block < p.width)
    r.page = __ldg(p.table + (int64_t)r.seq * p.table_row + r.pos / p.block);
}

// Any head size up to 512, any strides and alignment: one warp per row, staged in shared memory.
constexpr int WARPS = 4;

template <typename T, bool FOUR>
__global__ void __launch_bounds__(WARPS * 32) kv_append_rows_kernel(const Params p) {
  __shared__ float stage[WARPS][kMaxDim];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_token = p.H + 2 * p.HK;
  const int64_t item = (int64_t)blockIdx.x * WARPS + warp;
  if (item >= (int64_t)p.T * per_token) return;
  const int t = (int)(item / per_token), r = (int)(item % per_token);
  Raw raw = read_token(p, t);
  read_page(p, raw);
  Place at;
  if (!place_of(p, raw, at)) return;
  const bool is_q = r < p.H, is_v = r >= p.H + p.HK;
  const int h = is_q ? r : (is_v ? r - p.H - p.HK : r - p.H);
  const T *src = is_q ? (const T *)p.q + t * p.q_t + h * p.q_h
                      : (is_v ? (const T *)p.v + t * p.v_t + h * p.v_h
                              : (const T *)p.k + t * p.k_t + h * p.k_h);
  float *x = stage[warp];
  const int R = is_v ? 0 : p.R, half = R / 2;
  for (int i = lane; i < half; i += 32) {
    const int ia = p.interleaved ? 2 * i : i, ib = p.interleaved ? 2 * i + 1 : i + half;
    const float a = io<T>::load(src[ia]), b = io<T>::load(src[ib]);
    const float c = p.cos_t[(int64_t)at.pos * p.cos_row + i];
    const float s = p.sin_t[(int64_t)at.pos * p.sin_row + i];
    x[ia] = turn<T>(a, c, b, -s);
    x[ib] = turn<T>(b, c, a, s);
  }
  for (int i = R + lane; i < p.D; i += 32) x[i] = io<T>::load(src[i]);
  __syncwarp();  // the whole row is read: it may be written in place

  if (is_q) {
    T *dst = (T *)p.q_out + t * p.qo_t + h * p.qo_h;
    for (int i = lane; i < p.D; i += 32) dst[i] = io<T>::store(x[i]);
    return;
  }
  T *copy = is_v ? (T *)p.v_out : (T *)p.k_out;
  if (copy != nullptr) copy += is_v ? t * p.vo_t + h * p.vo_h : t * p.ko_t + h * p.ko_h;
  const int64_t slot = is_v ? at.page * p.vc_p + h * p.vc_h + at.row * p.vc_r
                            : at.page * p.kc_p + h * p.kc_h + at.row * p.kc_r;
  if constexpr (!FOUR) {
    T *dst = (T *)(is_v ? p.v_cache : p.k_cache) + slot;
    for (int i = lane; i < p.D; i += 32) {
      const T e = io<T>::store(x[i]);
      dst[i] = e;
      if (copy != nullptr) copy[i] = e;
    }
  } else {
    float low = INFINITY, high = -INFINITY;
    bool finite = true;
    for (int i = lane; i < p.D; i += 32) {
      low = fminf(low, x[i]);
      high = fmaxf(high, x[i]);
      finite = finite && fabsf(x[i]) < INFINITY;
    }
    high = warp_max(high);
    low = -warp_max(-low);
    finite = __all_sync(0xffffffffu, finite);
    float scale = scale_of<T>(low, high);
    if (!finite) scale = low = __int_as_float(0x7fffffff);  // the row reads back as NaN
    const float inv = 1.f / scale;
    uint8_t *dst = (uint8_t *)(is_v ? p.v_cache : p.k_cache) + slot;
    for (int i = lane; i < p.D / 2; i += 32) {
      const uint32_t a = code_of(x[2 * i], scale, low, inv), b = code_of(x[2 * i + 1], scale, low, inv);
      dst[i] = (uint8_t)(a | (b << 4));
      if (copy != nullptr) {
        copy[2 * i] = io<T>::store(fmaf((float)a, scale, low));
        copy[2 * i + 1] = io<T>::store(fmaf((float)b, scale, low));
      }
    }
    if (lane == 0) {
      T *par = is_v ? (T *)p.v_params + at.page * p.vp_p + h * p.vp_h + at.row * p.vp_r
                    : (T *)p.k_params + at.page * p.kp_p + h * p.kp_h + at.row * p.kp_r;
      par[0] = io<T>::store(scale);
      par[1] = io<T>::store(low);
    }
  }
}

// Rows of 8, 16 or 32 16-byte vectors on 16-byte boundaries (16-bit heads of 64, 128 and 256, 32-bit ones of
// 32, 64 and 128): a lane holds two vectors of a row, the two that the rotation pairs, so a row is
// read once, turned, reduced and written without leaving its lanes.  A block takes one token (or a
// part of its rows); a thread keeps its angles while it walks over the rows (heads), the next row on
// its way.
//
// Bound by HBM in a prefill, so the arithmetic of the exact rounding has to be cheap: a c + b s in
// plain 32-bit arithmetic is off by at most 2^-23 (|a c| + |b s|), and where the ends of that interval
// round to the same 16-bit value, so does the exact sum.  Only elements whose interval holds a
// border (one in some thousands) take the error-free path above.
//
// Small blocks, many of them: each begins with three dependent reads (sequence and position, page,
// angles), which only other blocks can hide.  128 threads, seven blocks per SM: 152 us where 256
// threads and four took 187 (16385 fp16 tokens, 96 rows of 128 each), and a persistent grid with the
// next token's reads on their way 211.
constexpr int THREADS = 128;

template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
  } else {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
  }
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  else
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}

// Two elements: own c + other s, rounded once to T -- unless *differ comes back non-zero: then the two
// ends of the interval round to different values.
template <typename T>
__device__ __forceinline__ uint32_t turn_two(float2 own, float2 other, float2 c, float2 s, uint32_t &differ) {
  constexpr float kOff = 1.4901161193847656e-07f;  // 1.25 * 2^-23
  const float2 p = mul2(own, c), q = mul2(other, s), sum = fma2(other, s, p);
  const float2 size = make_float2(fabsf(p.x) + fabsf(q.x), fabsf(p.y) + fabsf(q.y));
  const float2 low = fma2(size, splat(-kOff), sum), high = fma2(size, splat(kOff), sum);
  const uint32_t r = pack2<T>(low.x, low.y);
  differ = r ^ pack2<T>(high.x, high.y);
  return r;
}
template <typename T>
__device__ __forceinline__ uint32_t turn_two_exactly(float2 own, float2 other, float2 c, float2 s) {
  return pack2<T>(turn<T>(own.x, c.x, other.x, s.x), turn<T>(own.y, c.y, other.y, s.y));
}

// The angles of a lane's two vectors: by pairs of elements for vectors that turn with one another
// (c, s for both), one each per pair of neighbours for vectors that turn in themselves.
template <typename T, bool NEIGHBOURS> struct Angles {
  static constexpr int N = vec16<T>::N;
  float c[N], s[N];

  __device__ __forceinline__ void load(const float *cs, const float *sn, int first, int second) {
    if constexpr (NEIGHBOURS) {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        c[i] = __ldg(cs + first / 2 + i);
        s[i] = __ldg(sn + first / 2 + i);
        c[N / 2 + i] = __ldg(cs + second / 2 + i);
        s[N / 2 + i] = __ldg(sn + second / 2 + i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const float4 a = __ldg(reinterpret_cast<const float4 *>(cs + first + i));
        const float4 b = __ldg(reinterpret_cast<const float4 *>(sn + first + i));
        c[i] = a.x; c[i + 1] = a.y; c[i + 2] = a.z; c[i + 3] = a.w;
        s[i] = b.x; s[i + 1] = b.y; s[i + 2] = b.z; s[i + 3] = b.w;
      }
    }
  }
  // c, s of elements 2i, 2i + 1 of vector v (0, 1); the sign of the sine in it
  __device__ __forceinline__ float2 cos2(int v, int i) const {
    if constexpr (NEIGHBOURS) return splat(c[v * (N / 2) + i]);
    else return make_float2(c[2 * i], c[2 * i + 1]);
  }
  __device__ __forceinline__ float2 sin2(int v, int i) const {
    if constexpr (NEIGHBOURS) return make_float2(-s[v * (N / 2) + i], s[v * (N / 2) + i]);
    else return v == 0 ? make_float2(-s[2 * i], -s[2 * i + 1]) : make_float2(s[2 * i], s[2 * i + 1]);
  }
};

// Elements 2i, 2i + 1 of a vector as floats, and back.
template <typename T> __device__ __forceinline__ float2 two_of(const uint32_t (&x)[4], int i) {
  if constexpr (std::is_same<T, float>::value) return make_float2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1]));
  else return unpack2<T>(x[i]);
}
template <typename T> __device__ __forceinline__ void put_two(uint32_t (&x)[4], int i, float2 v) {
  if constexpr (std::is_same<T, float>::value) {
    x[2 * i] = __float_as_uint(v.x);
    x[2 * i + 1] = __float_as_uint(v.y);
  } else {
    x[i] = pack2<T>(v.x, v.y);
  }
}

// A lane's two vectors, turned.
template <typename T, bool NEIGHBOURS>
__device__ __forceinline__ void turn_vectors(uint32_t (&x)[2][4], const Angles<T, NEIGHBOURS> &angle) {
  constexpr int N = vec16<T>::N;
  float2 own[2][N / 2];
#pragma unroll
  for (int v = 0; v < 2; ++v)
#pragma unroll
    for (int i = 0; i < N / 2; ++i) own[v][i] = two_of<T>(x[v], i);
  auto other = [&](int v, int i) {
    return NEIGHBOURS ? make_float2(own[v][i].y, own[v][i].x) : own[1 - v][i];
  };
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        const float2 o = other(v, i), c = angle.cos2(v, i), s = angle.sin2(v, i);
        put_two<T>(x[v], i, make_float2(turn<T>(own[v][i].x, c.x, o.x, s.x), turn<T>(own[v][i].y, c.y, o.y, s.y)));
      }
  } else {
    uint32_t differ[2][4], any = 0;
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[v][i] = turn_two<T>(own[v][i], other(v, i), angle.cos2(v, i), angle.sin2(v, i), differ[v][i]);
        any |= differ[v][i];
      }
    if (any != 0) {
#pragma unroll
      for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (differ[v][i] != 0) x[v][i] = turn_two_exactly<T>(own[v][i], other(v, i), angle.cos2(v, i), angle.sin2(v, i));
    }
  }
}

// (high - low) / 15 rounded once to T, without 64-bit arithmetic for 16-bit types: the difference with its
// rounding error, a quotient corrected once by its remainder, and the sign of the remainder that is
// left for the second rounding.
template <typename T> __device__ __forceinline__ float scale_of_fast(float low, float high) {
  if constexpr (std::is_same<T, float>::value) return scale_of<T>(low, high);
  float d, e;
  two_sum(high, -low, d, e);
  if (!(d < INFINITY)) return scale_of<T>(low, high);
  constexpr float k15 = 1.f / 15.f;
  const float q0 = __fmul_rn(d, k15);
  const float q = __fmaf_rn(__fadd_rn(__fmaf_rn(-15.f, q0, d), e), k15, q0);
  const float left = __fadd_rn(__fmaf_rn(-15.f, q, d), e);
  uint32_t u = __float_as_uint(q);
  if (left != 0.f && (u & 1u) == 0u) u += left > 0.f ? 1u : 0xffffffffu;  // q >= 0; if 0, nothing is left
  return io<T>::load(io<T>::store(__uint_as_float(u)));
}

__device__ __forceinline__ void load16(uint32_t (&x)[4], const void *src) {
  const uint4 v = *reinterpret_cast<const uint4 *>(src);
  x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
}
__device__ __forceinline__ void store16(void *dst, const uint32_t (&x)[4]) {
  *reinterpret_cast<uint4 *>(dst) = make_uint4(x[0], x[1], x[2], x[3]);
}

// LANES lanes with two vectors each hold a row.
template <typename T, bool FOUR, bool NEIGHBOURS, int LANES>
__global__ void __launch_bounds__(THREADS, 7) kv_append_vector_kernel(const Params p, int chunks) {
  constexpr int N = vec16<T>::N, GROUPS = THREADS / LANES;
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const int t = (int)(blockIdx.x / chunks), rows = p.H + 2 * p.HK;
  const int per_chunk = (rows + chunks - 1) / chunks;
  const int first = (int)(blockIdx.x % chunks) * per_chunk, last = min(rows, first + per_chunk);
  // query rows [first, q_last), key and value rows [kv_first, last) of the token are this block's
  const int q_last = min(last, p.H), kv_first = max(first, p.H);
  // this lane's vectors begin at elements e0 and e1: partners of the rotation, or two behind it
  const int turning = p.R / (2 * N);  // lanes whose vectors turn
  const bool turns = lane < turning;
  const int e0 = turns ? lane * N : 2 * lane * N, e1 = turns ? e0 + p.R / 2 : e0 + N;
  const T *q_src = (const T *)p.q + t * p.q_t + (int64_t)(first + group) * p.q_h;
  const T *k_src = (const T *)p.k + t * p.k_t, *v_src = (const T *)p.v + t * p.v_t;
  auto kv_row = [&](int r) { return r < p.H + p.HK ? k_src + (r - p.H) * p.k_h : v_src + (r - p.H - p.HK) * p.v_h; };
  uint32_t q_next[2][4];
  auto load_row = [&](uint32_t (&x)[2][4], const T *row) {
    load16(x[0], row + e0);
    load16(x[1], row + e1);
  };
  if (first + group < q_last) load_row(q_next, q_src);
  Raw raw = read_token(p, t);
  read_page(p, raw);
  Place at;
  if (!place_of(p, raw, at)) return;  // the same for the whole block

  Angles<T, NEIGHBOURS> angle;
  if (turns) angle.load(p.cos_t + (int64_t)at.pos * p.cos_row, p.sin_t + (int64_t)at.pos * p.sin_row, e0, e1);

  T *q_dst = (T *)p.q_out + t * p.qo_t + (int64_t)(first + group) * p.qo_h;
  const int64_t q_step = GROUPS * p.q_h, qo_step = GROUPS * p.qo_h;
  for (int r = first + group; r < q_last; r += GROUPS) {
    uint32_t x[2][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[0][i] = q_next[0][i];
      x[1][i] = q_next[1][i];
    }
    q_src += q_step;
    if (r + GROUPS < q_last) load_row(q_next, q_src);
    if (turns) turn_vectors<T, NEIGHBOURS>(x, angle);
    store16(q_dst + e0, x[0]);
    store16(q_dst + e1, x[1]);
    q_dst += qo_step;
  }

  const int64_t k_slot = at.page * p.kc_p + at.row * p.kc_r, v_slot = at.page * p.vc_p + at.row * p.vc_r;
  for (int base = kv_first; base < last; base += GROUPS) {  // whole warps: the exchanges below are full
    const int r = base + group;
    const bool have = r < last, is_v = r >= p.H + p.HK;
    uint32_t x[2][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[0][i] = x[1][i] = 0u;
    }
    if (have) load_row(x, kv_row(r));
    if (turns && have && !is_v) turn_vectors<T, NEIGHBOURS>(x, angle);
    const int h = is_v ? r - p.H - p.HK : r - p.H;
    T *copy = is_v ? (T *)p.v_out : (T *)p.k_out;
    if (copy != nullptr) copy += is_v ? t * p.vo_t + h * p.vo_h : t * p.ko_t + h * p.ko_h;
    const int64_t slot = is_v ? v_slot + h * p.vc_h : k_slot + h * p.kc_h;
    if constexpr (!FOUR) {
      if (!have) continue;
      T *dst = (T *)(is_v ? p.v_cache : p.k_cache) + slot;
      store16(dst + e0, x[0]);
      store16(dst + e1, x[1]);
      if (copy != nullptr) {
        store16(copy + e0, x[0]);
        store16(copy + e1, x[1]);
      }
    } else {
      float2 f[2][N / 2];
      float low = INFINITY, high = -INFINITY;
      float2 odd = splat(0.f);
#pragma unroll
      for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          f[v][i] = two_of<T>(x[v], i);
          low = fminf(low, fminf(f[v][i].x, f[v][i].y));
          high = fmaxf(high, fmaxf(f[v][i].x, f[v][i].y));
          odd = fma2(f[v][i], splat(0.f), odd);  // not a number once an element is not finite
        }
#pragma unroll
      for (int o = 1; o < LANES; o <<= 1) {
        low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
        high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
      }
      constexpr uint32_t kGroup = (1u << LANES) - 1u;
      const uint32_t broken =
          __ballot_sync(0xffffffffu, !(odd.x + odd.y == 0.f)) >> ((threadIdx.x & 31) / LANES * LANES) & kGroup;
      if (!have) continue;
      float scale = scale_of_fast<T>(low, high);
      if (broken != 0) scale = low = __int_as_float(0x7fffffff);  // the row reads back as NaN
      const float inv = __fdividef(1.f, scale);
      // Codes by adding 1.5 * 2^23, which rounds to whole numbers, ties to even: the sum's bits are the
      // constant's plus the code, so the word of codes is a sum of bits times powers of 16.
      constexpr float kMove = 12582912.f;
      constexpr uint32_t kMoveBits = 0x4b400000u;
      uint32_t word[2] = {0u, 0u};
      float2 code[2][N / 2];
      float far = 0.f;
#pragma unroll
      for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          const float2 y = mul2(add2(f[v][i], splat(-low)), splat(inv));
          const float2 moved = add2(make_float2(fminf(y.x, 15.f), fminf(y.y, 15.f)), splat(kMove));
          code[v][i] = add2(moved, splat(-kMove));
          const float2 off = fma2(code[v][i], splat(-1.f), y);
          far = fmaxf(far, fmaxf(fabsf(off.x), fabsf(off.y)));
          word[v] += (__float_as_uint(moved.x) - kMoveBits) * (1u << (8 * i));
          word[v] += (__float_as_uint(moved.y) - kMoveBits) * (16u << (8 * i));
        }
      // a border within the quotient's error, a quotient above 15.5, a scale of zero or not a number
      if (!(far < 0.49999f) || !(scale >= 1e-30f)) {
        const float exact_inv = 1.f / scale;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          word[v] = 0;
#pragma unroll
          for (int i = 0; i < N / 2; ++i) {
            const uint32_t a = code_of(f[v][i].x, scale, low, exact_inv), b = code_of(f[v][i].y, scale, low, exact_inv);
            word[v] |= (a << (8 * i)) | (b << (8 * i + 4));
            code[v][i] = make_float2((float)a, (float)b);
          }
        }
      }
      uint8_t *dst = (uint8_t *)(is_v ? p.v_cache : p.k_cache) + slot;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const int e = v == 0 ? e0 : e1;
        if constexpr (N == 8) *reinterpret_cast<uint32_t *>(dst + e / 2) = word[v];
        else *reinterpret_cast<uint16_t *>(dst + e / 2) = (uint16_t)word[v];
        if (copy != nullptr) {
          uint32_t out[4];
#pragma unroll
          for (int i = 0; i < N / 2; ++i) put_two<T>(out, i, fma2(code[v][i], splat(scale), splat(low)));
          store16(copy + e, out);
        }
      }
      if (lane == 0) {
        T *par = is_v ? (T *)p.v_params + at.page * p.vp_p + h * p.vp_h + at.row * p.vp_r
                      : (T *)p.k_params + at.page * p.kp_p + h * p.kp_h + at.row * p.kp_r;
        par[0] = io<T>::store(scale);
        par[1] = io<T>::store(low);
      }
    }
  }
}

// What the vector kernel takes.
template <typename T> static bool takes_vectors(const Params &p, bool four) {
  constexpr int N = vec16<T>::N;
  const int vectors = p.D / N;
  if (p.D % N != 0 || (vectors != 8 && vectors != 16 && vectors != 32)) return false;
  if (p.R > 0) {
    if (p.R % (2 * N) != 0) return false;  // whole vectors that turn with one another
    if (!p.interleaved && (((uintptr_t)p.cos_t | (uintptr_t)p.sin_t) % 16 != 0 || p.cos_row % 4 != 0 || p.sin_row % 4 != 0))
      return false;
  }
  uintptr_t bases = (uintptr_t)p.q | (uintptr_t)p.k | (uintptr_t)p.v | (uintptr_t)p.q_out | (uintptr_t)p.k_out | (uintptr_t)p.v_out;
  int64_t strides = p.q_t | p.q_h | p.k_t | p.k_h | p.v_t | p.v_h | p.qo_t | p.qo_h | p.ko_t | p.ko_h | p.vo_t | p.vo_h;
  const int64_t cache = p.kc_p | p.kc_h | p.kc_r | p.vc_p | p.vc_h | p.vc_r;
  const uintptr_t cache_base = (uintptr_t)p.k_cache | (uintptr_t)p.v_cache;
  if (four) {
    if (cache % (N / 2) != 0 || cache_base % (N / 2) != 0) return false;
  } else {
    strides |= cache;
    bases |= cache_base;
  }
  return bases % 16 == 0 && strides % N == 0;
}

template <typename T, bool FOUR, int LANES> static int launch_vectors(const Params &p, cudaStream_t stream) {
  // a block per token; few tokens: its rows in as many blocks as there are passes over them
  const int rows = p.H + 2 * p.HK, passes = (rows + THREADS / LANES - 1) / (THREADS / LANES);
  const int chunks = p.T >= 8 * sm_count() ? 1 : passes;
  auto kernel = p.interleaved ? kv_append_vector_kernel<T, FOUR, true, LANES> : kv_append_vector_kernel<T, FOUR, false, LANES>;
  kernel<<<(unsigned)((int64_t)p.T * chunks), THREADS, 0, stream>>>(p, chunks);
  B200_CUDA_OK(cudaGetLastError());
  return B200_OK;
}

template <typename T, bool FOUR> static int launch(const Params &p, cudaStream_t stream) {
  if (takes_vectors<T>(p, FOUR) && (int64_t)p.T * (p.H + 2 * p.HK) < (1ll << 31)) {
    switch (p.D / vec16<T>::N) {
      case 8: return launch_vectors<T, FOUR, 4>(p, stream);
      case 16: return launch_vectors<T, FOUR, 8>(p, stream);
      default: return launch_vectors<T, FOUR, 16>(p, stream);
    }
  }
  const int64_t rows = (int64_t)p.T * (p.H + 2 * p.HK);
  kv_append_rows_kernel<T, FOUR><<<(unsigned)((rows + WARPS - 1) / WARPS), WARPS * 32, 0, stream>>>(p);
  B200_CUDA_OK(cudaGetLastError());
  return B200_OK;
}

}  // namespace append
}  // namespace b200

extern "C" int b200_kv_append(const b200_tensor *k, const b200_tensor *v, b200_tensor *k_cache,
                              b200_tensor *v_cache, b200_tensor *k_params, b200_tensor *v_params,
                              const b200_tensor *page_table, const b200_tensor *seq,
                              const b200_tensor *pos, const b200_tensor *cos_table,
                              const b200_tensor *sin_table, int interleaved, const b200_tensor *q,
                              b200_tensor *q_out, b200_tensor *k_out, b200_tensor *v_out,
                              void *stream) {
  using namespace b200;
  int st;
  if ((st = check_tensor(k, "k", 3)) || (st = check_tensor(v, "v", 3)) ||
      (st = check_tensor(k_cache, "k_cache", 4)) || (st = check_tensor(v_cache, "v_cache", 4)) ||
      (st = check_tensor(page_table, "page_table", 2)) || (st = check_tensor(seq, "seq", 1)) ||
      (st = check_tensor(pos, "pos", 1)))
    return st;
  const int64_t T = k->shape[0], HK = k->shape[1], D = k->shape[2];
  const uint32_t dt = k->dtype;
  B200_REQUIRE(is_float_io(dt), "k: dtype %u is not f16/bf16/f32", dt);
  B200_REQUIRE(v->dtype == dt, "k and v have different dtypes");
  B200_REQUIRE(v->shape[0] == T && v->shape[1] == HK && v->shape[2] == D, "k and v must both be [T, H_KV, D]");
  B200_REQUIRE(D >= 1 && D <= append::kMaxDim, "head size %lld out of range 1..%d", (long long)D, append::kMaxDim);
  B200_REQUIRE(HK >= 1, "no K / V heads");
  const bool four = k_cache->dtype == B200_DTYPE_UINT8;
  B200_REQUIRE(k_cache->dtype == v_cache->dtype && (four || k_cache->dtype == dt),
               "the caches must both be of k's dtype, or uint8 (4-bit codes)");
  B200_REQUIRE(!four || D % 2 == 0, "a 4-bit cache needs an even head size");
  const int64_t pages = k_cache->shape[0], block = k_cache->shape[2];
  const int64_t last = four ? D / 2 : D;
  for (const b200_tensor *c : {(const b200_tensor *)k_cache, (const b200_tensor *)v_cache}) {
    B200_REQUIRE(c->shape[0] == pages && c->shape[1] == HK && c->shape[2] == block && c->shape[3] == last,
                 "both caches must be [pages, H_KV, block, %lld]", (long long)last);
    B200_REQUIRE(c->stride[3] == 1, "the caches need a unit last stride");
  }
  B200_REQUIRE(block >= 1 && pages < (1ll << 31) && block < (1ll << 31), "block size or pages out of range");
  B200_REQUIRE((k_params != nullptr) == four && (v_params != nullptr) == four,
               "k_params and v_params belong to a 4-bit cache, and only to it");
  if (four) {
    if ((st = check_tensor(k_params, "k_params", 4)) || (st = check_tensor(v_params, "v_params", 4))) return st;
    for (const b200_tensor *c : {(const b200_tensor *)k_params, (const b200_tensor *)v_params}) {
      B200_REQUIRE(c->dtype == dt, "the params must have k's dtype");
      B200_REQUIRE(c->shape[0] == pages && c->shape[1] == HK && c->shape[2] == block && c->shape[3] == 2,
                   "the params must be [pages, H_KV, block, 2]");
      B200_REQUIRE(c->stride[3] == 1, "the params need a unit last stride");
    }
  }
  B200_REQUIRE(page_table->dtype == B200_DTYPE_INT32 && seq->dtype == B200_DTYPE_INT32 &&
                   pos->dtype == B200_DTYPE_INT32, "page_table, seq and pos must be int32");
  B200_REQUIRE(page_table->stride[1] == 1, "page_table needs a unit last stride");
  B200_REQUIRE(seq->shape[0] == T && pos->shape[0] == T, "seq and pos need one entry per token");
  B200_REQUIRE(seq->stride[0] == 1 && pos->stride[0] == 1, "seq and pos must be contiguous");
  B200_REQUIRE(page_table->shape[0] < (1ll << 31) && page_table->shape[1] < (1ll << 31), "page_table out of range");
  B200_REQUIRE((cos_table != nullptr) == (sin_table != nullptr), "cos and sin come together");
  int64_t R = 0, angles = 0;
  if (cos_table != nullptr) {
    if ((st = check_tensor(cos_table, "cos", 2)) || (st = check_tensor(sin_table, "sin", 2))) return st;
    R = 2 * cos_table->shape[1];
    angles = cos_table->shape[0];
    B200_REQUIRE(cos_table->dtype == B200_DTYPE_FLOAT32 && sin_table->dtype == B200_DTYPE_FLOAT32,
                 "cos and sin must be f32");
    B200_REQUIRE(sin_table->shape[0] == angles && sin_table->shape[1] * 2 == R, "cos and sin differ in shape");
    B200_REQUIRE(R <= D, "%lld rotated elements in a head of %lld", (long long)R, (long long)D);
    B200_REQUIRE(cos_table->stride[1] == 1 && sin_table->stride[1] == 1, "cos and sin need a unit last stride");
    B200_REQUIRE(angles < (1ll << 31), "cos and sin out of range");
  }
  B200_REQUIRE((q != nullptr) == (q_out != nullptr), "q and q_out come together");
  int64_t H = 0;
  if (q != nullptr) {
    if ((st = check_tensor(q, "q", 3)) || (st = check_tensor(q_out, "q_out", 3))) return st;
    H = q->shape[1];
    for (const b200_tensor *c : {q, (const b200_tensor *)q_out})
      B200_REQUIRE(c->dtype == dt && c->shape[0] == T && c->shape[1] == H && c->shape[2] == D && c->stride[2] == 1,
                   "q and q_out must be [T, H, D] in k's dtype with a unit last stride");
  }
  B200_REQUIRE(k->stride[2] == 1 && v->stride[2] == 1, "k and v need a unit last stride");
  for (const b200_tensor *c : {(const b200_tensor *)k_out, (const b200_tensor *)v_out})
    if (c != nullptr) {
      if ((st = check_tensor(c, "k_out / v_out", 3))) return st;
      B200_REQUIRE(c->dtype == dt && c->shape[0] == T && c->shape[1] == HK && c->shape[2] == D && c->stride[2] == 1,
                   "k_out and v_out must be [T, H_KV, D] in k's dtype with a unit last stride");
    }
  B200_REQUIRE(H + 2 * HK < (1 << 20) && T < (1ll << 31) && T * (H + 2 * HK) < (1ll << 32), "tokens or heads out of range");
  if (T == 0) return B200_OK;

  append::Params p = {};
  const b200_tensor *all[] = {k, v, k_cache, v_cache, k_params, v_params, page_table, seq, pos,
                              cos_table, sin_table, q, q_out, k_out, v_out};
  static const char *const names[] = {"k", "v", "k_cache", "v_cache", "k_params", "v_params",
                                      "page_table", "seq", "pos", "cos", "sin", "q", "q_out", "k_out", "v_out"};
  for (int i = 0; i < 15; ++i)
    if (all[i] != nullptr && (st = check_reachable(all[i]->data, names[i]))) return st;
  p.k = k->data; p.v = v->data; p.k_cache = k_cache->data; p.v_cache = v_cache->data;
  p.k_t = k->stride[0]; p.k_h = k->stride[1]; p.v_t = v->stride[0]; p.v_h = v->stride[1];
  p.kc_p = k_cache->stride[0]; p.kc_h = k_cache->stride[1]; p.kc_r = k_cache->stride[2];
  p.vc_p = v_cache->stride[0]; p.vc_h = v_cache->stride[1]; p.vc_r = v_cache->stride[2];
  if (four) {
    p.k_params = k_params->data; p.v_params = v_params->data;
    p.kp_p = k_params->stride[0]; p.kp_h = k_params->stride[1]; p.kp_r = k_params->stride[2];
    p.vp_p = v_params->stride[0]; p.vp_h = v_params->stride[1]; p.vp_r = v_params->stride[2];
  }
  if (q != nullptr) {
    p.q = q->data; p.q_out = q_out->data;
    p.q_t = q->stride[0]; p.q_h = q->stride[1]; p.qo_t = q_out->stride[0]; p.qo_h = q_out->stride[1];
  }
  if (k_out != nullptr) { p.k_out = k_out->data; p.ko_t = k_out->stride[0]; p.ko_h = k_out->stride[1]; }
  if (v_out != nullptr) { p.v_out = v_out->data; p.vo_t = v_out->stride[0]; p.vo_h = v_out->stride[1]; }
  if (cos_table != nullptr) {
    p.cos_t = (const float *)cos_table->data; p.sin_t = (const float *)sin_table->data;
    p.cos_row = cos_table->stride[0]; p.sin_row = sin_table->stride[0];
  }
  p.table = (const int *)page_table->data; p.seq = (const int *)seq->data; p.pos = (const int *)pos->data;
  p.table_row = page_table->stride[0];
  p.T = (int)T; p.H = (int)H; p.HK = (int)HK; p.D = (int)D; p.R = (int)R;
  p.pages = (int)pages; p.width = (int)page_table->shape[1]; p.seqs = (int)page_table->shape[0];
  p.block = (int)block; p.angles = (int)angles; p.interleaved = interleaved != 0;
  p.status = device_status_word();
  if (p.status == nullptr) return fail(B200_RESOURCE, "no status word on this device");
  cudaStream_t s = (cudaStream_t)stream;
  if (dt == B200_DTYPE_FLOAT32) return four ? append::launch<float, true>(p, s) : append::launch<float, false>(p, s);
  if (dt == B200_DTYPE_FLOAT16) return four ? append::launch<__half, true>(p, s) : append::launch<__half, false>(p, s);
  return four ? append::launch<__nv_bfloat16, true>(p, s) : append::launch<__nv_bfloat16, false>(p, s);
}
