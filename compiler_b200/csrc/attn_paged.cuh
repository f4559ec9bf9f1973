// The paged attention's parameters, and its tensor-core kernel (one query type per source file).
#pragma once

#include "sm100.cuh"

#include <type_traits>

namespace b200 {
namespace paged {

constexpr int kMaxDim = 512;
constexpr unsigned kSiteLength = 52, kSitePage = 53;

struct Params {
  const void *q, *k_cache, *v_cache, *k_params, *v_params;
  void *out;
  float *lse;
  const int *table, *lengths, *cu;   // cu may be null
  int64_t q_t, q_h, o_t, o_h, l_t, l_h;
  int64_t kc_p, kc_h, kc_r, vc_p, vc_h, vc_r;
  int64_t kp_p, kp_h, kp_r, vp_p, vp_h, vp_r;
  int64_t table_row;
  int T, Z, H, HK, D, pages, width, block;
  int causal;
  float scale;
  unsigned int *status;
};

// Query tokens [begin, end) of sequence z, whatever cu_seqlens_q holds.
__device__ __forceinline__ void query_span(const Params &p, int z, int &begin, int &end) {
  if (p.cu == nullptr) {
    const int each = p.T / p.Z;
    begin = z * each;
    end = begin + each;
    return;
  }
  begin = min(max(p.cu[z], 0), p.T);
  end = min(max(p.cu[z + 1], begin), p.T);
}
// Keys of sequence z; a length outside its row of the page table is cut (and reported).
__device__ __forceinline__ int key_count(const Params &p, int z) {
  const int n = p.lengths[z];
  const int64_t room = (int64_t)p.width * p.block;
  if (n < 0 || (int64_t)n > room) {
    report_rejected(p.status, kSiteLength);
    return n < 0 ? 0 : (int)room;
  }
  return n;
}

// ------------------------------------------------------------------ tensor-core kernel
// Head sizes 64 and 128, 16-bit queries, 16-byte aligned cache rows, pages of a multiple of 16 keys.
//
// A decode step reads every cached key and value once and does a few dozen operations per byte, so
// the kernel is built around the reads: every warp takes tiles of 16 keys through a ring of its own in
// shared memory (cp.async, no barrier between warps) into mma.sync m16n8k16: with 8 or 16 query rows
// most of a tcgen05 tile would be padding.
//   S^T = K Q^T: keys are the instruction's 16 rows, query rows (the heads of a K / V group times
//   the new tokens) its 8 columns; lane (g, t) = (lane / 4, lane % 4) holds elements of keys g and
//   g + 8.  The sum over the head's elements may run in any order, so a lane takes 16 consecutive
//   bytes of a key row and Q is laid out to match.
//   O^T = V^T P^T: the head's elements are the rows, keys the contraction; V comes from shared memory
//   by transposing matrix loads, P goes from the accumulator's layout to the operand's by movmatrix.
//
// 4-bit rows are never turned into floating-point rows.  A code's four bits alone, read as fp16, are
// the subnormal code * 2^-24 (or code * 2^-20 in the next four), which the tensor core multiplies
// exactly -- a mask and no conversion per pair of codes -- and the scales act on the sums:
//   q . k_j = scale_j (q . c_j) + low_j sum(q)
//   sum_j p_j v_j = sum_j (p_j scale_j) c_j + sum_j p_j low_j
// q is scaled by a power of two to fill fp16's range (a bf16 value keeps all its bits down to 2^-28
// of the row's largest); p_j scale_j is rounded to fp16 (2^-11, the rounding any 16-bit attention
// gives its weights) after a power of two that the largest scale so far sets.
//
// The running maximum is lazy: the weights refer to a maximum that is raised only when a score
// passes it by 4 (in log2), so most tiles need one vote instead of shuffles.
//
// For values, bytes are the rows: a row of whole bytes sums c_even + 16 c_odd and one of masked bytes
// c_even, so the odd element is a sixteenth of the difference, taken once at the end.
//
// Work is dealt as in attn_decode.cu: the keys of all (sequence, K / V head, tile of query rows)
// items form one sequence of units of UNIT keys and every CTA takes an equal range of it, so one
// wave of CTAs carries any batch however ragged.  Ranges that begin or end inside an item leave
// softmax states in the workspace, and the CTA that brings the last piece of an item joins them, in the
// pieces' order (a second kernel for it, launched as a programmatic dependent, cost 7 us).  With few
// items a cluster of eight CTAs takes each and joins it over distributed shared memory, launch_mode().
//
// Measured, 32 query and 8 K / V heads of 128: 8 users x 131072 keys of 4 bits 147 us (5.6 TB/s; the
// copy rate would give 125), one user 6.8 us at 1000 16-bit keys, 9.9 at 4097 4-bit keys, 34 at 32000
// 16-bit keys; 64 ragged users of up to 4096 16-bit keys, 28 and 4 heads of 64, 41 us (4.5 TB/s; 28).
// The long ones wait for HBM, with 7 us at the end for marks and joins; the short ones are the latency
// of the chain page table, keys, softmax, join.  16 query rows over 4-bit keys are bound by arithmetic.
using sm100::cluster_arrive;
using sm100::cluster_wait;
using sm100::map_to_cta;

constexpr int TC_WARPS = 4;
constexpr int TC_THREADS = TC_WARPS * 32;
constexpr int kMaxCtas = 640;
constexpr int64_t kClusterKeys4 = 32768, kClusterKeys16 = 16384;  // see launch_mode()
// A CTA has at least so many units before another one takes part: a piece costs its states' way through
// the workspace.  Over ranges, with 4 / 8: one user of 500 4-bit keys 9.0 / 14.9 us, 16000 22.4 / 22.4,
// 32000 29.6 / 25.8, four users of 4000 18.7 / 19.7.
constexpr int kLeastUnits = 4;
constexpr int kMaxRows = 16;
constexpr float kLazy = 4.f;
constexpr float kNoMax = -1e30f;   // no key seen yet; far below any score, and still a number

// Shape of a warp's work: tiles of 16 keys per step, steps in its shared-memory ring (all but one of
// them in flight), CTAs per SM the registers are held to.  Some 40 KiB per SM are to be on their
// way at any time (6.6 TB/s x 0.9 us / 148); steps are 8704 bytes of 4-bit rows, 8192 of 16-bit ones
// (D = 128), so that 12 warps with one step in flight each have 100 KiB.
template <bool FOUR, int D, int NT> struct Shape {
  static constexpr int U = FOUR ? 2 : 1;
  static constexpr int UNIT = TC_WARPS * 16 * U;
  static constexpr int ROW = FOUR ? D / 2 : 2 * D;                 // bytes of a cached row
  static constexpr int TILE = 16 * (2 * ROW + (FOUR ? 8 : 0));     // K, V and both params of 16 keys
  static constexpr int STEP = U * TILE;
  static constexpr int CTAS = NT == 1 ? 3 : 2;
  static constexpr int STAGES = STEP >= 8192 ? (NT == 1 ? 2 : 3) : (NT == 1 ? 3 : 4);
  static constexpr int RING = TC_WARPS * STAGES * STEP;
  static constexpr int STATES = TC_WARPS * 8 * NT * (D + 2) * 4;   // the warps' states at the end of a segment
  // room for the states beside the ring: the next segment's copies can begin before they are joined
  static constexpr bool AHEAD = CTAS * (RING + STATES + 1024 + 128) <= 227 * 1024;
  static constexpr int SMEM = RING + (AHEAD ? STATES : 0);
  static_assert(STAGES * STEP >= 8 * NT * (D + 2) * 4, "the ring takes a warp's state at the end");
};

struct TcParams {
  Params p;
  float *states;               // [ctas][2][R (m), R (l), R x D]
  unsigned long long *flags;   // [ctas][2]: the launch whose state is in that slot, see all_there()
  unsigned long long launch;   // this launch's number, not 0
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
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
__device__ __forceinline__ float pow2i(int e) {  // 2^e, e clamped to the normal numbers
  return __uint_as_float((uint32_t)(min(max(e, -126), 127) + 127) << 23);
}
template <int BYTES> __device__ __forceinline__ void load_shared(uint32_t at, uint32_t *r) {
  if constexpr (BYTES == 16)
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
  else if constexpr (BYTES == 8)
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(at));
  else
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r[0]) : "r"(at));
}
__device__ __forceinline__ void load_matrices_transposed(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ float load_cluster(uint32_t at) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const uint8_t *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

// -- the sequence of units -----------------------------------------------------------------
// How a launch is dealt out.  kRanges: equal ranges of units.  kDense: the same with the rows of a page and
// head following each other without gaps (head-major pages), so that a tile's rows lie at constant
// distances.  kCluster: few items over short contexts -- a cluster of eight CTAs per item, each with
// an eighth of its keys, joined through distributed shared memory.
constexpr int kRanges = 0, kDense = 1, kCluster = 2, kClusterSize = 8;

struct Span {        // one sequence's share of the units
  int begin, count;  // its query tokens
  int length;        // its keys
  int row_tiles, key_units;
  int64_t units;
};
template <int R, int UNIT, int MODE> __device__ __forceinline__ Span span_of(const Params &p, int z) {
  Span s;
  int end;
  query_span(p, z, s.begin, end);
  s.count = end - s.begin;
  s.length = key_count(p, z);
  s.row_tiles = (int)(((int64_t)s.count * (p.H / p.HK) + R - 1) / R);
  s.key_units = max(1, (s.length + UNIT - 1) / UNIT);  // an empty sequence still writes its rows
  s.units = (int64_t)p.HK * s.row_tiles * (MODE == kCluster ? 1 : s.key_units);
  return s;
}
// A cut piece of an item, waiting in the workspace for the others.
struct Piece {
  int64_t item_u0;       // the item's first unit
  int key_units;         // and how many it has; 0: no such piece
  int kv, row0;          // its K / V head and first query row
  int begin, count;      // its sequence's query tokens
};
struct alignas(128) Deal {
  int64_t scratch[TC_WARPS];
  int64_t start;
  int found;
  Piece piece[2];        // by slot: what the range begins in the middle of, and what it ends in
  int joins[2];          // how many pieces this CTA joins into its item, mostly none
  int first[2];          // and the CTA of the first of them
};
// Sum of all sequences' units; every thread gets it.  
template <int R, int UNIT, int MODE> __device__ __forceinline__ int64_t total_units(const Params &p, Deal &d) {
  int64_t sum = 0;
  for (int z = threadIdx.x; z < p.Z; z += TC_THREADS) sum += span_of<R, UNIT, MODE>(p, z).units;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) d.scratch[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = 0;
#pragma unroll
  for (int w = 0; w < TC_WARPS; ++w) sum += d.scratch[w];
  __syncthreads();
  return sum;
}
// The block's units before this thread's, and all of them.
__device__ __forceinline__ int64_t scan_units(Deal &d, int64_t mine, int64_t &sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t other = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += other;
  }
  if (lane == 31) d.scratch[warp] = upto;
  __syncthreads();
  int64_t before = upto - mine;
  sum = 0;
#pragma unroll
  for (int w = 0; w < TC_WARPS; ++w) {
    if (w < warp) before += d.scratch[w];
    sum += d.scratch[w];
  }
  return before;
}
// The sequence that unit u belongs to, and its first unit.
template <int R, int UNIT, int MODE>
__device__ __forceinline__ int locate(const Params &p, Deal &d, int64_t u, int64_t &start) {
  int64_t base = 0;
  for (int z0 = 0; z0 < p.Z; z0 += TC_THREADS) {
    const int z = z0 + (int)threadIdx.x;
    const int64_t mine = z < p.Z ? span_of<R, UNIT, MODE>(p, z).units : 0;
    if (threadIdx.x == 0) d.found = -1;
    int64_t chunk;
    const int64_t before = base + scan_units(d, mine, chunk);
    if (mine > 0 && before <= u && u < before + mine) {
      d.found = z;
      d.start = before;
    }
    __syncthreads();
    const int found = d.found;
    start = d.start;
    __syncthreads();
    if (found >= 0) return found;
    base += chunk;
  }
  return p.Z;  // not reached for u < total
}

// a / b of non-negative numbers, in 32 bits where they fit (a 64-bit division takes a third of a microsecond)
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}
// the first unit of CTA c's range, and the CTA whose range holds unit u
__device__ __forceinline__ int64_t range_begin(int64_t c, int64_t units, int64_t ctas) { return quotient(c * units, ctas); }
__device__ __forceinline__ int64_t cta_of(int64_t u, int64_t units, int64_t ctas) { return quotient((u + 1) * ctas - 1, units); }

template <int R, int D> constexpr int state_floats() { return R * (D + 2); }

// -- finishing a row -------------------------------------------------------------------------
// Row r of a tile of sequence `s`: where it goes in out / lse.
struct RowPlace {
  int token, head;
};
__device__ __forceinline__ bool row_place(const Params &p, const Span &s, int kv, int row, RowPlace &at) {
  const int group = p.H / p.HK;
  if (row >= s.count * group) return false;
  at.token = s.begin + row / group;
  at.head = kv * group + row % group;
  return true;
}

// Elements d, d + 1 of a finished row; with element 0 its log-sum-exp.  No key seen: zeros and +inf.
template <typename T>
__device__ __forceinline__ void finish(const Params &p, const RowPlace &at, int d, float top, float sum, float2 v) {
  const bool empty = sum == 0.f;
  const float inv = empty ? 0.f : 1.f / sum;
  *reinterpret_cast<uint32_t *>((T *)p.out + at.token * p.o_t + at.head * p.o_h + d) =
      empty ? 0u : pack2<T>(v.x * inv, v.y * inv);
  if (d == 0 && p.lse != nullptr)
    p.lse[at.token * p.l_t + at.head * p.l_h] = empty ? INFINITY : top * 0.6931471805599453f + logf(sum);
}

// A CTA marks its pieces as written and then looks whether all of an item's are: the one that does so last
// finds all (of several that finish together the one that takes the first piece's mark: a quarter of
// the grid joined the same eight items else, 38 us against 34).  A slot's flag holds the number of the launch that
// wrote it, so whatever the workspace held before counts as not there and nothing has to be cleared
// first; who joins sets them back, so that the same launch can be replayed from a graph.  Marks and looks are separated by a fence on both sides, so of two
// CTAs at least one sees the other's mark -- and no counter is fought over (one word per item,
// counted up by compare-and-swap, cost 10 us for 16 pieces and 19 us for 33).
__device__ __forceinline__ void mark(unsigned long long *flag, unsigned long long launch) {
  *reinterpret_cast<volatile unsigned long long *>(flag) = launch;
}
template <typename FlagOf>
__device__ __forceinline__ bool all_there(unsigned long long launch, int pieces, FlagOf flag_of) {  // by one warp
  const int lane = threadIdx.x & 31;
  bool there = true;
  for (int i = lane; i < pieces; i += 32)
    there = there && *reinterpret_cast<volatile unsigned long long *>(flag_of(i)) == launch;
  if (!__all_sync(0xffffffffu, there)) return false;
  // of those that find all, the one that takes the first mark joins
  bool mine = false;
  if (lane == 0) mine = atomicExch(flag_of(0), 0ull) == launch;
  if (!__shfl_sync(0xffffffffu, mine, 0)) return false;
  __threadfence();  // the others' states, after their marks
  for (int i = lane; i < pieces; i += 32) mark(flag_of(i), 0ull);
  return true;
}

// The query rows of a tile from their pieces' states, in the order of the pieces; by the whole block, a warp
// per row.  The states come through shared memory, as many at a time as its BYTES hold: a trip to L2
// takes most of a microsecond, and with four of them under way per row in registers the 55 pieces of a
// single user's item took 15 of them (32000 16-bit keys: 50 us in all, 38 this way).
template <typename T, int R, int D, int BYTES, typename StateOf>
__device__ __forceinline__ void join_rows(const Params &p, const Span &s, int kv, int row0, int group, int pieces,
                                          float *room, StateOf state_of) {
  constexpr int PER = D / 32, ROWS = R / TC_WARPS;  // elements of a lane, rows of a warp
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rows = min(R, s.count * group - row0);
  const int each = 2 * R + rows * D;  // floats of a state in use
  const int fit = min(32, BYTES / (each * 4));
  const uint32_t room_at = (uint32_t)__cvta_generic_to_shared(room);
  float top[ROWS], sum[ROWS], acc[ROWS][PER];
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    top[k] = -INFINITY;
    sum[k] = 0.f;
#pragma unroll
    for (int e = 0; e < PER; ++e) acc[k][e] = 0.f;
  }
  for (int base = 0; base < pieces; base += fit) {
    const int count = min(fit, pieces - base);
    __syncthreads();  // whatever was there before is no longer read
    for (int j = warp; j < count; j += TC_WARPS) {
      const float *state = state_of(base + j);
      for (int c = lane; c < each / 4; c += 32) copy16(room_at + (j * each + c * 4) * 4, reinterpret_cast<const uint8_t *>(state + c * 4));
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      const int row = warp + k * TC_WARPS;
      if (row >= rows) break;
      const bool have = lane < count;  // a lane per piece
      const float m = have ? room[lane * each + row] : -INFINITY, l = have ? room[lane * each + R + row] : 0.f;
      const float high = fmaxf(top[k], warp_max(m));
      const float keep = top[k] == -INFINITY ? 0.f : ex2(top[k] - high);
      const float f = m == -INFINITY ? 0.f : ex2(m - high);
      float part = l * f;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
      sum[k] = sum[k] * keep + part;
      top[k] = high;
#pragma unroll
      for (int e = 0; e < PER; ++e) acc[k][e] *= keep;
#pragma unroll 8
      for (int j = 0; j < count; ++j) {
        const float fj = __shfl_sync(0xffffffffu, f, j);
        uint32_t x[PER];
        load_shared<PER * 4>(room_at + (j * each + 2 * R + row * D + lane * PER) * 4, x);
#pragma unroll
        for (int e = 0; e < PER; ++e) acc[k][e] = fmaf(fj, __uint_as_float(x[e]), acc[k][e]);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    RowPlace at;
    if (!row_place(p, s, kv, row0 + warp + k * TC_WARPS, at)) break;
#pragma unroll
    for (int e = 0; e < PER; e += 2)
      finish<T>(p, at, lane * PER + e, top[k], sum[k], make_float2(acc[k][e], acc[k][e + 1]));
  }
}

template <typename T, bool FOUR, int D, int NT, int MODE>
__global__ void __launch_bounds__(TC_THREADS, Shape<FOUR, D, NT>::CTAS)
attn_paged_tile_kernel(const __grid_constant__ TcParams tp) {
  using S = Shape<FOUR, D, NT>;
  constexpr int R = 8 * NT, UNIT = S::UNIT, U = S::U, ROW = S::ROW, STAGES = S::STAGES;
  // K: lane t of 4 reads ROW / 4 bytes of a key row
  constexpr int KW = ROW / 16;  // 32-bit words of K per lane and row
  constexpr int KSTEPS = D / 16, MTILES = D / 16;
  // [TC_WARPS][STAGES][U tiles]; at the end the warps' states.  Whole 128-byte lines: 16 bytes off (behind
  // 48 bytes of static shared memory) the copies took a seventh longer
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ Deal deal;
  const Params &p = tp.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int group = p.H / p.HK;

  constexpr bool CLUSTER = MODE == kCluster, DENSE = MODE == kDense;
  const int part = CLUSTER ? (int)(blockIdx.x % kClusterSize) : 0;  // which eighth of the keys
  int64_t ctas;  // that take part
  auto range = [&](int64_t units, int64_t &from, int64_t &to) {
    ctas = max((int64_t)1, min((int64_t)gridDim.x, quotient(units, kLeastUnits)));
    const int64_t c = min((int64_t)blockIdx.x, ctas);  // those behind have nothing to do
    from = CLUSTER ? blockIdx.x / kClusterSize : range_begin(c, units, ctas);
    to = CLUSTER ? min(from + 1, units) : range_begin(min(c + 1, ctas), units, ctas);
  };
  if (threadIdx.x == 0) deal.piece[0].key_units = deal.piece[1].key_units = 0;
  int64_t total, u0, u1, z_start;
  int z;
  if (p.Z <= TC_THREADS) {  // a thread per sequence: one scan gives the sum and the place in it
    const int64_t mine = (int)threadIdx.x < p.Z ? span_of<R, UNIT, MODE>(p, threadIdx.x).units : 0;
    const int64_t before = scan_units(deal, mine, total);
    range(total, u0, u1);
    if (u0 >= u1) return;
    if (mine > 0 && before <= u0 && u0 < before + mine) {
      deal.found = threadIdx.x;
      deal.start = before;
    }
    __syncthreads();
    z = deal.found;
    z_start = deal.start;
  } else {
    total = total_units<R, UNIT, MODE>(p, deal);
    range(total, u0, u1);
    if (u0 >= u1) return;
    z = locate<R, UNIT, MODE>(p, deal, u0, z_start);
  }

  // A segment: one item, and the units of it that are this CTA's.
  struct Segment {
    Span s;
    int64_t item_u0;
    int z, kv, row0, key0, key1, units;
    bool from_start, whole;
  } seg;
  seg.z = z;
  seg.s = span_of<R, UNIT, MODE>(p, z);
  auto enter = [&](int64_t u) {  // the segment that begins at unit u
    while (u >= z_start + seg.s.units) {  // the next sequence with anything to do
      z_start += seg.s.units;
      seg.s = span_of<R, UNIT, MODE>(p, ++seg.z);
    }
    const int item = CLUSTER ? (int)(u - z_start) : (int)quotient(u - z_start, seg.s.key_units);
    seg.item_u0 = z_start + (CLUSTER ? item : (int64_t)item * seg.s.key_units);
    const int unit0 = CLUSTER ? (int)((int64_t)seg.s.key_units * part / kClusterSize) : (int)(u - seg.item_u0);
    const int unit1 = CLUSTER ? (int)((int64_t)seg.s.key_units * (part + 1) / kClusterSize)
                              : (int)(min(u1, seg.item_u0 + seg.s.key_units) - seg.item_u0);
    seg.kv = item / seg.s.row_tiles;
    seg.row0 = (item % seg.s.row_tiles) * R;
    seg.key0 = unit0 * UNIT;
    // (with the causal mask, no further than the tile's last row sees)
    const int last_row = min(seg.row0 + R, seg.s.count * group) - 1;
    const int seen = p.causal ? max(0, min(seg.s.length, seg.s.length - seg.s.count + last_row / group + 1)) : seg.s.length;
    seg.key1 = min(seen, unit1 * UNIT);
    seg.units = unit1 - unit0;
    seg.from_start = unit0 == 0;
    seg.whole = seg.from_start && unit1 == seg.s.key_units;
  };

  // ---- this warp's tiles, 32 at a time: lane i holds where tile base + i lies (K and V have the same
  // strides, so one offset serves both); negative: no such tile, or no such page
  int64_t cache_now, params_now, cache_next, params_next;
  uint32_t live = 0;  // one bit per tile copied, the latest lowest
  auto lookup = [&](int n, int64_t &cache_at, int64_t &params_at) {
    const int key = seg.key0 + ((n / U) * TC_WARPS + warp) * (16 * U) + (n % U) * 16;
    cache_at = -1;
    params_at = 0;
    if (key < seg.key1) {
      const int index = key / p.block, row = key - index * p.block;
      const int page = __ldg(p.table + seg.z * p.table_row + index);
      if (page < 0 || page >= p.pages) {
        report_rejected(p.status, kSitePage);
      } else {
        cache_at = ((int64_t)page * p.kc_p + (int64_t)row * p.kc_r) * (FOUR ? 1 : 2);
        if constexpr (FOUR) params_at = ((int64_t)page * p.kp_p + (int64_t)row * p.kp_r) * 2;
      }
    }
  };

  // ---- copies: a warp fills its own ring, 16 bytes per lane and copy, row by row, with the chunks of a row
  // exchanged by the row's number so that no two rows of a read meet in a bank: K is read across rows
  // by 16-byte loads (only 16-bit rows, 128 bytes and more, need their halves swapped), V by
  // transposing matrix loads of eight rows.
  constexpr int ES = FOUR ? 1 : 2, CH = ROW / 16;  // chunks of a row
  const int64_t row_step = DENSE ? ROW : p.kc_r * ES;
  const int copy_row = lane / CH, copy_chunk = lane % CH;
  const uint8_t *k_src, *v_src, *par_src = nullptr;
  auto v_chunk = [](int chunk, int key) {  // where a chunk of V's row `key` lies
    return FOUR ? (CH == 4 ? chunk ^ ((key >> 1) & 3) : chunk ^ ((key >> 2) & 1)) : chunk ^ (key & 7);
  };
  const uint32_t my_ring = (uint32_t)__cvta_generic_to_shared(ring) + warp * (STAGES * S::STEP);
  auto copy_step = [&](int n, int stage) {  // n: first tile of a step (a multiple of U)
    if (n > 0 && (n & 31) == 0) {
      cache_now = cache_next;
      params_now = params_next;
      lookup(n + 32 + lane, cache_next, params_next);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t at = __shfl_sync(0xffffffffu, cache_now, (n + i) & 31);
      const int64_t par_at = FOUR ? __shfl_sync(0xffffffffu, params_now, (n + i) & 31) : 0;
      live = (live << 1) | (at >= 0 ? 1u : 0u);
      if (at >= 0) {
        const uint32_t k_dst = my_ring + stage * S::STEP + i * S::TILE, v_dst = k_dst + 16 * ROW;
        const uint8_t *ks = k_src + at, *vs = v_src + at;
#pragma unroll
        for (int c = 0; c < CH / 2; ++c) {
          const int key = c * (32 / CH) + copy_row;
          copy16(k_dst + key * ROW + (copy_chunk ^ (FOUR ? 0 : (key & 1) * 4)) * 16, ks + c * (32 / CH) * row_step);
          copy16(v_dst + key * ROW + v_chunk(copy_chunk, key) * 16, vs + c * (32 / CH) * row_step);
        }
        if constexpr (FOUR) copy4(v_dst + 16 * ROW + lane * 4, par_src + par_at);
      }
    }
  };
  auto first_copies = [&]() {  // of the segment that was entered
    k_src = (const uint8_t *)p.k_cache + seg.kv * p.kc_h * ES + copy_row * row_step + copy_chunk * 16;
    v_src = (const uint8_t *)p.v_cache + seg.kv * p.vc_h * ES + copy_row * row_step + copy_chunk * 16;
    if constexpr (FOUR)
      par_src = (lane < 16 ? (const uint8_t *)p.k_params + seg.kv * p.kp_h * 2
                           : (const uint8_t *)p.v_params + seg.kv * p.vp_h * 2) + (lane & 15) * (DENSE ? 4 : p.kp_r * 2);
    lookup(lane, cache_now, params_now);
    lookup(32 + lane, cache_next, params_next);
#pragma unroll
    for (int s0 = 0; s0 < STAGES - 1; ++s0) {
      copy_step(s0 * U, s0);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  };

  enter(u0);
  first_copies();
  for (int64_t u = u0;;) {
    const Span s = seg.s;
    const int kv = seg.kv, row0 = seg.row0, key0 = seg.key0, key1 = seg.key1;
    const int steps = key1 > key0 + warp * (16 * U) ? (key1 - key0 - warp * (16 * U) + UNIT - 1) / UNIT : 0;
    // ---- meanwhile the query rows of this item, in the layout of the B operand
    uint32_t qf[NT][KSTEPS][2];
    float score_mul[NT][2], low_mul[NT][2];   // of query columns 2t, 2t + 1
    int limit[NT][2];                          // keys they see
    // keys that every row of the tile sees
    const int least = p.causal ? max(0, min(s.length, s.length - s.count + row0 / group + 1)) : s.length;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = row0 + nt * 8 + g;
      RowPlace at;
      const bool have = row_place(p, s, kv, row, at);
      const uint32_t *src = have ? reinterpret_cast<const uint32_t *>((const T *)p.q + at.token * p.q_t + at.head * p.q_h) : nullptr;
      float mul = p.scale * 1.4426950408889634f, low = 0.f;
      if constexpr (FOUR) {
        // elements t * D/4 ..: words of 8 codes; a code word gives (0,4), (1,5) * 16, (2,6), (3,7) * 16
        float x[D / 4];
        float top = 0.f, sum = 0.f;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          const float2 v = have ? unpack2<T>(__ldg(src + t * (D / 8) + i)) : make_float2(0.f, 0.f);
          x[2 * i] = v.x;
          x[2 * i + 1] = v.y;
          top = fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
          sum += v.x + v.y;
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        // the largest element at 2^13 .. 2^14; a NaN row keeps its NaN
        const int e = top > 0.f ? 13 - ((int)(__float_as_uint(top) >> 23) - 127) : 0;
        const float up = pow2i(e), up16 = up * 0.0625f;
#pragma unroll
        for (int w = 0; w < KW; ++w) {
          qf[nt][2 * w][0] = pack2<__half>(x[8 * w] * up, x[8 * w + 4] * up);
          qf[nt][2 * w][1] = pack2<__half>(x[8 * w + 1] * up16, x[8 * w + 5] * up16);
          qf[nt][2 * w + 1][0] = pack2<__half>(x[8 * w + 2] * up, x[8 * w + 6] * up);
          qf[nt][2 * w + 1][1] = pack2<__half>(x[8 * w + 3] * up16, x[8 * w + 7] * up16);
        }
        low = mul * sum;
        mul = mul * 16777216.f / up;
      } else {
        // 16-byte vector j of lane t: elements 8 (4 j + t) ..
#pragma unroll
        for (int j = 0; j < KW / 4; ++j)
#pragma unroll
          for (int w = 0; w < 4; ++w)
            qf[nt][2 * j + w / 2][w % 2] = have ? __ldg(src + 4 * (4 * j + t) + w) : 0u;
      }
      int lim = 0;
      if (have) lim = p.causal ? max(0, min(s.length, s.length - s.count + (row / group) + 1)) : s.length;
#pragma unroll
      for (int c = 0; c < 2; ++c) {  // the lanes of query column 2t + c hold it as g = 2t + c
        const int from = 8 * t + 4 * c;
        score_mul[nt][c] = __shfl_sync(0xffffffffu, mul, from);
        low_mul[nt][c] = __shfl_sync(0xffffffffu, low, from);
        limit[nt][c] = __shfl_sync(0xffffffffu, lim, from);
      }
    }

    float o[NT][MTILES][4], m[NT][2];
    float2 l[NT], lows[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < MTILES; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.f;
      m[nt][0] = m[nt][1] = kNoMax;
      l[nt] = lows[nt] = make_float2(0.f, 0.f);
    }
    float inv_f = pow2i(100);  // 4 bits: weights * scales carry this power of two


    for (int step = 0, stage = 0; step < steps; ++step, stage = stage + 1 == STAGES ? 0 : stage + 1) {
      // the oldest step has arrived, and every lane is done with the slot of the one before it
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
      __syncwarp();
      copy_step((step + STAGES - 1) * U, stage == 0 ? STAGES - 1 : stage - 1);
      asm volatile("cp.async.commit_group;" ::: "memory");
      const uint32_t here = my_ring + stage * S::STEP;

      float sc[U][NT][4];
      int key[U];
      bool masked[U];
      uint32_t kpar[U][2], vpar[U][2];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        key[i] = key0 + (step * TC_WARPS + warp) * (16 * U) + i * 16;
        const bool absent = ((live >> ((STAGES - 1) * U + U - 1 - i)) & 1u) == 0;  // no such tile, or no such page
        masked[i] = absent || key[i] + 16 > least;  // some row does not see some key
        if (absent) key[i] = key1;
        uint32_t kr[2][KW];
        const uint32_t k_at = here + i * S::TILE, par_at = k_at + 32 * ROW + g * 4;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if constexpr (FOUR) {
            load_shared<KW * 4>(k_at + (g + 8 * h) * ROW + t * (KW * 4), kr[h]);
            load_shared<4>(par_at + h * 32, &kpar[i][h]);
            load_shared<4>(par_at + 64 + h * 32, &vpar[i][h]);
          } else {
#pragma unroll
            for (int j = 0; j < KW / 4; ++j)
              load_shared<16>(k_at + (g + 8 * h) * ROW + ((4 * j + t) ^ ((g & 1) * 4)) * 16, &kr[h][4 * j]);
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[i][nt][e] = 0.f;
        // ---- scores
        if constexpr (FOUR) {
#pragma unroll
          for (int w = 0; w < KW; ++w) {
            const uint32_t a = kr[0][w], b = kr[1][w], a8 = a >> 8, b8 = b >> 8;
            const uint32_t f0[4] = {a & 0x000f000fu, b & 0x000f000fu, a & 0x00f000f0u, b & 0x00f000f0u};
            const uint32_t f1[4] = {a8 & 0x000f000fu, b8 & 0x000f000fu, a8 & 0x00f000f0u, b8 & 0x00f000f0u};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma16816<__half>(sc[i][nt], f0, qf[nt][2 * w][0], qf[nt][2 * w][1]);
              mma16816<__half>(sc[i][nt], f1, qf[nt][2 * w + 1][0], qf[nt][2 * w + 1][1]);
            }
          }
        } else {
#pragma unroll
          for (int k = 0; k < KSTEPS; ++k) {
            const uint32_t f[4] = {kr[0][2 * k], kr[1][2 * k], kr[0][2 * k + 1], kr[1][2 * k + 1]};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816<T>(sc[i][nt], f, qf[nt][k][0], qf[nt][k][1]);
          }
        }
      }
      // ---- scores minus the running maximum, log2 domain: columns 2t, 2t + 1 as one pair
      uint32_t wf[U][NT][2];
      auto softmax = [&](auto any_masked) {
        constexpr bool MASKED = decltype(any_masked)::value;
        [[maybe_unused]] float2 k_par[U][2], v_par[U][2];
        if constexpr (FOUR) {
#pragma unroll
          for (int i = 0; i < U; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              k_par[i][h] = unpack2<T>(kpar[i][h]);
              v_par[i][h] = unpack2<T>(vpar[i][h]);
              // what stands behind the last key is nobody's: weights of 0 must meet numbers
              if (MASKED && key[i] + g + 8 * h >= key1) v_par[i][h] = make_float2(0.f, 0.f);
            }
        }
        float2 sx[U][NT][2];
        auto relative = [&](bool first) {
#pragma unroll
          for (int i = 0; i < U; ++i)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const float2 minus = make_float2(-m[nt][0], -m[nt][1]);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float2 raw = make_float2(sc[i][nt][2 * h], sc[i][nt][2 * h + 1]);
                const float2 mul = make_float2(score_mul[nt][0], score_mul[nt][1]);
                if constexpr (FOUR) {
                  const float2 low = make_float2(low_mul[nt][0], low_mul[nt][1]);
                  sx[i][nt][h] = fma2(raw, mul2(splat(k_par[i][h].x), mul),
                                      first ? mul2(splat(k_par[i][h].y), low) : fma2(splat(k_par[i][h].y), low, minus));
                } else {
                  sx[i][nt][h] = first ? mul2(raw, mul) : fma2(raw, mul, minus);
                }
                if constexpr (MASKED) {
                  const int j = key[i] + g + 8 * h;
                  if (j >= min(limit[nt][0], key1)) sx[i][nt][h].x = -INFINITY;
                  if (j >= min(limit[nt][1], key1)) sx[i][nt][h].y = -INFINITY;
                }
              }
            }
        };
        relative(false);
        float high = -INFINITY, high_scale = 0.f;
#pragma unroll
        for (int i = 0; i < U; ++i) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int h = 0; h < 2; ++h) high = fmaxf(high, fmaxf(sx[i][nt][h].x, sx[i][nt][h].y));
          if constexpr (FOUR) high_scale = fmaxf(high_scale, fmaxf(fabsf(v_par[i][0].x), fabsf(v_par[i][1].x)));
        }
        if (__any_sync(0xffffffffu, high > kLazy || (FOUR && high_scale * inv_f > 2048.f))) {
          float keep_f = 1.f;
          if constexpr (FOUR) {
            // the largest finite scale so far at 2^10 .. 2^11 (weights reach 2^4: products stay below 2^15)
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < U; ++i)
#pragma unroll
              for (int h = 0; h < 2; ++h)
                if (fabsf(v_par[i][h].x) < INFINITY) top = fmaxf(top, fabsf(v_par[i][h].x));
            top = warp_max(top);
            if (top * inv_f > 2048.f) {
              const float inv = pow2i(10 - max((int)(__float_as_uint(top) >> 23) - 127, -90));
              keep_f = inv / inv_f;
              inv_f = inv;
            }
          }
          relative(true);  // the scores themselves: next to a first maximum nothing would be left of them
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float keep[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float top = -INFINITY;
#pragma unroll
              for (int i = 0; i < U; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) top = fmaxf(top, c == 0 ? sx[i][nt][h].x : sx[i][nt][h].y);
#pragma unroll
              for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
              const float m_new = fmaxf(m[nt][c], top);
              keep[c] = ex2(m[nt][c] - m_new);
              m[nt][c] = m_new;
            }
            l[nt] = mul2(l[nt], make_float2(keep[0], keep[1]));
            lows[nt] = mul2(lows[nt], make_float2(keep[0], keep[1]));
#pragma unroll
            for (int i = 0; i < MTILES; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[nt][i][e] *= keep[e & 1] * keep_f;
          }
          relative(false);
        }
        // ---- weights and their sums; p_j scale_j and p_j low_j go where the codes' scale and low are
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float2 x = make_float2(ex2(sx[i][nt][h].x), ex2(sx[i][nt][h].y));
              l[nt] = add2(l[nt], x);
              float2 w = x;
              if constexpr (FOUR) {
                const float by = v_par[i][h].x * inv_f;
                w = mul2(x, splat(by));
                float2 low = fma2(x, splat(v_par[i][h].y), lows[nt]);
                if constexpr (MASKED) {
                  // a key that a row does not see adds nothing, whatever its scale and low are
                  if (sx[i][nt][h].x == -INFINITY) { w.x = 0.f; low.x = lows[nt].x; }
                  if (sx[i][nt][h].y == -INFINITY) { w.y = 0.f; low.y = lows[nt].y; }
                }
                lows[nt] = low;
              }
              wf[i][nt][h] = transpose8x8(pack2<typename std::conditional<FOUR, __half, T>::type>(w.x, w.y));
            }
      };
      bool any_masked = masked[0];
#pragma unroll
      for (int i = 1; i < U; ++i) any_masked = any_masked || masked[i];
      if (any_masked)  // the same for the whole warp
        softmax(std::true_type());
      else
        softmax(std::false_type());
      // ---- values.  A transposing load of eight key rows hands lane (g, t) the 16-bit columns g of keys
      // 2t and 2t + 1 in one register: neighbours of the contraction, as the operand wants them.
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const uint32_t v_at = here + i * S::TILE + 16 * ROW;
        const int key_in = lane & 7, matrix = lane >> 3;  // this lane's row of the four matrices
        if constexpr (FOUR) {
          const uint32_t row = v_at + (key_in + 8 * (matrix & 1)) * ROW;
#pragma unroll
          for (int c = 0; c < CH; c += 2) {
            uint32_t r[4];  // keys 0-7 and 8-15 of chunk c, then of chunk c + 1: four codes of two keys each
            load_matrices_transposed(row + v_chunk(c + (matrix >> 1), key_in) * 16, r);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              // rows of whole bytes and rows of their low codes: the high codes' sums are a sixteenth of
              // the difference, taken once at the end, and cost no mask of their own
              const uint32_t a = r[2 * h], b = r[2 * h + 1];
              const uint32_t a0 = a & 0x00ff00ffu, b0 = b & 0x00ff00ffu;
              const uint32_t a1 = __byte_perm(a, 0u, 0x4341), b1 = __byte_perm(b, 0u, 0x4341);
              const uint32_t f0[4] = {a0 & 0x000f000fu, a0, b0 & 0x000f000fu, b0};
              const uint32_t f1[4] = {a1 & 0x000f000fu, a1, b1 & 0x000f000fu, b1};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma16816<__half>(o[nt][2 * (c + h)], f0, wf[i][nt][0], wf[i][nt][1]);
                mma16816<__half>(o[nt][2 * (c + h) + 1], f1, wf[i][nt][0], wf[i][nt][1]);
              }
            }
          }
        } else {
          const uint32_t row = v_at + (key_in + 8 * (matrix >> 1)) * ROW;
          // registers 0, 1: keys 2t, 2t + 1 of the tile; 2, 3: keys 8 + those.  Keep the keys below `upto`.
          auto keep_keys = [&](uint32_t (&r)[4], int upto) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int j = key[i] + 2 * t + 8 * (e >> 1);
              if (j >= upto) r[e] = 0u;
              else if (j + 1 >= upto) r[e] &= 0xffffu;
            }
          };
          uint32_t vr[MTILES][4];
#pragma unroll
          for (int w = 0; w < MTILES; ++w)
            load_matrices_transposed(row + v_chunk(2 * w + (matrix & 1), key_in) * 16, vr[w]);
          // values behind the last key may be anything: a weight of 0 does not silence a NaN
          bool odd = false;
          if (masked[i]) {
            const uint32_t top = std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
#pragma unroll
            for (int w = 0; w < MTILES; ++w) {
              keep_keys(vr[w], key1);
#pragma unroll
              for (int e = 0; e < 4; ++e) odd = odd || (vr[w][e] & top) == top || ((vr[w][e] >> 16) & top) == top;
            }
            odd = __any_sync(0xffffffffu, odd);
          }
          if (!odd) {
#pragma unroll
            for (int w = 0; w < MTILES; ++w)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma16816<T>(o[nt][w], vr[w], wf[i][nt][0], wf[i][nt][1]);
          } else {
            // infinities or NaN among keys that some rows see and others do not: one pass per number
            // of keys seen, with the keys behind at zero, kept by the rows that see that many
            const int end = min(key1, key[i] + 16);
            for (int seen = max(least, key[i]); seen <= end; ++seen) {
#pragma unroll
              for (int w = 0; w < MTILES; ++w) {
                uint32_t r[4] = {vr[w][0], vr[w][1], vr[w][2], vr[w][3]};
                keep_keys(r, seen);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                  float part[4] = {0.f, 0.f, 0.f, 0.f};
                  mma16816<T>(part, r, wf[i][nt][0], wf[i][nt][1]);
#pragma unroll
                  for (int e = 0; e < 4; ++e)
                    if (min(limit[nt][e & 1], end) == seen) o[nt][w][e] += part[e];
                }
              }
            }
          }
        }
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();
    // the next segment's first keys are on their way while this one is put together
    const bool from_start = seg.from_start, whole = seg.whole;
    const int64_t item_u0 = seg.item_u0;
    u += CLUSTER ? 1 : seg.units;
    const bool more = !CLUSTER && u < u1;
    if (more) {
      enter(u);
      if constexpr (S::AHEAD) first_copies();
    }

    // ---- the warps' states to shared memory
    constexpr int STATE = S::AHEAD ? state_floats<R, D>() * 4 : STAGES * S::STEP;  // from one warp's to the next
    uint8_t *states = S::AHEAD ? ring + S::RING : ring;
    float *mine = reinterpret_cast<float *>(states + warp * STATE);
    const float unit = 16777216.f / inv_f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float sum = c == 0 ? l[nt].x : l[nt].y, low = c == 0 ? lows[nt].x : lows[nt].y;
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          sum += __shfl_xor_sync(0xffffffffu, sum, x);
          if constexpr (FOUR) low += __shfl_xor_sync(0xffffffffu, low, x);
        }
        const int row = nt * 8 + 2 * t + c;
        if (g == 0) {
          mine[row] = m[nt][c] == kNoMax ? -INFINITY : m[nt][c];
          mine[R + row] = sum;
        }
#pragma unroll
        for (int i = 0; i < MTILES; ++i) {
          const float a = o[nt][i][c], b = o[nt][i][c + 2];
          float *to = mine + 2 * R + row * D;
          if constexpr (FOUR) {  // the second row summed the first element's codes + 16 times the second's
            const int d = 32 * (i / 2) + 4 * g + 2 * (i % 2);
            *reinterpret_cast<float2 *>(to + d) = make_float2(fmaf(a, unit, low), fmaf(b - a, unit * 0.0625f, low));
          } else {
            to[16 * i + g] = a;
            to[16 * i + 8 + g] = b;
          }
        }
      }
    }
    __syncthreads();
    // ---- and together; a whole item's are the result, a cut one's go to the workspace (a cluster's: to
    // this CTA's shared memory)
    float *slot = CLUSTER ? reinterpret_cast<float *>(ring + S::SMEM)
                          : tp.states + ((int64_t)blockIdx.x * 2 + (from_start ? 1 : 0)) * state_floats<R, D>();
    for (int i = threadIdx.x; i < R * (D / 2); i += TC_THREADS) {
      const int row = i / (D / 2), d = (i % (D / 2)) * 2;
      RowPlace at;
      if (!row_place(p, s, kv, row0 + row, at)) break;  // the rows behind it are not there either
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < TC_WARPS; ++w) top = fmaxf(top, reinterpret_cast<const float *>(states + w * STATE)[row]);
      float sum = 0.f;
      float2 v = make_float2(0.f, 0.f);
#pragma unroll
      for (int w = 0; w < TC_WARPS; ++w) {
        const float *from = reinterpret_cast<const float *>(states + w * STATE);
        const float f = from[row] == -INFINITY ? 0.f : ex2(from[row] - top);
        const float2 x = *reinterpret_cast<const float2 *>(from + 2 * R + row * D + d);
        sum += f * from[R + row];
        v.x += f * x.x;
        v.y += f * x.y;
      }
      if (!CLUSTER && whole) {
        finish<T>(p, at, d, top, sum, v);
      } else {
        *reinterpret_cast<float2 *>(slot + 2 * R + row * D + d) = v;
        if (d == 0) {
          slot[row] = top;
          slot[R + row] = sum;
        }
      }
    }
    if constexpr (CLUSTER) {
      cluster_arrive();
      cluster_wait();
      // row r is finished by CTA r % 8, which reads its state from all eight
      const uint32_t state = (uint32_t)__cvta_generic_to_shared(slot);
      for (int i = threadIdx.x; i < R / kClusterSize * (D / 2); i += TC_THREADS) {
        const int row = part + i / (D / 2) * kClusterSize, d = (i % (D / 2)) * 2;
        RowPlace at;
        if (!row_place(p, s, kv, row0 + row, at)) break;
        float tops[kClusterSize], top = -INFINITY, sum = 0.f;
        float2 v = make_float2(0.f, 0.f);
#pragma unroll
        for (int c = 0; c < kClusterSize; ++c) {
          tops[c] = load_cluster(map_to_cta(state, c) + row * 4);
          top = fmaxf(top, tops[c]);
        }
#pragma unroll
        for (int c = 0; c < kClusterSize; ++c) {
          const uint32_t from = map_to_cta(state, c);
          const float f = tops[c] == -INFINITY ? 0.f : ex2(tops[c] - top);
          sum += f * load_cluster(from + (R + row) * 4);
          v.x += f * load_cluster(from + (2 * R + row * D + d) * 4);
          v.y += f * load_cluster(from + (2 * R + row * D + d + 1) * 4);
        }
        finish<T>(p, at, d, top, sum, v);
      }
      cluster_arrive();  // the other CTAs read this one's state until they arrive
      cluster_wait();
    } else if (!whole && threadIdx.x == 0) {
      deal.piece[from_start ? 1 : 0] = Piece{item_u0, s.key_units, kv, row0, s.begin, s.count};
    }
    if (!more) break;
    __syncthreads();  // the next segment's states go to the same place
    if constexpr (!S::AHEAD) first_copies();
  }

  if constexpr (!CLUSTER) {
    // The CTA that brings the last piece of an item joins them all.  Both pieces of this CTA are marked
    // at its end, behind one pair of fences (marking the first when it is done held the CTA up for
    // the fences' microseconds in between, and the others are no earlier).
    __syncthreads();
    // one warp looks after each piece
    const Piece c = deal.piece[warp & 1];
    const bool cut = warp < 2 && c.key_units > 0;
    const int first = cut ? (int)cta_of(c.item_u0, total, ctas) : 0;
    const int pieces = cut ? (int)cta_of(c.item_u0 + c.key_units - 1, total, ctas) - first + 1 : 0;
    // the first piece is the second slot of its CTA (its range ends in it), the others first slots
    auto slot_of = [&](int from, int i) { return (from + i) * 2 + (i == 0 ? 1 : 0); };
    if (threadIdx.x == 0 && (deal.piece[0].key_units | deal.piece[1].key_units) != 0) {
      __threadfence();  // this CTA's states, before its marks
      for (int i = 0; i < 2; ++i)
        if (deal.piece[i].key_units > 0) mark(tp.flags + blockIdx.x * 2 + i, tp.launch);
      __threadfence();
    }
    __syncthreads();
    if (warp < 2) {
      const bool all = cut && all_there(tp.launch, pieces, [&](int j) { return tp.flags + slot_of(first, j); });
      if (lane == 0) {
        deal.joins[warp] = all ? pieces : 0;
        deal.first[warp] = first;
      }
    }
    __syncthreads();
    for (int i = 0; i < 2; ++i) {
      if (deal.joins[i] == 0) continue;
      const int from = deal.first[i];
      Span s = {};
      s.begin = deal.piece[i].begin;
      s.count = deal.piece[i].count;
      join_rows<T, R, D, S::RING>(p, s, deal.piece[i].kv, deal.piece[i].row0, group, deal.joins[i],
                                  reinterpret_cast<float *>(ring),
                                  [&](int j) { return tp.states + slot_of(from, j) * state_floats<R, D>(); });
    }
  }
}

// Numbers launches for all_there(): one process never gives a number twice.
unsigned long long next_launch();

template <typename T, bool FOUR, int D, int NT, int MODE>
static int launch_tiles(const Params &p, int64_t items, void *workspace, cudaStream_t stream) {
  constexpr int R = 8 * NT;
  constexpr int smem = Shape<FOUR, D, NT>::SMEM + (MODE == kCluster ? state_floats<R, D>() * (int)sizeof(float) : 0);
  static_assert(R <= kMaxRows, "the workspace is sized for kMaxRows");
  auto kernel = attn_paged_tile_kernel<T, FOUR, D, NT, MODE>;
  static int resident[64] = {0};
  int dev = 0;
  B200_CUDA_OK(cudaGetDevice(&dev));
  if (dev >= 64) return fail(B200_RESOURCE, "device index %d out of range", dev);
  if (resident[dev] == 0) {
    int per_sm = 0;
    B200_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    B200_CUDA_OK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, TC_THREADS, smem));
    if (per_sm < 1) return fail(B200_RESOURCE, "the paged attention kernel does not fit on an SM");
    resident[dev] = per_sm;
  }
  TcParams tp;
  tp.p = p;
  tp.flags = (unsigned long long *)workspace;
  tp.states = (float *)((uint8_t *)workspace + kMaxCtas * 2 * sizeof(unsigned long long));
  tp.launch = next_launch();
  if (MODE == kCluster) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(items * kClusterSize));
    cfg.blockDim = dim3(TC_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kClusterSize;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    B200_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, tp));
    return B200_OK;
  }
  const int ctas = resident[dev] * sm_count() < kMaxCtas ? resident[dev] * sm_count() : kMaxCtas;
  kernel<<<ctas, TC_THREADS, smem, stream>>>(tp);
  B200_CUDA_OK(cudaGetLastError());
  return B200_OK;
}

template <typename T, bool FOUR, int D, int NT> static int launch_mode(const Params &p, void *workspace, cudaStream_t stream) {
  // no batch of T tokens in Z sequences has more items than this
  const int64_t items = ((int64_t)p.T * (p.H / p.HK) / (8 * NT) + p.Z) * p.HK;
  // Clusters while all of them are resident and a CTA's eighth of the longest context the table has
  // room for stays short.  One user, 8 K / V heads, clusters against ranges: 500 4-bit keys 7.2 and
  // 9.2 us, 16000 16.9 and 21.9, 32000 27.0 and 29.5, 64000 47 and 35; 500 16-bit keys 6.3 and 11.1,
  // 16000 22.5 and 24.8, 32000 54 and 34.
  if (items * kClusterSize <= 2 * sm_count() && (int64_t)p.width * p.block <= (FOUR ? kClusterKeys4 : kClusterKeys16))
    return launch_tiles<T, FOUR, D, NT, kCluster>(p, items, workspace, stream);
  if constexpr (FOUR)
    if (p.kc_r == D / 2 && p.kp_r == 2) return launch_tiles<T, FOUR, D, NT, kDense>(p, items, workspace, stream);
  return launch_tiles<T, FOUR, D, NT, kRanges>(p, items, workspace, stream);
}

template <typename T, bool FOUR, int D> static int launch_rows_of(const Params &p, void *workspace, cudaStream_t stream) {
  // Tiles of 8 query rows, or of 16 when a sequence has many on average: the keys are then read and
  // unpacked once for both, but fewer warps fit.  48 sequences of 8192 keys, tiles of 8 against 16: 16-bit
  // keys, 16 rows 220 and 166 us, 32 rows 384 and 248; 4-bit keys, whose reads count less, 16 rows 92 and
  // 98, 24 rows 117 and 124, 32 rows 145 and 139.
  const int64_t rows = ((int64_t)p.T + p.Z - 1) / p.Z * (p.H / p.HK);
  return rows > (FOUR ? 24 : 8) ? launch_mode<T, FOUR, D, 2>(p, workspace, stream) : launch_mode<T, FOUR, D, 1>(p, workspace, stream);
}

// Defined for one query type per source file (attn_paged_bf16.cu, attn_paged_f16.cu).
template <typename T> int launch_tensor_core(const Params &p, bool four, void *workspace, cudaStream_t stream);

#define B200_PAGED_TENSOR_CORE(T)                                                                    \
  namespace b200 {                                                                                   \
  namespace paged {                                                                                  \
  template <>                                                                                        \
  int launch_tensor_core<T>(const Params &p, bool four, void *workspace, cudaStream_t stream) {      \
    if (p.D == 128)                                                                                  \
      return four ? launch_rows_of<T, true, 128>(p, workspace, stream)                               \
                  : launch_rows_of<T, false, 128>(p, workspace, stream);                             \
    return four ? launch_rows_of<T, true, 64>(p, workspace, stream)                                  \
                : launch_rows_of<T, false, 64>(p, workspace, stream);                                \
  }                                                                                                  \
  }                                                                                                  \
  }

}  // namespace paged
}  // namespace b200
