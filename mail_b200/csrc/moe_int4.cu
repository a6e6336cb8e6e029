// Experts with 4-bit weights (int4.cuh has the format): quantising and reading
// back, products grouped by expert for few rows an expert, and the C entry
// points of the 4-bit operators.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "int4.cuh"
#include "rows.cuh"
#include "scan.cuh"

namespace moe {
namespace {

using u4::Act;

// ---------------------------------------------------------------------------
// Quantising with group scales.
//   s = T(absmax / 7)  (fp32 quotient, then the scales' type)
//   q = clamp(rint(w / s), -8, 7) + 8, 8 where s is 0
// GROUP / 16 lanes share a group; a lane loads sixteen weights and stores their
// eight bytes. The rounding is that of the exact quotient, half to even. For
// 16-bit weights the correctly rounded fp32 quotient (a reciprocal for the
// group, then one correction by the exact remainder) is enough: a quotient of
// two such numbers that is not on a border is further from it than fp32's
// rounding. For fp32 weights the remainder w - i s (one fma; exact) tells
// whether a neighbour of i is nearer or, on the border, even.
// A group with a NaN or an infinity, or whose scale is too large for its type,
// gets a NaN scale and q = 8, so what it stands for shows as NaN.
//
// Both directions stream: 32768 x 14336 bf16 in groups of 32, there and back,
// takes 414 us, 5.8 TB/s of the 2.4 GB moved (467 with eight weights a lane).
// A division for each weight bound the quantiser by its instructions, about 30
// a weight (806 us).

// Sixteen weights as loaded, their largest magnitude (infinity or NaN if one
// is), and eight of them as fp32. The bits of magnitudes are in the order of the
// numbers, with infinity and NaN on top.
template <typename T>
struct Sixteen {
  uint4 raw[2];
  __device__ __forceinline__ void load(const T* p) {
    raw[0] = *reinterpret_cast<const uint4*>(p);
    raw[1] = *reinterpret_cast<const uint4*>(p + 8);
  }
  __device__ __forceinline__ void zero() { raw[0] = raw[1] = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ float amax() const {
    constexpr uint32_t kAbs = 0x7fff7fffu;
    uint32_t m = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      m = __vmaxu2(m, __vmaxu2(__vmaxu2(raw[h].x & kAbs, raw[h].y & kAbs), __vmaxu2(raw[h].z & kAbs, raw[h].w & kAbs)));
    const uint16_t top = (uint16_t)max(m & 0xffffu, m >> 16);
    return Act<T>::to_float(*reinterpret_cast<const T*>(&top));
  }
  __device__ __forceinline__ void floats(int half, float (&v)[8]) const {
    rows::load8(reinterpret_cast<const T*>(&raw[half]), v);
  }
};
template <>
struct Sixteen<float> {
  float f[2][8];
  __device__ __forceinline__ void load(const float* p) {
    rows::load8(p, f[0]);
    rows::load8(p + 8, f[1]);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int j = 0; j < 16; ++j) f[j / 8][j % 8] = 0.f;
  }
  __device__ __forceinline__ float amax() const {
    int bits = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) bits = max(bits, __float_as_int(f[j / 8][j % 8]) & 0x7fffffff);
    return __int_as_float(bits);
  }
  __device__ __forceinline__ void floats(int half, float (&v)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = f[half][j];
  }
};

// The eight steps of one word, s > 0 and its reciprocal given.
template <bool EXACT_QUOTIENT>
__device__ __forceinline__ uint32_t quant_word(const float (&v)[8], float s, float inv) {
  constexpr float kRound = 12582912.f;  // 1.5 * 2^23: adding it rounds to a whole number
  uint32_t word = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float t;  // kRound + the step
    if constexpr (EXACT_QUOTIENT) {
      const float quot = v[j] * inv;
      t = fmaf(fmaf(-quot, s, v[j]), inv, quot) + kRound;
    } else {
      t = fmaf(v[j], inv, kRound);
      const float rest = fmaf(kRound - t, s, v[j]);
      const float past = fmaf(2.f, fabsf(rest), -s);  // > 0: beyond half a step, 0: on the border
      if (past > 0.f || (past == 0.f && (__float_as_int(t) & 1))) t += rest > 0.f ? 1.f : -1.f;
    }
    word += (uint32_t)__float_as_int(t) << (4 * j);
  }
  // the bits of kRound out of every place, 8 into it: a step is in -8 .. 7
  constexpr uint32_t kBits = 0x4b400000u;
  constexpr uint32_t kOut = kBits * 0x11111111u;
  return word - kOut + 0x88888888u;
}

template <typename Tw, typename Ts, int GROUP>
__global__ void __launch_bounds__(256) quant_groups_kernel(const Tw* __restrict__ src, int64_t n16,
                                                           uint2* __restrict__ dst, Ts* __restrict__ scale) {
  pdl_begin();
  constexpr int kLanes = GROUP / 16;
  constexpr int kVec = sizeof(Tw) == 2 ? 2 : 1;             // vectors of sixteen in flight
  const int64_t stride = (int64_t)gridDim.x * blockDim.x;   // a multiple of kLanes: a group's lanes stay together
  const int64_t last = (n16 + 31) / 32 * 32;                // whole warps take part in the shuffles
  for (int64_t base = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; base < last; base += kVec * stride) {
    Sixteen<Tw> in[kVec];
#pragma unroll
    for (int u = 0; u < kVec; ++u) {
      const int64_t i = base + u * stride;
      if (i < n16) in[u].load(src + i * 16);
      else in[u].zero();
    }
#pragma unroll
    for (int u = 0; u < kVec; ++u) {
      const int64_t i = base + u * stride;
      if (i >= last) break;  // the same for the whole warp
      int bits = __float_as_int(in[u].amax());
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
      Ts st = Act<Ts>::from_float(__fdiv_rn(__int_as_float(bits), 7.0f));
      float s = Act<Ts>::to_float(st);
      uint2 words = make_uint2(0x88888888u, 0x88888888u);
      if (!isfinite(s)) {
        st = Act<Ts>::from_float(NAN);
      } else if (s > 0.f) {
        float v[2][8];
        in[u].floats(0, v[0]);
        in[u].floats(1, v[1]);
        if (s < 6.2e-5f) {
          // a scale that may be subnormal: it can be well below absmax / 7, so
          // the steps are clamped, and its reciprocal may overflow
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j / 8][j % 8] = fminf(fmaxf(v[j / 8][j % 8], -8.f * s), 7.f * s) * 0x1p64f;
          s *= 0x1p64f;
        }
        const float inv = __frcp_rn(s);
        words.x = quant_word<sizeof(Tw) == 2>(v[0], s, inv);
        words.y = quant_word<sizeof(Tw) == 2>(v[1], s, inv);
      }
      if (i < n16) {
        dst[i] = words;
        if (i % kLanes == 0) scale[i / kLanes] = st;
      }
    }
  }
}

template <typename Ts, typename To, int GROUP>
__global__ void __launch_bounds__(256) dequant_groups_kernel(const uint32_t* __restrict__ src,
                                                             const Ts* __restrict__ scale, int64_t n8,
                                                             To* __restrict__ dst) {
  pdl_begin();
  constexpr int kVec = 4;
  const int64_t stride = (int64_t)gridDim.x * blockDim.x;
  for (int64_t base = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; base < n8; base += kVec * stride) {
    uint32_t w[kVec];
    float s[kVec];
#pragma unroll
    for (int u = 0; u < kVec; ++u) {
      const int64_t i = base + u * stride;
      w[u] = i < n8 ? src[i] : 0u;
      s[u] = i < n8 ? Act<Ts>::to_float(scale[i / (GROUP / 8)]) : 0.f;
    }
#pragma unroll
    for (int u = 0; u < kVec; ++u) {
      const int64_t i = base + u * stride;
      if (i >= n8) break;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)  // 2^23 + q, exactly
        v[j] = (__int_as_float((int)((w[u] >> (4 * j)) & 15u) | 0x4b000000) - 8388616.f) * s[u];
      rows::store8(dst + i * 8, v);
    }
  }
}

// ---------------------------------------------------------------------------
// Products grouped by expert, few rows an expert:
//   out[r, n] = sum_k x[r, k] W[e(r), n, k]
// SWIGLU: W holds I gate rows and I up rows and out[r, n] = silu(g) u.
//
// A warp works on strips of 32 weight rows of an expert, two mma tiles (m16n8k16:
// sixteen weight rows by eight of the expert's rows). The grid is persistent:
// each CTA first lists the experts that have rows, then its groups of `wk` warps
// take strips in turn, each warp of a group a share of K; the shares are added
// through shared memory in the order of the warps, so results do not depend on
// timing. With SWIGLU a tile's sixteen rows are eight gate rows and the eight up
// rows that go with them. (A CTA for each strip and possible expert, most of
// which leave at once, took 93 us for two rows of 4096 over eight experts of
// 28672 rows.)
//
// A lane (row g = lane / 4, t = lane % 4) holds GROUP / 4 consecutive k of its
// weight rows at a time, so that the four lanes of a row cover exactly one
// group of scales: the products of a group are summed from whole numbers, which
// 16-bit types hold exactly, and the fp32 sum is scaled once, which rounds no
// weight. The numbers are M + q (int4.cuh); the mma tile of the offsets -(M + 8)
// with the same activations comes first and serves both weight tiles, so no
// weight is corrected by itself. The terms of the two cancel to at most 136 / 8
// of their size (bf16; 72 / 8 in fp16), which costs the fp32 sums five bits of
// the eight (fp16: eight) that they have to spare over a 24-bit significand
// against the output's.
//
// What bounds it is the latency of decoding beside the mma chain with the 16
// warps an SM that the registers leave: two rows of 4096 through eight experts
// of 28672 rows take 43 us, 2.8 TB/s, ALU 42 % and DRAM 32 % busy (the same
// loads without products run at 6.5 TB/s). One tile a warp with 24 warps: 52 us,
// with 32: 59.
constexpr int kMvThreads = 256;
constexpr int kMvWarps = kMvThreads / 32;
constexpr int kMaxExperts = 1024;
constexpr int kMaxSlots = 1024;  // routed slots of the form that reads top-k ids
constexpr int kDownSlots = 256;  // and of the fused down projection

struct MvParams {
  const void* x;         // [.., K]
  const uint8_t* w;      // [E, w_rows, K / 2]
  const void* scale;     // [E, w_rows, K / group]
  void* out;             // [rows, n_out]
  int64_t K;
  int n_out, w_rows;     // output features; weight rows of an expert (2 n_out with SWIGLU)
  int E;
  int out_f32;           // out is fp32, else the activations' type
  // rows: either the top-k ids of `slots` slots (row r of x is slot / x_div, row
  // of out is the slot), or counts of consecutive rows
  const int32_t* ids;
  int slots;
  const void* counts;
  int counts_is64;
  int64_t total_rows;    // rows of out; those that no expert has are zeroed
  const int32_t* row_map;  // counts form: row r reads x row row_map[r] / x_div (NULL: r)
  int x_div;
};

// A block of 128 k of a lane's weight rows: rows g and g + 8 of MT tiles.
template <typename T, int GROUP, int MT>
struct Block4 {
  static constexpr int kWords = GROUP / 32;  // 32-bit words a lane holds of a row and group
  static constexpr int kPer = 128 / GROUP;   // groups in the block
  static constexpr int kRows = 2 * MT;
  static constexpr int kBytes = 512 * kRows;  // of a warp in shared memory
  uint32_t q[kRows][4];
  T s[kRows][kPer];
};

// Copies this lane's words of a block to its own 16 bytes for each row in
// shared memory, asynchronously. Nobody else reads them, so waiting for the
// copies is all the synchronisation there is. Groups past the end are left out:
// any words will do, their scales and activations are zero.
template <int GROUP, int R>
__device__ __forceinline__ void copy_words(uint32_t dst, const uint8_t* const (&w)[R], int b, int groups) {
  constexpr int kPer = 128 / GROUP, kBytes = 16 / kPer;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int g = b * kPer + j;
    if (GROUP == 128 || g < groups) {
      const int at = g * (GROUP / 2);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if constexpr (GROUP == 128)
          asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst + r * 512), "l"(w[r] + at)
                       : "memory");
        else
          asm volatile("cp.async.ca.shared.global.L2::128B [%0], [%1], %2;" ::"r"(dst + r * 512 + j * kBytes),
                       "l"(w[r] + at), "n"(kBytes)
                       : "memory");
      }
    }
  }
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void read_words(uint32_t src, uint32_t (&v)[4]) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(src)
               : "memory");
}

// The scales of a block; 0 for groups past the end.
template <typename T, int GROUP, int MT>
__device__ __forceinline__ void load_scales(Block4<T, GROUP, MT>& k, const T* const (&sc)[2 * MT], int b, int groups) {
  using B = Block4<T, GROUP, MT>;
#pragma unroll
  for (int j = 0; j < B::kPer; ++j) {
    const int g = b * B::kPer + j;
#pragma unroll
    for (int r = 0; r < B::kRows; ++r) k.s[r][j] = GROUP == 128 || g < groups ? __ldg(sc[r] + g) : Act<T>::from_float(0.f);
  }
}

// The activations of eight rows for the block: this lane's row, its words' k.
// Lanes without a row read the last one's: their columns are not used.
template <typename T, int GROUP>
__device__ __forceinline__ void load_acts(uint4 (&v)[4], const T* x, int b, int groups) {
  using B = Block4<T, GROUP, 1>;
#pragma unroll
  for (int j = 0; j < B::kPer; ++j)
#pragma unroll
    for (int i = 0; i < B::kWords; ++i) {
      const int g = b * B::kPer + j;
      v[j * B::kWords + i] = GROUP == 128 || g < groups ? __ldg(reinterpret_cast<const uint4*>(x + g * GROUP + i * 8))
                                                        : make_uint4(0, 0, 0, 0);
    }
}

// acc += the block's products, in units of kUnit: MT tiles of sixteen weight rows
// by 8 NT tokens.
template <typename T, int GROUP, int MT, int NT>
__device__ __forceinline__ void multiply_block(float (&acc)[MT][NT][4], const Block4<T, GROUP, MT>& k,
                                               const uint4 (&x)[NT][4], const u4::Exponents& ex) {
  using B = Block4<T, GROUP, MT>;
  constexpr uint32_t off_lo[4] = {Act<T>::kOffset[0], Act<T>::kOffset[0], Act<T>::kOffset[1], Act<T>::kOffset[1]};
  constexpr uint32_t off_hi[4] = {Act<T>::kOffset[2], Act<T>::kOffset[2], Act<T>::kOffset[3], Act<T>::kOffset[3]};
#pragma unroll
  for (int j = 0; j < B::kPer; ++j) {
    uint32_t bx[B::kWords][NT][4];
    float base[NT][4];
#pragma unroll
    for (int i = 0; i < B::kWords; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        u4::pair_up(x[n][j * B::kWords + i], bx[i][n]);
        if (i == 0) Act<T>::mma_first(base[n], off_lo, bx[i][n][0], bx[i][n][1]);
        else Act<T>::mma(base[n], off_lo, bx[i][n][0], bx[i][n][1]);
        Act<T>::mma(base[n], off_hi, bx[i][n][2], bx[i][n][3]);
      }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float part[NT][4];
#pragma unroll
      for (int i = 0; i < B::kWords; ++i) {
        uint32_t a0[4], a1[4];
        Act<T>::decode(k.q[2 * m][j * B::kWords + i], ex, a0);
        Act<T>::decode(k.q[2 * m + 1][j * B::kWords + i], ex, a1);
        const uint32_t lo[4] = {a0[0], a1[0], a0[1], a1[1]}, hi[4] = {a0[2], a1[2], a0[3], a1[3]};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (i == 0) Act<T>::mma_first(part[n], lo, bx[i][n][0], bx[i][n][1]);
          else Act<T>::mma(part[n], lo, bx[i][n][0], bx[i][n][1]);
          Act<T>::mma(part[n], hi, bx[i][n][2], bx[i][n][3]);
        }
      }
      const float s0 = Act<T>::to_float(k.s[2 * m][j]), s1 = Act<T>::to_float(k.s[2 * m + 1][j]);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        acc[m][n][0] = fmaf(s0, part[n][0] + base[n][0], acc[m][n][0]);
        acc[m][n][1] = fmaf(s0, part[n][1] + base[n][1], acc[m][n][1]);
        acc[m][n][2] = fmaf(s1, part[n][2] + base[n][2], acc[m][n][2]);
        acc[m][n][3] = fmaf(s1, part[n][3] + base[n][3], acc[m][n][3]);
      }
    }
  }
}

// The experts that have rows, in order: expert, first place in the list of
// rows, number of rows. Rows in counts form are the places themselves; in ids
// form s.list holds the slots expert by expert: with IN_ORDER those of an expert
// in order, the same for every CTA and in every run; else as the warps arrive,
// which is enough where a row's values do not depend on its place.
struct RowLists {
  int expert[kMaxExperts], first[kMaxExperts], rows[kMaxExperts];
  int list[kMaxSlots];
  int total;   // rows in all
  int active;  // experts listed
};

// Inclusive sum over the lanes of a warp.
__device__ __forceinline__ int warp_inclusive(int v) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, v, o);
    if ((int)(threadIdx.x & 31) >= o) v += n;
  }
  return v;
}

// seen [kMaxExperts], IN_ORDER only: shared memory that is free until the
// return. It holds, for each expert, how many of its slots each of the eight
// warps has, a byte for a warp.
template <bool IN_ORDER>
__device__ __forceinline__ void list_rows(RowLists& s, const MvParams& p, uint2* seen) {
  __shared__ int64_t warp_sums[32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (p.ids && p.slots <= 32) {
    // a slot for each lane of one warp: experts in the order of their first slots
    if (tid < 32) {
      const int id = tid < p.slots ? p.ids[tid] : -1;
      const bool live = id >= 0 && id < p.E;
      const unsigned mates = __match_any_sync(0xffffffffu, live ? id : -1);
      const unsigned below = (1u << tid) - 1;
      const bool leads = live && (mates & below) == 0;
      const unsigned leaders = __ballot_sync(0xffffffffu, leads);
      const int rows = leads ? __popc(mates) : 0;
      const int incl = warp_inclusive(rows);
      const int first = __shfl_sync(0xffffffffu, incl - rows, __ffs(mates) - 1);
      if (leads) {
        const int a = __popc(leaders & below);
        s.expert[a] = id;
        s.first[a] = first;
        s.rows[a] = rows;
      }
      if (live) s.list[first + __popc(mates & below)] = tid;
      if (tid == 31) {
        s.total = incl;
        s.active = __popc(leaders);
      }
    }
    __syncthreads();
    return;
  }
  const int per = (p.E + kMvThreads - 1) / kMvThreads;
  const int lo = min(p.E, tid * per), hi = min(p.E, lo + per);
  if (tid == 0) s.active = 0;
  // IN_ORDER: thread t takes slot t. Its place among its expert's slots is the
  // number of them before it: in its warp here, and in the warps below. (In
  // order for up to 1024 slots, four a thread: 218 us for the layer of 128 experts
  // at 128 tokens, 211 this way.)
  static_assert(kDownSlots <= kMvThreads && kMvWarps == 8, "a slot a thread, a byte of seen for each warp");
  int id = -1, before = 0;
  if (p.ids) {
    for (int e = tid; e < p.E; e += kMvThreads) {
      if constexpr (IN_ORDER) seen[e] = make_uint2(0, 0);
      else s.rows[e] = 0;
    }
    __syncthreads();
    if constexpr (IN_ORDER) {
      if (tid < p.slots) id = p.ids[tid];
      if (id < 0 || id >= p.E) id = -1;
      const unsigned mates = __match_any_sync(0xffffffffu, id);
      before = __popc(mates & ((1u << lane) - 1));
      if (id >= 0 && before == 0) reinterpret_cast<uint8_t*>(&seen[id])[warp] = (uint8_t)__popc(mates);
    } else {
      for (int i = tid; i < p.slots; i += kMvThreads) {
        const int e = p.ids[i];
        if (e >= 0 && e < p.E) atomicAdd(&s.rows[e], 1);
      }
    }
    __syncthreads();
  }
  int cnt[kMaxExperts / kMvThreads];
  int64_t mine = 0;  // rows << 11 | experts that have some
#pragma unroll
  for (int i = 0; i < kMaxExperts / kMvThreads; ++i) {
    cnt[i] = 0;
    if (lo + i < hi) {
      if (p.ids) {
        if constexpr (IN_ORDER) {
          const uint2 v = seen[lo + i];
          cnt[i] = (int)__dp4a(v.x, 0x01010101u, __dp4a(v.y, 0x01010101u, 0u));
        } else {
          cnt[i] = s.rows[lo + i];
        }
      } else {
        const int64_t c = p.counts_is64 ? static_cast<const int64_t*>(p.counts)[lo + i]
                                        : (int64_t) static_cast<const int32_t*>(p.counts)[lo + i];
        cnt[i] = (int)max((int64_t)0, min(c, p.total_rows));
      }
      mine += ((int64_t)cnt[i] << 11) + (cnt[i] > 0);
    }
  }
  const int64_t incl = block_inclusive_scan<int64_t>(mine, warp_sums);  // ends with a barrier: rows[] may be reused
  const int64_t limit = p.ids ? (int64_t)p.slots : p.total_rows;
  int64_t run = (incl - mine) >> 11;
  int a = (int)((incl - mine) & 2047);
#pragma unroll
  for (int i = 0; i < kMaxExperts / kMvThreads; ++i) {
    if (cnt[i] > 0) {
      if (run < limit) {  // counts past the last row are cut off, and experts behind it not listed
        s.expert[a] = lo + i;
        s.first[a] = (int)run;
        s.rows[a] = (int)min((int64_t)cnt[i], limit - run);
        atomicMax(&s.active, a + 1);
      }
      ++a;
      run += cnt[i];
    }
  }
  if (tid == kMvThreads - 1) s.total = (int)min(incl >> 11, limit);
  __syncthreads();
  if (p.ids) {
    auto listed = [&](int e) {  // place of expert e among those listed
      int l = 0, h = s.active - 1;
      while (l < h) {
        const int m = (l + h) >> 1;
        if (s.expert[m] < e) l = m + 1;
        else h = m;
      }
      return l;
    };
    if constexpr (IN_ORDER) {
      if (id >= 0) {
        const uint2 v = seen[id];  // the bytes of the warps below are added
        const uint32_t lo4 = warp < 4 ? (1u << (8 * warp)) - 1 : 0xffffffffu;
        const uint32_t hi4 = warp < 4 ? 0u : (1u << (8 * (warp - 4))) - 1;
        before += (int)__dp4a(v.x & lo4, 0x01010101u, __dp4a(v.y & hi4, 0x01010101u, 0u));
        s.list[s.first[listed(id)] + before] = tid;
      }
    } else {  // its expert's first, then one after the other
      for (int i = tid; i < p.slots; i += kMvThreads) {
        const int e = p.ids[i];
        if (e >= 0 && e < p.E) s.list[atomicAdd(&s.first[listed(e)], 1)] = i;
      }
      __syncthreads();
      for (int i = tid; i < s.active; i += kMvThreads) s.first[i] -= s.rows[i];
    }
    __syncthreads();
  }
}

__device__ __forceinline__ void group_barrier(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Blocks of 128 k whose words a warp has in flight.
constexpr int kRowsDeep = 4;
// Weight tiles of a warp and CTAs of an SM.
constexpr int kRowsTiles = 2;
constexpr int kRowsCtas = 2;

// A place in a warp's run of work: the unit (an expert's strip), the chunk of
// the expert's rows, the block of K.
struct RowsWork {
  int64_t unit;
  int c0, b;
};

template <typename T, int GROUP, int NT, bool SWIGLU>
__global__ void __launch_bounds__(kMvThreads, kRowsCtas) int4_rows_kernel(const MvParams p) {
  pdl_begin();
  constexpr int kWords = GROUP / 32;      // 32-bit words a lane loads of a row and group
  constexpr int kTokens = 8 * NT;
  constexpr int MT = kRowsTiles;
  constexpr int kFeat = (SWIGLU ? 8 : 16) * MT;  // output features of a strip
  using B = Block4<T, GROUP, MT>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

  extern __shared__ __align__(16) uint8_t s_words[];
  __shared__ RowLists s;
  __shared__ float s_red[kMvWarps][16 * MT][kTokens + 1];
  list_rows<false>(s, p, nullptr);

  const int strips = (p.n_out + kFeat - 1) / kFeat;
  const int blocks = (int)((p.K + 127) / 128);
  const int64_t units = (int64_t)s.active * strips;
  // warps that share a strip along K: the number that leaves the longest run of
  // blocks of any warp shortest, at two blocks' worth for each strip's end
  int wk = 1;
  int64_t best = INT64_MAX;
#pragma unroll 1
  for (int w = 1; w <= kMvWarps && w <= blocks; w *= 2) {
    const int64_t teams = (int64_t)gridDim.x * (kMvWarps / w);
    const int64_t cost = (units + teams - 1) / teams * ((blocks + w - 1) / w + 2);
    if (cost < best) {
      best = cost;
      wk = w;
    }
  }
  const int groups_in_cta = kMvWarps / wk, group = warp / wk, share = warp % wk;
  const int b0 = (int)((int64_t)blocks * share / wk), b1 = (int)((int64_t)blocks * (share + 1) / wk);
  const int kgroups = (int)(p.K / GROUP);
  const T* x = static_cast<const T*>(p.x);
  const int64_t stride = (int64_t)gridDim.x * groups_in_cta;
  // rows of W of this lane: rows g and g + 8 of both tiles (rows past the end
  // read the last row and are not stored)
  auto weight_row = [&](int64_t unit, int r) -> int64_t {
    const int e = s.expert[unit / strips], strip = (int)(unit % strips);
    int row;
    if (SWIGLU) row = min(strip * kFeat + (r >> 1) * 8 + g, p.n_out - 1) + (r & 1) * p.n_out;
    else row = min(strip * kFeat + r * 8 + g, p.n_out - 1);
    return (int64_t)e * p.w_rows + row;
  };
  auto next = [&](RowsWork& w) -> bool {  // the next block; true: of another unit
    if (++w.b < b1) return false;
    w.b = b0;
    w.c0 += kTokens;
    if (w.c0 < s.rows[w.unit / strips]) return false;
    w.c0 = 0;
    w.unit += stride;
    return true;
  };

  // neighbouring units on different CTAs: a small launch spreads over the SMs
  const RowsWork start{(int64_t)group * gridDim.x + blockIdx.x, 0, b0};
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(s_words) + warp * kRowsDeep * B::kBytes + lane * 16;
  RowsWork in = start;  // of the block copied next
  const uint8_t* w[2 * MT] = {};
  bool moved = true;
  auto copy_next = [&](int slot) {
    if (in.unit < units) {
      if (moved) {
#pragma unroll
        for (int r = 0; r < 2 * MT; ++r) w[r] = p.w + weight_row(in.unit, r) * (p.K / 2) + t * 4 * kWords;
      }
      copy_words<GROUP, 2 * MT>(ring + slot * B::kBytes, w, in.b, kgroups);
      moved = next(in);
    }
    copy_commit();
  };
#pragma unroll 1
  for (int i = 0; i < kRowsDeep - 1; ++i) copy_next(i);
  const u4::Exponents ex = Act<T>::exponents();
  int slot = 0;
  for (int64_t unit = start.unit; unit < units; unit += stride) {
    const int a = (int)(unit / strips), strip = (int)(unit % strips);
    const int first = s.first[a], cnt = s.rows[a];
    const T* sc[2 * MT];
#pragma unroll
    for (int r = 0; r < 2 * MT; ++r) sc[r] = static_cast<const T*>(p.scale) + weight_row(unit, r) * kgroups;
    for (int c0 = 0; c0 < cnt; c0 += kTokens) {
      float acc[MT][NT][4];
      const T* xp[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < 4 * MT; ++i) acc[i / 4][n][i % 4] = 0.f;
        const int place = first + min(c0 + n * 8 + g, cnt - 1);
        const int row = p.ids ? s.list[place] / p.x_div : (p.row_map ? p.row_map[place] / p.x_div : place);
        xp[n] = x + (int64_t)row * p.K + t * 8 * kWords;
      }
#pragma unroll 1
      for (int b = b0; b < b1; ++b) {
        B k;
        uint4 xv[NT][4];
        load_scales<T, GROUP, MT>(k, sc, b, kgroups);
#pragma unroll
        for (int n = 0; n < NT; ++n) load_acts<T, GROUP>(xv[n], xp[n], b, kgroups);
        // the slot freed by the last block takes the block kRowsDeep - 1 ahead
        copy_next(slot == 0 ? kRowsDeep - 1 : slot - 1);
        copy_wait<kRowsDeep - 1>();
#pragma unroll
        for (int r = 0; r < 2 * MT; ++r) read_words(ring + slot * B::kBytes + r * 512, k.q[r]);
        multiply_block<T, GROUP, MT, NT>(acc, k, xv, ex);
        slot = slot + 1 == kRowsDeep ? 0 : slot + 1;
      }
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) s_red[warp][m * 16 + (i >> 1) * 8 + g][n * 8 + 2 * t + (i & 1)] = acc[m][n][i];
      group_barrier(1 + group, 32 * wk);
      // feature f, token n: the shares added in order
      const int tokens = min(kTokens, cnt - c0);
      for (int i = share * 32 + lane; i < kFeat * tokens; i += 32 * wk) {
        const int f = i % kFeat, n = i / kFeat;
        const int feat = strip * kFeat + f;
        if (feat >= p.n_out) continue;
        float v = 0.f, u = 0.f;
        const int at_row = SWIGLU ? (f & 8) * 2 + (f & 7) : f;
        for (int k = 0; k < wk; ++k) {
          v += s_red[group * wk + k][at_row][n];
          if (SWIGLU) u += s_red[group * wk + k][at_row + 8][n];
        }
        v *= Act<T>::kUnit;
        if (SWIGLU) v = u4::silu_mul(v, u * Act<T>::kUnit);
        const int place = first + c0 + n;
        const int64_t at = (int64_t)(p.ids ? s.list[place] : place) * p.n_out + feat;
        if (p.out_f32) static_cast<float*>(p.out)[at] = v;
        else static_cast<T*>(p.out)[at] = Act<T>::from_float(v);
      }
      group_barrier(1 + group, 32 * wk);
    }
  }
  copy_wait<0>();
  if (!p.ids) {  // rows behind the last expert's are zero
    const int64_t n0 = (int64_t)s.total * p.n_out, n1 = p.total_rows * p.n_out;
    for (int64_t i = n0 + (int64_t)blockIdx.x * kMvThreads + threadIdx.x; i < n1;
         i += (int64_t)gridDim.x * kMvThreads) {
      if (p.out_f32) static_cast<float*>(p.out)[i] = 0.f;
      else static_cast<uint16_t*>(p.out)[i] = 0;
    }
  }
}

// ---------------------------------------------------------------------------
// The down projection and the combine of a decode batch in one launch:
//   y[t, c] = sum_j weight[t, j] sum_k h[slot (t, j), k] W2[id(t, j), c, k]
//
// A cluster of CTAs takes a strip of sixteen output features and every expert
// that has rows; its warps share the blocks of all experts' rows evenly and add
// their tiles, times the routing weights, to sums of their own for each token.
// Those are added over the warps of a CTA, then over the CTAs of the cluster
// through distributed shared memory, always in the same order, and rounded
// once: no buffer of rows and no third launch. All CTAs of a cluster have to cut
// the same tiles from the lists, so these are in order (list_rows). The lists and the
// first words do not depend on h, so they are read before the wait for the
// gate_up launch (which itself has waited for whatever wrote ids and weights).
constexpr int kDownTokens = 32;
constexpr int kDownDeep = 6;

struct DownParams {
  const void* h;         // [slots, K]
  const uint8_t* w;      // [E, n_out, K / 2]
  const void* scale;
  const float* weights;  // [slots]
  const int32_t* ids;    // [slots]
  void* y;               // [tokens, n_out]
  int64_t K;
  int n_out, E, tokens, top_k, slots, cluster;
};

template <typename T, int GROUP>
__global__ void __launch_bounds__(kMvThreads, 2) int4_down_kernel(const DownParams p) {
  constexpr int kWords = GROUP / 32;
  using B = Block4<T, GROUP, 1>;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  extern __shared__ __align__(16) uint8_t s_words[];
  __shared__ RowLists s;
  __shared__ int s_tile_expert[kDownSlots], s_tile_first[kDownSlots], s_tile_rows[kDownSlots], s_tiles;
  __shared__ __align__(16) float s_sum[kMvWarps][kDownTokens][17];
  static_assert(sizeof(s_sum) >= kMaxExperts * sizeof(uint2), "list_rows needs it for a while");

  MvParams lists{};
  lists.ids = p.ids;
  lists.slots = p.slots;
  lists.E = p.E;
  list_rows<true>(s, lists, reinterpret_cast<uint2*>(s_sum));
  if (warp == 0) {  // tiles of up to eight rows of an expert
    int tiles = 0;
    for (int a0 = 0; a0 < s.active; a0 += 32) {
      const int a = a0 + lane;
      const int rows = a < s.active ? s.rows[a] : 0;
      const int mine = (rows + 7) / 8;
      const int incl = warp_inclusive(mine);
      for (int i = 0; i < mine; ++i) {
        const int at = tiles + incl - mine + i;
        s_tile_expert[at] = s.expert[a];
        s_tile_first[at] = s.first[a] + 8 * i;
        s_tile_rows[at] = min(8, rows - 8 * i);
      }
      tiles += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) s_tiles = tiles;
  }
  for (int i = lane; i < p.tokens * 17; i += 32) s_sum[warp][i / 17][i % 17] = 0.f;
  __syncthreads();

  const int rank = blockIdx.x % p.cluster, strip = blockIdx.x / p.cluster;
  const int blocks = (int)((p.K + 127) / 128), kgroups = (int)(p.K / GROUP);
  const int64_t work = (int64_t)s_tiles * blocks;
  const int me = rank * kMvWarps + warp, all = p.cluster * kMvWarps;
  const int64_t lo = work * me / all, hi = work * (me + 1) / all;
  const int r0 = min(strip * 16 + g, p.n_out - 1), r1 = min(strip * 16 + g + 8, p.n_out - 1);

  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(s_words) + warp * kDownDeep * B::kBytes + lane * 16;
  int64_t in = lo;
  int in_tile = (int)(lo / blocks), in_b = (int)(lo % blocks);
  const uint8_t* w[2] = {};
  bool moved = true;
  auto copy_next = [&](int slot) {
    if (in < hi) {
      if (moved) {
        const int64_t base = (int64_t)s_tile_expert[in_tile] * p.n_out;
        w[0] = p.w + (base + r0) * (p.K / 2) + t * 4 * kWords;
        w[1] = p.w + (base + r1) * (p.K / 2) + t * 4 * kWords;
      }
      copy_words<GROUP, 2>(ring + slot * B::kBytes, w, in_b, kgroups);
      ++in;
      moved = ++in_b == blocks;
      if (moved) {
        in_b = 0;
        ++in_tile;
      }
    }
    copy_commit();
  };
#pragma unroll 1
  for (int i = 0; i < kDownDeep - 1; ++i) copy_next(i);
  pdl_begin();  // h

  const u4::Exponents ex = Act<T>::exponents();
  int slot = 0;
  int64_t at = lo;
  int tile = (int)(lo / blocks), b = (int)(lo % blocks);
  while (at < hi) {
    const int64_t base = (int64_t)s_tile_expert[tile] * p.n_out;
    const T* sc[2] = {static_cast<const T*>(p.scale) + (base + r0) * kgroups,
                      static_cast<const T*>(p.scale) + (base + r1) * kgroups};
    const int rows = s_tile_rows[tile], first = s_tile_first[tile];
    const T* xp = static_cast<const T*>(p.h) + (int64_t)s.list[first + min(g, rows - 1)] * p.K + t * 8 * kWords;
    const int end = (int)min((int64_t)blocks, b + (hi - at));
    float acc[1][1][4] = {};
    at += end - b;
#pragma unroll 1
    for (; b < end; ++b) {
      B k;
      uint4 xv[1][4];
      load_scales<T, GROUP, 1>(k, sc, b, kgroups);
      load_acts<T, GROUP>(xv[0], xp, b, kgroups);
      copy_next(slot == 0 ? kDownDeep - 1 : slot - 1);
      copy_wait<kDownDeep - 1>();
      read_words(ring + slot * B::kBytes, k.q[0]);
      read_words(ring + slot * B::kBytes + 512, k.q[1]);
      multiply_block<T, GROUP, 1, 1>(acc, k, xv, ex);
      slot = slot + 1 == kDownDeep ? 0 : slot + 1;
    }
    // column by column: two rows of a tile may belong to one token
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      if (n < rows && t == n / 2) {
        const int sl = s.list[first + n];
        const float weight = p.weights[sl];
        float* sum = s_sum[warp][sl / p.top_k];
        sum[g] = fmaf(weight, acc[0][0][n & 1], sum[g]);
        sum[g + 8] = fmaf(weight, acc[0][0][2 + (n & 1)], sum[g + 8]);
      }
      __syncwarp();
    }
    b = 0;
    ++tile;
  }
  copy_wait<0>();
  __syncthreads();
  // this CTA's sums, into the first warp's place
  for (int i = tid; i < p.tokens * 16; i += kMvThreads) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < kMvWarps; ++k) v += s_sum[k][i >> 4][i & 15];
    s_sum[0][i >> 4][i & 15] = v;
  }
  cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  cluster.sync();
  if (rank == 0) {
    for (int i = tid; i < p.tokens * 16; i += kMvThreads) {
      const int tok = i >> 4, f = i & 15;
      float v = s_sum[0][tok][f];
      for (int c = 1; c < p.cluster; ++c) v += *cluster.map_shared_rank(&s_sum[0][tok][f], c);
      if (strip * 16 + f < p.n_out)
        static_cast<T*>(p.y)[(int64_t)tok * p.n_out + strip * 16 + f] = Act<T>::from_float(v * Act<T>::kUnit);
    }
  }
  cluster.sync();  // no CTA leaves while its sums are read
}

// y[t] = sum_j weight[t, j] * o[row of slot (t, j)], slots in order; a slot
// whose id names no expert adds nothing. slot_row NULL: the row is the slot.
template <typename T>
__global__ void __launch_bounds__(256) int4_combine_kernel(const float* __restrict__ o,
                                                           const int32_t* __restrict__ ids,
                                                           const int32_t* __restrict__ slot_row,
                                                           const float* __restrict__ weight, int64_t T8, int64_t H8,
                                                           int k, int E, T* __restrict__ y) {
  pdl_begin();
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < T8; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t t = i / H8, c = i % H8 * 8;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int j = 0; j < k; ++j) {
      const int64_t s = t * k + j;
      const int id = ids[s];
      if (id < 0 || id >= E) continue;
      const int64_t row = slot_row ? (int64_t)slot_row[s] : s;
      const float w = weight[s];
      float v[8];
      rows::load8(o + row * H8 * 8 + c, v);
#pragma unroll
      for (int q = 0; q < 8; ++q) acc[q] = fmaf(w, v[q], acc[q]);
    }
    rows::store8(y + t * H8 * 8 + c, acc);
  }
}

// ---------------------------------------------------------------- host side
bool act_ok(int dtype) { return dtype == MOE_BF16 || dtype == MOE_F16; }

unsigned flat_grid(int64_t threads) {
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>(ceil_div(threads, 256), (int64_t)num_sms() * 16));
}

template <typename Tw, typename Ts>
int launch_quant(const void* src, int64_t n16, int group, void* dst, void* scale, cudaStream_t st) {
#define MOE_QUANT(G)                                                                                      \
  MOE_CUDA_TRY(launch_kernel(quant_groups_kernel<Tw, Ts, G>, dim3(flat_grid(n16)), dim3(256), 0, st,       \
                             static_cast<const Tw*>(src), n16, static_cast<uint2*>(dst), static_cast<Ts*>(scale)))
  if (group == 128) MOE_QUANT(128);
  else if (group == 64) MOE_QUANT(64);
  else MOE_QUANT(32);
#undef MOE_QUANT
  MOE_LAUNCH_CHECK("quant_groups_kernel");
  return MOE_OK;
}

template <typename Ts, typename To>
int launch_dequant(const void* src, const void* scale, int64_t n8, int group, void* dst, cudaStream_t st) {
#define MOE_DEQUANT(G)                                                                                     \
  MOE_CUDA_TRY(launch_kernel(dequant_groups_kernel<Ts, To, G>, dim3(flat_grid(n8)), dim3(256), 0, st,      \
                             static_cast<const uint32_t*>(src), static_cast<const Ts*>(scale), n8, static_cast<To*>(dst)))
  if (group == 128) MOE_DEQUANT(128);
  else if (group == 64) MOE_DEQUANT(64);
  else MOE_DEQUANT(32);
#undef MOE_DEQUANT
  MOE_LAUNCH_CHECK("dequant_groups_kernel");
  return MOE_OK;
}

template <typename T, int GROUP, int NT, bool SWIGLU>
int launch_rows_nt(MvParams p, int64_t rows, cudaStream_t st) {
  constexpr int kSmem = kMvWarps * kRowsDeep * Block4<T, GROUP, kRowsTiles>::kBytes;
  const int64_t units = ceil_div(p.n_out, (SWIGLU ? 8 : 16) * kRowsTiles) * std::min<int64_t>(p.E, rows);
  const int64_t ctas = std::min<int64_t>(units * ceil_div(p.K, 1024), kRowsCtas * num_sms());
  auto kfn = int4_rows_kernel<T, GROUP, NT, SWIGLU>;
  MOE_TRY((allow_smem<int4_rows_kernel<T, GROUP, NT, SWIGLU>>(kSmem)));
  MOE_CUDA_TRY(launch_kernel(kfn, dim3((unsigned)ctas), dim3(kMvThreads), kSmem, st, p));
  MOE_LAUNCH_CHECK("int4_rows_kernel");
  return MOE_OK;
}

template <typename T, int GROUP, bool SWIGLU>
int launch_rows_group(const MvParams& p, int64_t rows, cudaStream_t st) {
  if (rows <= 8 || rows <= 2 * (int64_t)p.E) return launch_rows_nt<T, GROUP, 1, SWIGLU>(p, rows, st);
  return launch_rows_nt<T, GROUP, 2, SWIGLU>(p, rows, st);
}

template <typename T, int GROUP>
int launch_down(DownParams p, cudaStream_t st) {
  // CTAs of a cluster: as many (1, 2, 4 or 8) as two a SM leave room for
  const int strips = (int)ceil_div(p.n_out, 16);
  p.cluster = 1;
  while (p.cluster < 8 && 2 * p.cluster * strips <= 2 * num_sms()) p.cluster *= 2;
  auto kfn = int4_down_kernel<T, GROUP>;
  const int smem = kMvWarps * kDownDeep * Block4<T, GROUP, 1>::kBytes;
  MOE_TRY((allow_smem<int4_down_kernel<T, GROUP>>(smem)));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3((unsigned)(strips * p.cluster));
  cfg.blockDim = dim3(kMvThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.numAttrs = 1;
  if (pdl_enabled()) {
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 2;
  }
  MOE_CUDA_TRY(cudaLaunchKernelEx(&cfg, kfn, p));
  MOE_LAUNCH_CHECK("int4_down_kernel");
  return MOE_OK;
}

int launch_down_any(const DownParams& p, int dtype, int group, cudaStream_t st) {
  if (dtype == MOE_BF16) {
    if (group == 128) return launch_down<__nv_bfloat16, 128>(p, st);
    if (group == 64) return launch_down<__nv_bfloat16, 64>(p, st);
    return launch_down<__nv_bfloat16, 32>(p, st);
  }
  if (group == 128) return launch_down<__half, 128>(p, st);
  if (group == 64) return launch_down<__half, 64>(p, st);
  return launch_down<__half, 32>(p, st);
}

// Tensor-core tiles or the row kernels (MOE_OPT_INT4_GEMM). Rows in us against
// tiles in us, by rows an expert, 128 experts of 2048 x 1536: 2: 60 / 87,
// 4: 90 / 98, 8: 95 / 99, 12: 125 / 99; 8 experts of 4096 x 14336: 2: 72 / 105,
// 8: 112 / 112, 12: 136 / 111. The counts are on the device, so the rule goes by
// the mean: with 8 on average and one expert of 100 or 500 rows the row kernels
// take 202 and 701 us, the tiles 97 and 99 (a caller that knows its routing to be
// that uneven sets the option).
constexpr int64_t kRowsPerExpert = 8;
bool use_gemm(int64_t rows, int64_t n_out, int64_t w_rows, int E) {
  const int opt = moe_get_option(MOE_OPT_INT4_GEMM);
  if (opt == 0 || rows == 0 || !int4_gemm_fits(rows, n_out, w_rows, E)) return false;
  return opt == 1 || rows > kRowsPerExpert * std::min<int64_t>(E, rows);
}

// rows: how many rows there are in all
template <bool SWIGLU>
int launch_rows(const MvParams& p, int dtype, int group, int64_t rows, cudaStream_t st) {
  if (dtype == MOE_BF16) {
    if (group == 128) return launch_rows_group<__nv_bfloat16, 128, SWIGLU>(p, rows, st);
    if (group == 64) return launch_rows_group<__nv_bfloat16, 64, SWIGLU>(p, rows, st);
    return launch_rows_group<__nv_bfloat16, 32, SWIGLU>(p, rows, st);
  }
  if (group == 128) return launch_rows_group<__half, 128, SWIGLU>(p, rows, st);
  if (group == 64) return launch_rows_group<__half, 64, SWIGLU>(p, rows, st);
  return launch_rows_group<__half, 32, SWIGLU>(p, rows, st);
}

// A product over consecutive rows of each expert, whichever way.
template <bool SWIGLU>
int launch_grouped(const MvParams& p, int dtype, int group, bool gemm, cudaStream_t st) {
  if (!gemm) return launch_rows<SWIGLU>(p, dtype, group, p.total_rows, st);
  return int4_gemm(p.x, dtype, p.total_rows, p.K, p.w, p.scale, group, p.E, p.n_out, SWIGLU, p.counts, p.counts_is64,
                   p.out, p.out_f32 != 0, st);
}

struct LayerWs {
  size_t xp, h, o, align, sorted, slot_pos, gs, poff, table, align_bytes, bytes;
  bool gemm;    // tensor-core tiles
  bool direct;  // the top-k ids are read by the product kernels themselves
  bool down;    // the down projection and the combine in one launch
};
LayerWs layer_ws(int64_t T, int64_t H, int64_t I, int E, int k) {
  LayerWs w{};
  const int64_t S = T * k;
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t o = off;
    off = align_up(off + bytes, 256);
    return o;
  };
  w.gemm = use_gemm(S, std::max(H, I), std::max(H, 2 * I), E);
  w.direct = !w.gemm && S <= kMaxSlots;
  w.down = w.direct && S <= kDownSlots && T <= kDownTokens;
  w.xp = take(w.gemm ? (size_t)S * H * 2 : 0);
  w.h = take((size_t)S * I * 2);
  w.o = take(w.down ? 0 : (size_t)S * H * sizeof(float));
  if (!w.direct) {
    w.align_bytes = moe_align_workspace_size(T, k, E, 1);
    w.align = take(w.align_bytes);
    w.sorted = take((size_t)moe_align_capacity(S, E, 1) * sizeof(int32_t));
    w.slot_pos = take((size_t)S * sizeof(int32_t));
    w.gs = take((size_t)E * sizeof(int32_t));
    w.poff = take((size_t)(E + 1) * sizeof(int32_t));
    w.table = take((size_t)moe_tile_table_ints(E, moe_align_capacity(S, E, 1)) * sizeof(int32_t));
  }
  w.bytes = off;
  return w;
}

int check_weights(const char* fn, int dtype, int64_t k, int64_t n, int E, int group) {
  MOE_CHECK_ARG(act_ok(dtype), "%s: 4-bit weights take bf16 or fp16 activations", fn);
  MOE_CHECK_ARG(u4::group_ok(group), "%s: group size %d is not 32, 64 or 128", fn, group);
  MOE_CHECK_ARG(k > 0 && k % group == 0 && k < (int64_t(1) << 30),
                "%s: reduction length %lld must be a positive multiple of the group size %d", fn, (long long)k, group);
  MOE_CHECK_ARG(n > 0 && n < (int64_t(1) << 30), "%s: bad output size %lld", fn, (long long)n);
  MOE_CHECK_ARG(E > 0 && E <= 1024, "%s: num_experts %d outside [1, 1024]", fn, E);
  return MOE_OK;
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" int moe_quant_int4_groups(const void* src, int src_dtype, int64_t rows, int64_t cols, int group_size,
                                     uint8_t* dst, void* dst_scale, int scale_dtype, void* stream) {
  MOE_CHECK_ARG(src_dtype == MOE_BF16 || src_dtype == MOE_F16 || src_dtype == MOE_F32,
                "moe_quant_int4_groups: source must be bf16, fp16 or fp32");
  MOE_CHECK_ARG(act_ok(scale_dtype), "moe_quant_int4_groups: scales must be bf16 or fp16");
  MOE_CHECK_ARG(u4::group_ok(group_size), "moe_quant_int4_groups: group size %d is not 32, 64 or 128", group_size);
  MOE_CHECK_ARG(rows >= 0 && cols > 0 && cols % group_size == 0,
                "moe_quant_int4_groups: columns (%lld) must be a positive multiple of the group size %d",
                (long long)cols, group_size);
  if (rows == 0) return MOE_OK;
  MOE_CHECK_ARG(src && dst && dst_scale, "moe_quant_int4_groups: NULL pointer");
  MOE_CHECK_ARG((uintptr_t)src % 16 == 0 && (uintptr_t)dst % 8 == 0,
                "moe_quant_int4_groups: source must be 16-byte and output 8-byte aligned");
  const int64_t n16 = rows * cols / 16;
  cudaStream_t st = as_stream(stream);
  if (scale_dtype == MOE_BF16) {
    if (src_dtype == MOE_BF16) return launch_quant<__nv_bfloat16, __nv_bfloat16>(src, n16, group_size, dst, dst_scale, st);
    if (src_dtype == MOE_F16) return launch_quant<__half, __nv_bfloat16>(src, n16, group_size, dst, dst_scale, st);
    return launch_quant<float, __nv_bfloat16>(src, n16, group_size, dst, dst_scale, st);
  }
  if (src_dtype == MOE_BF16) return launch_quant<__nv_bfloat16, __half>(src, n16, group_size, dst, dst_scale, st);
  if (src_dtype == MOE_F16) return launch_quant<__half, __half>(src, n16, group_size, dst, dst_scale, st);
  return launch_quant<float, __half>(src, n16, group_size, dst, dst_scale, st);
}

extern "C" int moe_dequant_int4_groups(const uint8_t* src, const void* scale, int scale_dtype, int64_t rows,
                                       int64_t cols, int group_size, void* dst, int dst_dtype, void* stream) {
  MOE_CHECK_ARG(dst_dtype == MOE_BF16 || dst_dtype == MOE_F16 || dst_dtype == MOE_F32,
                "moe_dequant_int4_groups: output must be bf16, fp16 or fp32");
  MOE_CHECK_ARG(act_ok(scale_dtype), "moe_dequant_int4_groups: scales must be bf16 or fp16");
  MOE_CHECK_ARG(u4::group_ok(group_size), "moe_dequant_int4_groups: group size %d is not 32, 64 or 128", group_size);
  MOE_CHECK_ARG(rows >= 0 && cols > 0 && cols % group_size == 0,
                "moe_dequant_int4_groups: columns (%lld) must be a positive multiple of the group size %d",
                (long long)cols, group_size);
  if (rows == 0) return MOE_OK;
  MOE_CHECK_ARG(src && scale && dst, "moe_dequant_int4_groups: NULL pointer");
  MOE_CHECK_ARG((uintptr_t)src % 4 == 0 && (uintptr_t)dst % 16 == 0,
                "moe_dequant_int4_groups: source must be 4-byte and output 16-byte aligned");
  const int64_t n8 = rows * cols / 8;
  cudaStream_t st = as_stream(stream);
  if (scale_dtype == MOE_BF16) {
    if (dst_dtype == MOE_BF16) return launch_dequant<__nv_bfloat16, __nv_bfloat16>(src, scale, n8, group_size, dst, st);
    if (dst_dtype == MOE_F16) return launch_dequant<__nv_bfloat16, __half>(src, scale, n8, group_size, dst, st);
    return launch_dequant<__nv_bfloat16, float>(src, scale, n8, group_size, dst, st);
  }
  if (dst_dtype == MOE_BF16) return launch_dequant<__half, __nv_bfloat16>(src, scale, n8, group_size, dst, st);
  if (dst_dtype == MOE_F16) return launch_dequant<__half, __half>(src, scale, n8, group_size, dst, st);
  return launch_dequant<__half, float>(src, scale, n8, group_size, dst, st);
}

extern "C" int moe_grouped_matmul_int4(const void* x, int dtype, int64_t num_rows, int64_t k, const uint8_t* w,
                                       const void* w_scale, int group_size, int num_experts, int64_t n,
                                       const void* group_sizes, int gs_dtype, void* out, void* stream) {
  MOE_TRY(check_weights("moe_grouped_matmul_int4", dtype, k, n, num_experts, group_size));
  MOE_CHECK_ARG(gs_dtype == MOE_I32 || gs_dtype == MOE_I64, "moe_grouped_matmul_int4: group sizes must be int32 or int64");
  MOE_CHECK_ARG(num_rows >= 0 && num_rows < (int64_t(1) << 31), "moe_grouped_matmul_int4: bad row count");
  if (num_rows == 0) return MOE_OK;
  MOE_CHECK_ARG(x && w && w_scale && group_sizes && out, "moe_grouped_matmul_int4: NULL pointer");
  MOE_CHECK_ARG((uintptr_t)x % 16 == 0 && (uintptr_t)w % 16 == 0 && (uintptr_t)out % 16 == 0,
                "moe_grouped_matmul_int4: pointers must be 16-byte aligned");
  MvParams p{};
  p.x = x;
  p.w = w;
  p.scale = w_scale;
  p.out = out;
  p.K = k;
  p.n_out = (int)n;
  p.w_rows = (int)n;
  p.E = num_experts;
  p.counts = group_sizes;
  p.counts_is64 = gs_dtype == MOE_I64;
  p.total_rows = num_rows;
  p.x_div = 1;
  return launch_grouped<false>(p, dtype, group_size, use_gemm(num_rows, n, n, num_experts), as_stream(stream));
}

extern "C" size_t moe_fused_experts_int4_workspace_size(int64_t num_tokens, int64_t hidden, int64_t inter,
                                                        int num_experts, int top_k) {
  if (num_tokens < 0 || hidden <= 0 || inter <= 0 || num_experts <= 0 || top_k <= 0) return 0;
  return layer_ws(num_tokens, hidden, inter, num_experts, top_k).bytes;
}

extern "C" int moe_fused_experts_int4(const void* x, int dtype, int64_t num_tokens, int64_t hidden,
                                      const uint8_t* w13, const void* w13_scale, const uint8_t* w2,
                                      const void* w2_scale, int group_size, int num_experts, int64_t inter,
                                      const float* topk_weights, const int32_t* topk_ids, int top_k, void* y,
                                      void* workspace, size_t workspace_bytes, void* stream) {
  MOE_TRY(check_weights("moe_fused_experts_int4", dtype, hidden, inter, num_experts, group_size));
  MOE_TRY(check_weights("moe_fused_experts_int4", dtype, inter, hidden, num_experts, group_size));
  MOE_CHECK_ARG(num_tokens >= 0 && top_k > 0 && num_tokens * top_k < (int64_t(1) << 31),
                "moe_fused_experts_int4: bad sizes");
  if (num_tokens == 0) return MOE_OK;
  MOE_CHECK_ARG(x && w13 && w13_scale && w2 && w2_scale && topk_weights && topk_ids && y,
                "moe_fused_experts_int4: NULL pointer");
  MOE_CHECK_ARG((uintptr_t)x % 16 == 0 && (uintptr_t)w13 % 16 == 0 && (uintptr_t)w2 % 16 == 0 && (uintptr_t)y % 16 == 0,
                "moe_fused_experts_int4: pointers must be 16-byte aligned");
  const LayerWs w = layer_ws(num_tokens, hidden, inter, num_experts, top_k);
  if (workspace_bytes < w.bytes || !workspace)
    return set_error(MOE_ERR_WORKSPACE, "moe_fused_experts_int4: workspace %zu < %zu bytes", workspace_bytes, w.bytes);
  char* ws = static_cast<char*>(workspace);
  cudaStream_t st = as_stream(stream);
  const int64_t S = num_tokens * top_k;
  MvParams p{};
  p.E = num_experts;
  p.total_rows = S;
  p.x_div = top_k;
  if (w.direct) {
    p.ids = topk_ids;
    p.slots = (int)S;
  } else {
    int32_t* sorted = reinterpret_cast<int32_t*>(ws + w.sorted);
    MOE_TRY(moe_align(topk_ids, num_tokens, top_k, num_experts, 1, sorted, reinterpret_cast<int32_t*>(ws + w.slot_pos),
                      reinterpret_cast<int32_t*>(ws + w.gs), reinterpret_cast<int32_t*>(ws + w.poff),
                      reinterpret_cast<int32_t*>(ws + w.table), ws + w.align, w.align_bytes, stream));
    p.counts = ws + w.gs;
    p.row_map = sorted;
  }
  p.x = x;
  if (w.gemm) {
    // each token's row to its place in every expert's run of rows
    const int32_t* slot_pos = reinterpret_cast<const int32_t*>(ws + w.slot_pos);
    if (scatter_rows_fits(hidden))
      MOE_TRY(scatter_rows(x, dtype, hidden, slot_pos, top_k, num_tokens, ws + w.xp, dtype, nullptr, st));
    else
      MOE_TRY(gather_rows(x, dtype, hidden, p.row_map, top_k, S,
                          reinterpret_cast<const int32_t*>(ws + w.table) + 1, ws + w.xp, dtype, nullptr, false, stream));
    p.x = ws + w.xp;
    p.row_map = nullptr;
    p.x_div = 1;
  }
  p.w = w13;
  p.scale = w13_scale;
  p.out = ws + w.h;
  p.K = hidden;
  p.n_out = (int)inter;
  p.w_rows = (int)(2 * inter);
  MOE_TRY(launch_grouped<true>(p, dtype, group_size, w.gemm, st));
  if (w.down) {
    DownParams d{};
    d.h = ws + w.h;
    d.w = w2;
    d.scale = w2_scale;
    d.weights = topk_weights;
    d.ids = topk_ids;
    d.y = y;
    d.K = inter;
    d.n_out = (int)hidden;
    d.E = num_experts;
    d.tokens = (int)num_tokens;
    d.top_k = top_k;
    d.slots = (int)S;
    return launch_down_any(d, dtype, group_size, st);
  }
  p.x = ws + w.h;
  p.w = w2;
  p.scale = w2_scale;
  p.out = ws + w.o;
  p.out_f32 = 1;
  p.K = inter;
  p.n_out = p.w_rows = (int)hidden;
  p.row_map = nullptr;
  p.x_div = 1;
  MOE_TRY(launch_grouped<false>(p, dtype, group_size, w.gemm, st));
  const int64_t h8 = hidden / 8;
  const int32_t* slot_row = w.direct ? nullptr : reinterpret_cast<const int32_t*>(ws + w.slot_pos);
  const float* o = reinterpret_cast<const float*>(ws + w.o);
  if (dtype == MOE_BF16)
    MOE_CUDA_TRY(launch_kernel(int4_combine_kernel<__nv_bfloat16>, dim3(flat_grid(num_tokens * h8)), dim3(256), 0, st,
                               o, topk_ids, slot_row, topk_weights, num_tokens * h8, h8, top_k, num_experts,
                               static_cast<__nv_bfloat16*>(y)));
  else
    MOE_CUDA_TRY(launch_kernel(int4_combine_kernel<__half>, dim3(flat_grid(num_tokens * h8)), dim3(256), 0, st, o,
                               topk_ids, slot_row, topk_weights, num_tokens * h8, h8, top_k, num_experts,
                               static_cast<__half*>(y)));
  MOE_LAUNCH_CHECK("int4_combine_kernel");
  return MOE_OK;
}

extern "C" size_t moe_fused_mlp_int4_workspace_size(int64_t num_tokens, int64_t inter, int num_experts) {
  if (num_tokens < 0 || inter <= 0 || num_experts <= 0) return 0;
  return align_up((size_t)num_tokens * inter * 2, 256);
}

extern "C" int moe_fused_mlp_int4(const void* x, int dtype, int64_t num_tokens, int64_t hidden, const uint8_t* w13,
                                  const void* w13_scale, const uint8_t* w2, const void* w2_scale, int group_size,
                                  int num_experts, int64_t inter, const void* group_sizes, int gs_dtype, void* out,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  MOE_TRY(check_weights("moe_fused_mlp_int4", dtype, hidden, inter, num_experts, group_size));
  MOE_TRY(check_weights("moe_fused_mlp_int4", dtype, inter, hidden, num_experts, group_size));
  MOE_CHECK_ARG(gs_dtype == MOE_I32 || gs_dtype == MOE_I64, "moe_fused_mlp_int4: group sizes must be int32 or int64");
  MOE_CHECK_ARG(num_tokens >= 0 && num_tokens < (int64_t(1) << 31), "moe_fused_mlp_int4: bad row count");
  if (num_tokens == 0) return MOE_OK;
  MOE_CHECK_ARG(x && w13 && w13_scale && w2 && w2_scale && group_sizes && out, "moe_fused_mlp_int4: NULL pointer");
  MOE_CHECK_ARG((uintptr_t)x % 16 == 0 && (uintptr_t)w13 % 16 == 0 && (uintptr_t)w2 % 16 == 0 && (uintptr_t)out % 16 == 0,
                "moe_fused_mlp_int4: pointers must be 16-byte aligned");
  const size_t need = moe_fused_mlp_int4_workspace_size(num_tokens, inter, num_experts);
  if (workspace_bytes < need || !workspace)
    return set_error(MOE_ERR_WORKSPACE, "moe_fused_mlp_int4: workspace %zu < %zu bytes", workspace_bytes, need);
  cudaStream_t st = as_stream(stream);
  MvParams p{};
  p.E = num_experts;
  p.total_rows = num_tokens;
  p.x_div = 1;
  p.counts = group_sizes;
  p.counts_is64 = gs_dtype == MOE_I64;
  p.x = x;
  p.w = w13;
  p.scale = w13_scale;
  p.out = workspace;
  p.K = hidden;
  p.n_out = (int)inter;
  p.w_rows = (int)(2 * inter);
  const bool gemm = use_gemm(num_tokens, std::max(hidden, inter), std::max(hidden, 2 * inter), num_experts);
  MOE_TRY(launch_grouped<true>(p, dtype, group_size, gemm, st));
  p.x = workspace;
  p.w = w2;
  p.scale = w2_scale;
  p.out = out;
  p.K = inter;
  p.n_out = p.w_rows = (int)hidden;
  return launch_grouped<false>(p, dtype, group_size, gemm, st);
}
