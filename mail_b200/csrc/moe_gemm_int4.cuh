// Products grouped by expert with 4-bit weights on the tensor cores (tcgen05).
//
// Included by moe_gemm.cu (same translation unit: it shares the device error
// flag, the tensor-map helpers and the PTX wrappers).
//
//   out[r, n] = sum_k x[r, k] W[e(r), n, k],  W = (q - 8) s   (int4.cuh)
//
// The 128 weight rows of a feature tile are the MMA's M operand and the
// expert's rows (up to 256, evenly split over its tiles, rounded up to 16) its
// N operand, so an expert with few rows costs few MMA columns. The tensor
// cores take 16-bit operands: twelve or sixteen warps turn the 4-bit words into
// (q - 8) s in shared memory while earlier blocks multiply. A weight is
// rounded to the activations' type there, by at most half a step (in fp16 to
// infinity beyond 65504, scales above 8188; a smaller unit would cost weights
// below 2^-11 bits instead): scaling after the product would read the
// accumulator once for every group.
//
// Measured: 8192 rows over eight experts of 4096 x 14336 738 us, 1304 TFLOP/s,
// 0.79 of the measured burst (878 us back to back, under the power limit);
// 2048 rows over 64 experts of 7168 x 4096 396 us, 2.4 TB/s of weights, bound by
// decoding and by the barriers between the roles (no decoding: 323 us, no
// decoding, products or rows of x: 314 us).
//
// Roles (one CTA per SM, persistent), a warp each:
//   issue      TMEM, MMAs into one of two accumulators
//   rows in    x by TMA: 64 k by up to 256 rows a block
//   words in   4-bit words by TMA: 128 k by 128 weight rows a block
//   scales in  the scales of those rows. The decoding warps do not load them
//              themselves: the proxy fence after their stores would wait for
//              every load in flight, a DRAM latency for each block.
//   epilogue   four warps
//   decode     three or four sets of four warps, a thread to a weight row
// With SWIGLU a tile's rows alternate between 16 gate rows and the 16 up rows
// that go with them, so gate and up of a feature sit sixteen TMEM lanes apart
// in one warp, and a shuffle for every two tokens brings them together.
#include "int4.cuh"

namespace moe {
namespace {

constexpr int Q4_FEAT = 128;             // weight rows of a tile (UMMA M)
constexpr int Q4_KB = 64;                // k of an MMA block (128 bytes of 16-bit type)
constexpr int Q4_RAW_ROW = 64;           // bytes of 4-bit words in a block of 128 k
constexpr uint32_t Q4_WORD_BYTES = Q4_FEAT * Q4_RAW_ROW;
constexpr uint32_t q4_raw_bytes(int group) { return Q4_WORD_BYTES + Q4_FEAT * 2 * (128 / group); }  // and scales
constexpr uint32_t Q4_A_BYTES = Q4_FEAT * ROW_BYTES;
constexpr int Q4_BOXES = 5;              // boxes of 16, 32, 64, 128 and 256 rows of x

// Rows of x of a tile and pipeline depth. Wide tiles for many rows an expert;
// narrow ones, with more blocks in flight, where the weights bound the launch.
//
// Set s of the decoding warps takes every kSets-th MMA block (64 k) and writes
// it to the stages s, s + kSets, .. in turn, so it waits for no use of a stage
// but the one after its own last. (A wait on a barrier's parity cannot tell a use
// from the use two before it; a set that shared stages could overtake a slower
// one.) The words' slots are shared, kRawStep by kRawStep between kMinRaw and
// kMaxRaw of them, so that the same holds there: three sets know the blocks of
// words up to five before the next one multiplied; four sets come to every
// second block, and an even number of slots makes a slot's last use their own.
// The host takes as many as shared memory holds: wide tiles four for groups of
// 128 over up to 91 experts, else two (8192 rows over eight experts of 4096 x
// 14336 with two: 799 us against 743; groups of 64 and 32 take 825 and 972);
// narrow ones nine, or eight for groups of 32, 64 and 128 over more than 91, 667
// and 955 experts.
// Narrow tiles have two stages for each set: it decodes one while the other
// multiplies. Wide ones multiply longer than they decode, and four sets with a
// stage each keep up.
template <bool NARROW>
struct Int4Shape {
  static constexpr int kRows = NARROW ? 64 : 256;  // rows of x of a tile at most (UMMA N)
  static constexpr int kSets = NARROW ? 3 : 4;
  static constexpr int kStages = NARROW ? 6 : 4;   // MMA blocks of decoded weights and rows of x
  static constexpr int kMaxRaw = NARROW ? 9 : 4;   // blocks (128 k) of words and scales
  static constexpr int kMinRaw = NARROW ? 6 : 2, kRawStep = NARROW ? 1 : 2;
  static constexpr uint32_t kXBytes = kRows * ROW_BYTES;
  static constexpr int kThreads = 32 * (8 + 4 * kSets);
};
// Narrow tiles up to this many rows an expert on average. Narrow in us against
// wide in us, 64 experts of 2048 x 1536: 32: 58 / 63, 48: 60 / 65, 64: 79 / 67;
// 16 experts of 4096 x 4096: 32: 70 / 79, 48: 72 / 82, 64: 102 / 84. Narrow as
// well where all of them run at once (777 rows, 5 experts of 1056 x 1001: 12.6 /
// 17.6; not so, 600 rows, 2 experts of 7168 x 2048: 60 / 40).
constexpr int64_t kInt4NarrowRows = 48;

struct Int4Maps {
  CUtensorMap w;
  CUtensorMap x[Q4_BOXES];
};

struct Int4Params {
  int E;
  int K;
  int nf;                // feature tiles
  int n_out;             // output features
  int w_rows;            // weight rows of an expert (n_out, or 2 n_out with SWIGLU)
  const void* scale;     // [E, w_rows, K / group]
  const void* counts;    // rows of each expert
  int counts_is64;
  int64_t total_rows;    // rows of x and out
  void* out;             // [total_rows, n_out]
  int out_f32;
  uint32_t idesc_m;      // instruction descriptor without the N field
  int raw;               // blocks of words in flight
};

struct Int4Smem {
  uint64_t raw_full[9], raw_empty[9], full[6], empty[6];
  uint64_t tfull[2], tempty[2], drain;
  uint32_t tmem_slot;
  int abort_flag;
};

// A tile of work: expert e, rows [row, row + rows), feature tile f.
struct Int4Item {
  int e, f, rows;
  int64_t row;
};

// Items run expert by expert, then feature tile, then the expert's row tiles,
// so CTAs that run together share weight tiles and rows of x in L2.
__device__ __forceinline__ Int4Item int4_item(int item, const int32_t* s_cum, const int32_t* s_off, int E, int nf) {
  int lo = 0, hi = E;  // s_cum[lo] * nf <= item < s_cum[hi] * nf
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s_cum[mid] * nf <= item) lo = mid;
    else hi = mid;
  }
  Int4Item it;
  it.e = lo;
  const int tiles = s_cum[lo + 1] - s_cum[lo];
  const int local = item - s_cum[lo] * nf;
  it.f = local / tiles;
  const int cnt = s_off[lo + 1] - s_off[lo];
  const int per = ((cnt + tiles - 1) / tiles + 15) & ~15;
  const int first = local % tiles * per;
  it.rows = min(per, cnt - first);
  it.row = (int64_t)s_off[lo] + first;
  return it;
}

__device__ __forceinline__ uint4 ld_shared16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ uint32_t ld_shared4(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t ld_shared2(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_shared16(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}

template <typename T>
struct Decode;
template <>
struct Decode<__nv_bfloat16> {
  static constexpr uint32_t kMagic = 0x43004300u;  // 128
  static __device__ __forceinline__ uint32_t value(uint32_t m, uint32_t s2) {
    return u4::as_u32(__hmul2(__hsub2(u4::as_bf162(m), u4::as_bf162(0x43084308u)), u4::as_bf162(s2)));
  }
};
template <>
struct Decode<__half> {
  static constexpr uint32_t kMagic = 0x64006400u;  // 1024
  static __device__ __forceinline__ uint32_t value(uint32_t m, uint32_t s2) {
    return u4::as_u32(__hmul2(__hsub2(u4::as_half2(m), u4::as_half2(0x64086408u)), u4::as_half2(s2)));
  }
};

// The eight weights of a word in the order of k, times the scale.
template <typename T>
__device__ __forceinline__ uint4 decode_word(uint32_t w, uint32_t s2) {
  const uint32_t v = w >> 4;
  uint32_t r[4];
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    // byte b of w (its low nibble is k = 2b) and of w >> 4 (2b + 1)
    const uint32_t t = __byte_perm(w, v, b | (b << 4) | ((4 + b) << 8) | ((4 + b) << 12));
    r[b] = Decode<T>::value(u4::and_or<0x000f000fu>(t, Decode<T>::kMagic), s2);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

// Waits at once if `ready` (an earlier look at the same phase found it
// complete). The same answer for the whole warp.
template <int NS>
__device__ __forceinline__ bool int4_wait(bool ready, uint64_t* bar, uint32_t parity, volatile int* abort) {
  if (__all_sync(0xffffffffu, ready)) return true;
  return __all_sync(0xffffffffu, NS == 0 ? ptx::mbar_wait(bar, parity, abort)
                                         : ptx::mbar_wait_sleepy<NS>(bar, parity, abort));
}

template <typename T, int GROUP, bool SWIGLU, bool NARROW>
__global__ void __launch_bounds__(Int4Shape<NARROW>::kThreads, 1)
    int4_gemm_kernel(const __grid_constant__ Int4Maps maps, const Int4Params p) {
  using Sh = Int4Shape<NARROW>;
  constexpr int kStages = Sh::kStages, kSets = Sh::kSets;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sX = sA + kStages * Q4_A_BYTES;
  uint8_t* sR = sX + kStages * Sh::kXBytes;          // words, then scales
  uint8_t* sS = sR + p.raw * Q4_WORD_BYTES;
  constexpr int NS = 128 / GROUP;                     // groups of a block of words
  constexpr uint32_t kScaleBytes = Q4_FEAT * 2 * NS;
  Int4Smem& sm = *reinterpret_cast<Int4Smem*>(sS + p.raw * kScaleBytes);
  int32_t* s_off = reinterpret_cast<int32_t*>(&sm + 1);  // [E + 1] first row of each expert
  int32_t* s_cum = s_off + p.E + 1;                      // [E + 1] row tiles before each expert
  volatile int* abort_flag = &sm.abort_flag;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  // Wide: warps 0..3 epilogue, 4..7 issue and loads, the others decode, four on
  // each scheduler. Narrow: issue, the loads and a quarter of the epilogue have
  // the scheduler of warps 1, 5, 9, .. to themselves, since there the MMAs of a
  // block take no longer than their issue (layer of 256 experts at 1024 tokens:
  // 2577 against 2693 us; the wide shape that way: 779 against 741 us).
  enum { kIssue, kRowsIn, kWordsIn, kScalesIn, kEpilogue, kDecode };
  int role, decoder;
  if constexpr (NARROW) {
    const int sub = warp & 3, level = warp >> 2;
    decoder = (level - 1) * 3 + (sub == 0 ? 0 : sub - 1);
    role = sub != 1 ? (level == 0 ? kEpilogue : kDecode)
                    : level == 0 ? kIssue : level == 1 ? kRowsIn : level == 2 ? kWordsIn
                                                     : level == 3 ? kEpilogue : kScalesIn;
    static_assert(!NARROW || 4 * kSets == 12, "decoding warps on three schedulers");
  } else {
    decoder = warp - 8;
    role = warp < 4 ? kEpilogue : warp == 4 ? kIssue : warp == 5 ? kRowsIn : warp == 6 ? kWordsIn
                                             : warp == 7 ? kScalesIn : kDecode;
  }
  const int E = p.E;
  if (threadIdx.x == 0) {
    for (int i = 0; i < p.raw; ++i) {
      ptx::mbar_init(&sm.raw_full[i], 1 + 32);  // words, the lanes that store the scales
      ptx::mbar_init(&sm.raw_empty[i], 8);  // the warps of two sets, one for each half
    }
    for (int i = 0; i < kStages; ++i) {
      ptx::mbar_init(&sm.full[i], 5);  // the rows' copy and the warps of a set
      ptx::mbar_init(&sm.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(&sm.tfull[i], 1);
      ptx::mbar_init(&sm.tempty[i], 4);  // epilogue warps
    }
    ptx::mbar_init(&sm.drain, 1);
    sm.abort_flag = 0;
    ptx::fence_mbar_init();
    ptx::prefetch_tmap(&maps.w);
  }
  pdl_begin();
  if (role == kWordsIn) {
    // rows and row tiles before each expert, counts cut off at total_rows
    const int per = (E + 31) / 32;
    const int lo = min(E, lane * per), hi = min(E, lo + per);
    auto count = [&](int e) -> int64_t {
      const int64_t c = p.counts_is64 ? static_cast<const int64_t*>(p.counts)[e]
                                      : (int64_t) static_cast<const int32_t*>(p.counts)[e];
      return max((int64_t)0, min(c, p.total_rows));
    };
    int64_t sum = 0;
    for (int e = lo; e < hi; ++e) sum += count(e);
    int64_t incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    int64_t run = incl - sum;
    int tiles = 0;
    for (int e = lo; e < hi; ++e) {
      const int64_t first = min(run, p.total_rows);
      run += count(e);
      const int64_t end = min(run, p.total_rows);
      s_off[e] = (int32_t)first;
      tiles += (int)((end - first + Sh::kRows - 1) / Sh::kRows);
    }
    const int64_t all = __shfl_sync(0xffffffffu, incl, 31);
    if (lane == 31) s_off[E] = (int32_t)min(all, p.total_rows);
    __syncwarp();
    int tincl = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, tincl, o);
      if (lane >= o) tincl += v;
    }
    int trun = tincl - tiles;
    for (int e = lo; e < hi; ++e) {
      s_cum[e] = trun;
      trun += (s_off[e + 1] - s_off[e] + Sh::kRows - 1) / Sh::kRows;
    }
    if (lane == 31) s_cum[E] = tincl;
  }
  if (role == kIssue) {
    ptx::tmem_alloc(&sm.tmem_slot, TMEM_COLS);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = sm.tmem_slot;
  const int total = s_cum[E] * p.nf;
  // blocks of words (128 k), each two MMA blocks (64 k); past K the words, their
  // scales and x read as zero
  const int nraw = (p.K + 2 * Q4_KB - 1) / (2 * Q4_KB);
  const int nkb = 2 * nraw;

  if (role == kRowsIn) {
    // ------------------------------------------------------------ rows of x
    // The rows of a tile come in up to three boxes whose heights are powers of
    // two, the last rounded up to 16.
    int item = blockIdx.x, kb = 0, h0 = 0, h1 = 0, h2 = 0, row = 0;
    uint32_t bytes = 0, phase = 0;
    auto start = [&]() {
      const Int4Item it = int4_item(item, s_cum, s_off, E, p.nf);
      row = (int)it.row;
      int left = (it.rows + 15) & ~15;
      auto take = [&](bool last) -> int {
        if (left == 0) return 0;
        const int h = 1 << (last ? 32 - __clz(left - 1) : 31 - __clz(left));
        left = max(0, left - h);
        return h;
      };
      h0 = take(false);
      h1 = take(false);
      h2 = take(true);
      bytes = (uint32_t)(h0 + h1 + h2) * ROW_BYTES;
    };
    auto box = [&](int h) { return &maps.x[h ? 31 - __clz(h) - 4 : 0]; };
    auto x_load = [&](uint32_t dst, const CUtensorMap* m, uint64_t* bar, int x, int y) {
      asm volatile(
          "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
              dst),
          "l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(y), "r"(ptx::smem_u32(bar))
          : "memory");
    };
    const bool issuer = ptx::elect_one();
    bool ok = true, ready = false;
    int st = 0, filled = 0;
    while (item < total) {
      start();
      const CUtensorMap *m0 = box(h0), *m1 = box(h1), *m2 = box(h2);
      for (kb = 0; kb < nkb; ++kb) {
        uint64_t* const full = &sm.full[st];
        const uint32_t dst = ptx::smem_u32(sX + st * Sh::kXBytes);
        ok = int4_wait<20>(ready, &sm.empty[st], phase ^ 1, abort_flag);
        if (!ok) break;
        if (++st == kStages) {
          st = 0;
          phase ^= 1;
        }
        ready = ptx::mbar_test_wait(&sm.empty[st], phase ^ 1);
        if (issuer) {
          ptx::mbar_arrive_expect_tx(full, bytes);
          x_load(dst, m0, full, kb * Q4_KB, row);
        }
        if (h1 && issuer) x_load(dst + h0 * ROW_BYTES, m1, full, kb * Q4_KB, row + h0);
        if (h2 && issuer) x_load(dst + (h0 + h1) * ROW_BYTES, m2, full, kb * Q4_KB, row + h0 + h1);
        __syncwarp();
        filled = min(filled + 1, kStages);
      }
      if (!ok) break;
      item += gridDim.x;
    }
    if (!ok && lane == 0) {
      raise_device_error(1);
      *abort_flag = 1;
      volatile int never = 0;  // copies in flight land before the CTA exits
      for (; filled > 0; --filled) {
        if (st == 0) {
          st = kStages;
          phase ^= 1;
        }
        --st;
        ptx::mbar_wait(&sm.full[st], phase, &never, 100000000ull);
      }
    }
    __syncwarp();
  } else if (role == kWordsIn) {
    // ------------------------------------------------------------ 4-bit words
    int slot = 0, filled = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int item = blockIdx.x; ok && item < total; item += gridDim.x) {
      const Int4Item it = int4_item(item, s_cum, s_off, E, p.nf);
      const int wrow = it.e * p.w_rows + it.f * (SWIGLU ? Q4_FEAT / 2 : Q4_FEAT);
      for (int kb = 0; kb < nraw; ++kb) {
        ok = int4_wait<40>(false, &sm.raw_empty[slot], phase ^ 1, abort_flag);
        if (!ok) break;
        if (ptx::elect_one()) {
          uint64_t* bar = &sm.raw_full[slot];
          uint8_t* dst = sR + slot * Q4_WORD_BYTES;
          ptx::mbar_arrive_expect_tx(bar, Q4_WORD_BYTES);
          ptx::tma_load_2d(dst, &maps.w, bar, kb * Q4_RAW_ROW, wrow);
          if constexpr (SWIGLU)
            ptx::tma_load_2d(dst + Q4_WORD_BYTES / 2, &maps.w, bar, kb * Q4_RAW_ROW, wrow + p.n_out);
        }
        __syncwarp();
        if (++slot == p.raw) {
          slot = 0;
          phase ^= 1;
        }
        filled = min(filled + 1, p.raw);
      }
    }
    if (!ok && lane == 0) {
      raise_device_error(1);
      *abort_flag = 1;
      volatile int never = 0;
      for (; filled > 0; --filled) {  // newest first
        if (slot == 0) {
          slot = p.raw;
          phase ^= 1;
        }
        --slot;
        ptx::mbar_wait(&sm.raw_full[slot], phase, &never, 100000000ull);
      }
    }
    __syncwarp();
  } else if (role == kIssue) {
    // ------------------------------------------------------------ MMA issuer
    // The whole warp runs the loop and one lane issues. The loop over the
    // stages is unrolled, so each descriptor is a constant away from one in
    // uniform registers, and the next stage's barrier is looked at before this
    // one's MMAs are issued. A block of four MMAs with few columns takes 157
    // cycles on the tensor cores; issued from a single lane with the stage in
    // a register it took 530, this way it takes 190.
    const uint32_t a_desc = ptx::smem_desc_k128_lo(ptx::smem_u32(sA));
    const uint32_t x_desc = ptx::smem_desc_k128_lo(ptx::smem_u32(sX));
    const bool issuer = ptx::elect_one();
    int item = blockIdx.x, n = 0, kb = 0;
    uint32_t phase = 0, idesc = 0, d = 0;
    bool ok = true, ready = false;
    auto start = [&]() {  // the next tile's accumulator, free
      if (item >= total) return;
      const Int4Item it = int4_item(item, s_cum, s_off, E, p.nf);
      idesc = p.idesc_m | ((uint32_t)((it.rows + 15) / 16 * 2) << 17);
      d = tmem_base + (uint32_t)((n & 1) * Sh::kRows);
      ok = int4_wait<0>(false, &sm.tempty[n & 1], ((n >> 1) & 1) ^ 1, abort_flag);
    };
    start();
    while (ok && item < total) {
#pragma unroll
      for (int st = 0; st < kStages; ++st) {
        if (!ok || item >= total) break;
        ok = int4_wait<0>(ready, &sm.full[st], phase, abort_flag);
        if (!ok) break;
        ptx::tc_fence_after();
        ready = ptx::mbar_test_wait(&sm.full[(st + 1) % kStages], st + 1 == kStages ? phase ^ 1 : phase);
        if (issuer) {
          const uint32_t ad = a_desc + st * (Q4_A_BYTES >> 4), xd = x_desc + st * (Sh::kXBytes >> 4);
#pragma unroll
          for (int k = 0; k < ROW_BYTES / 32; ++k)
            ptx::umma_k128(d, ad + 2 * k, xd + 2 * k, idesc, (kb > 0 || k > 0) ? 1u : 0u);
          ptx::umma_commit(&sm.empty[st]);
        }
        __syncwarp();
        if (++kb == nkb) {  // (apart from the block above: a condition inside it costs 117 cycles a block)
          if (issuer) ptx::umma_commit(&sm.tfull[n & 1]);
          __syncwarp();
          kb = 0;
          ++n;
          item += gridDim.x;
          start();
        }
      }
      phase ^= 1;
    }
    if (!ok && lane == 0) {
      raise_device_error(2);
      *abort_flag = 1;
    }
    if (issuer) {
      ptx::umma_commit(&sm.drain);  // all MMAs complete before TMEM is released
      volatile int never = 0;
      if (!ptx::mbar_wait(&sm.drain, 0, &never)) raise_device_error(4);
    }
    __syncwarp();
  } else if (role == kEpilogue) {
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3;  // TMEM lanes 32 q .. 32 q + 31
    bool ok = true;
    int n = 0;
    for (int item = blockIdx.x; item < total; item += gridDim.x, ++n) {
      const Int4Item it = int4_item(item, s_cum, s_off, E, p.nf);
      const int buf = n & 1;
      ok = int4_wait<200>(false, &sm.tfull[buf], (n >> 1) & 1, abort_flag);
      if (!ok) break;
      ptx::tc_fence_after();
      const uint32_t tbase = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * Sh::kRows);
      const int feat = SWIGLU ? it.f * (Q4_FEAT / 2) + q * 16 + (lane & 15) : it.f * Q4_FEAT + q * 32 + lane;
      const bool feat_ok = feat < p.n_out;
      const int64_t base = it.row * p.n_out + feat;
#pragma unroll 1
      for (int c = 0; c < it.rows; c += 32) {
        uint32_t v[32];
        ptx::tmem_ld32(tbase + c, v);
        ptx::tmem_ld_wait();
        if constexpr (SWIGLU) {
          // even tokens finish in the gate lanes, odd ones in the up lanes
          const bool up_lane = lane >= 16;
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const uint32_t got = __shfl_xor_sync(0xffffffffu, up_lane ? v[j] : v[j + 1], 16);
            const float g = __uint_as_float(up_lane ? got : v[j]);
            const float u = __uint_as_float(up_lane ? v[j + 1] : got);
            const int tok = c + j + (up_lane ? 1 : 0);
            if (feat_ok && tok < it.rows)
              static_cast<T*>(p.out)[base + (int64_t)tok * p.n_out] = u4::Act<T>::from_float(u4::silu_mul(g, u));
          }
        } else if (feat_ok) {
          if (p.out_f32) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (c + j < it.rows)
                static_cast<float*>(p.out)[base + (int64_t)(c + j) * p.n_out] = __uint_as_float(v[j]);
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (c + j < it.rows)
                static_cast<T*>(p.out)[base + (int64_t)(c + j) * p.n_out] =
                    u4::Act<T>::from_float(__uint_as_float(v[j]));
          }
        }
        __syncwarp();
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&sm.tempty[buf]);
    }
    if (!ok) {
      if (lane == 0) raise_device_error(3);
      *abort_flag = 1;
    }
    // rows behind the last expert's are zero
    const int64_t n0 = (int64_t)s_off[E] * p.n_out, n1 = p.total_rows * p.n_out;
    for (int64_t i = n0 + (int64_t)blockIdx.x * 128 + q * 32 + lane; i < n1; i += (int64_t)gridDim.x * 128) {
      if (p.out_f32) static_cast<float*>(p.out)[i] = 0.f;
      else static_cast<uint16_t*>(p.out)[i] = 0;
    }
  } else if (role == kScalesIn) {
    // ------------------------------------------------------------ scales
    // A lane loads four rows' scales, kAhead blocks before their slot is due;
    // groups past K are 0.
    constexpr int kAhead = GROUP == 128 ? 4 : 2;
    const int groups = p.K / GROUP;
    int item = blockIdx.x, kb = 0;  // of the block loaded next
    const uint16_t* rows[4];
    auto start = [&]() {
      if (item >= total) return;
      const Int4Item it = int4_item(item, s_cum, s_off, E, p.nf);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = i * 32 + lane;
        int wr;
        if (SWIGLU)
          wr = min(it.f * (Q4_FEAT / 2) + (r >> 5) * 16 + (r & 15), p.n_out - 1) + ((r & 16) ? p.n_out : 0);
        else
          wr = min(it.f * Q4_FEAT + r, p.n_out - 1);
        rows[i] = static_cast<const uint16_t*>(p.scale) + ((int64_t)it.e * p.w_rows + wr) * groups;
      }
    };
    start();
    auto load = [&](uint16_t (&v)[4][NS]) {
      if (item >= total) return;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < NS; ++j) v[i][j] = kb * NS + j < groups ? rows[i][kb * NS + j] : (uint16_t)0;
      if (++kb == nraw) {
        kb = 0;
        item += gridDim.x;
        start();
      }
    };
    const int items = (int)blockIdx.x < total ? (total - 1 - (int)blockIdx.x) / (int)gridDim.x + 1 : 0;
    int64_t left = (int64_t)items * nraw;
    uint16_t v[kAhead][4][NS];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) load(v[i]);
    int slot = 0;
    uint32_t phase = 0;
    bool ok = true;
    while (ok && left > 0) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (!ok || left == 0) break;
        ok = int4_wait<40>(false, &sm.raw_empty[slot], phase ^ 1, abort_flag);
        if (!ok) break;
        uint16_t* dst = reinterpret_cast<uint16_t*>(sS + slot * kScaleBytes);
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int j = 0; j < NS; ++j) dst[(q * 32 + lane) * NS + j] = v[i][q][j];
        ptx::mbar_arrive(&sm.raw_full[slot]);  // every lane, for its own stores
        load(v[i]);
        if (++slot == p.raw) {
          slot = 0;
          phase ^= 1;
        }
        --left;
      }
    }
    if (!ok && lane == 0) {
      raise_device_error(1);
      *abort_flag = 1;
    }
  } else if (role == kDecode) {
    // ------------------------------------------------------------ decoding
    const int set = decoder >> 2;
    const int r = (decoder & 3) * 32 + lane;  // row of the tile
    // its row of the word block (gate rows first, then up rows)
    const int rr = SWIGLU ? ((r & 16) ? Q4_FEAT / 2 : 0) + (r >> 5) * 16 + (r & 15) : r;
    const int items = (int)blockIdx.x < total ? (total - 1 - (int)blockIdx.x) / (int)gridDim.x + 1 : 0;
    const int64_t blocks = (int64_t)items * nkb;  // this CTA's MMA blocks
    int slot = set >> 1;                          // of the words of block kb
    uint32_t raw_phase = 0, phase = 0;
    int stage = set;
    bool ok = true;
    // this row in stage 0 and in slot 0, with the swizzles' share of the row
    const uint32_t dst0 = ptx::smem_u32(sA + r * ROW_BYTES) | ((r & 7) << 4);
    const uint32_t src0 = ptx::smem_u32(sR + rr * Q4_RAW_ROW) | (((rr >> 1) & 3) << 4);
    const uint32_t scale0 = ptx::smem_u32(sS + r * 2 * NS);
    for (int64_t kb = set; kb < blocks; kb += kSets) {
      const int half = (int)(kb & 1);
      const bool freed = ptx::mbar_test_wait(&sm.empty[stage], phase ^ 1);
      ok = int4_wait<20>(ptx::mbar_test_wait(&sm.raw_full[slot], raw_phase), &sm.raw_full[slot], raw_phase, abort_flag);
      if (!ok) break;
      const uint32_t src = (src0 + slot * Q4_WORD_BYTES) ^ (half << 5);
      const uint4 q0 = ld_shared16(src), q1 = ld_shared16(src ^ 16);
      uint32_t s01;  // the scales of this row's two halves of 32 k
      if constexpr (NS == 4) {
        s01 = ld_shared4(scale0 + slot * kScaleBytes + 4 * half);
      } else {
        const uint32_t s1 = ld_shared2(scale0 + slot * kScaleBytes + (NS == 2 ? 2 * half : 0));
        s01 = __byte_perm(s1, s1, 0x1010);
      }
      ok = int4_wait<20>(freed, &sm.empty[stage], phase ^ 1, abort_flag);
      if (!ok) break;
      // The loop stays rolled: the roles of this kernel run side by side from
      // one instruction cache, and unrolled they evict one another (the whole
      // block unrolled, three blocks deep: 5464 us against 3421 for the layer
      // of 256 experts at 1024 tokens).
      const uint32_t dst = dst0 + stage * Q4_A_BYTES;
#pragma unroll 1
      for (int c = 0; c < 2; ++c) {  // 32 k: 16 bytes of words, half a row of the stage
        const uint4 q = c ? q1 : q0;
        const uint32_t two = __byte_perm(s01, s01, c ? 0x3232 : 0x1010);
        const uint32_t at = dst ^ (c << 6);
        st_shared16(at, decode_word<T>(q.x, two));
        st_shared16(at ^ 16, decode_word<T>(q.y, two));
        st_shared16(at ^ 32, decode_word<T>(q.z, two));
        st_shared16(at ^ 48, decode_word<T>(q.w, two));
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        ptx::mbar_arrive(&sm.full[stage]);
        // only now: an arrive overtakes shared loads whose values nothing has
        // waited for, and the slot's next words came in under them
        ptx::mbar_arrive(&sm.raw_empty[slot]);
      }
      stage += kSets;
      if (stage >= kStages) {
        stage = set;
        phase ^= 1;
      }
      slot += ((int)kb + kSets) / 2 - (int)kb / 2;
      if (slot >= p.raw) {
        slot -= p.raw;
        raw_phase ^= 1;
      }
    }
    if (!ok) {
      if (lane == 0) raise_device_error(3);
      *abort_flag = 1;
    }
  }

  __syncthreads();
  if (role == kIssue) {
    __syncwarp();
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

template <bool NARROW>
size_t int4_gemm_smem(int raw, int group, int E) {
  using Sh = Int4Shape<NARROW>;
  return 1024 + (size_t)Sh::kStages * (Q4_A_BYTES + Sh::kXBytes) + (size_t)raw * q4_raw_bytes(group) + sizeof(Int4Smem) +
         2 * (size_t)(E + 1) * sizeof(int32_t);
}

template <typename T, int GROUP, bool SWIGLU, bool NARROW>
int launch_int4_gemm(const Int4Maps& maps, Int4Params p, int64_t rows_hit, cudaStream_t st) {
  using Sh = Int4Shape<NARROW>;
  p.raw = Sh::kMaxRaw;
  while (p.raw > Sh::kMinRaw && int4_gemm_smem<NARROW>(p.raw, GROUP, p.E) > (size_t)kMaxSmem) p.raw -= Sh::kRawStep;
  const size_t smem = int4_gemm_smem<NARROW>(p.raw, GROUP, p.E);
  auto kfn = int4_gemm_kernel<T, GROUP, SWIGLU, NARROW>;
  MOE_TRY((allow_smem<int4_gemm_kernel<T, GROUP, SWIGLU, NARROW>>(kMaxSmem)));
  const int64_t items_ub = (ceil_div(p.total_rows, Sh::kRows) + rows_hit) * p.nf;
  const unsigned grid = (unsigned)std::min<int64_t>(num_sms(), items_ub);
  MOE_CUDA_TRY(launch_kernel(kfn, dim3(grid), dim3(Sh::kThreads), smem, st, maps, p));
  MOE_LAUNCH_CHECK("int4_gemm_kernel");
  return MOE_OK;
}

template <typename T, int GROUP>
int launch_int4_shape(bool swiglu, const Int4Maps& maps, const Int4Params& p, int64_t hit, cudaStream_t st) {
  const int64_t narrow_items = (ceil_div(p.total_rows, Int4Shape<true>::kRows) + hit) * p.nf;
  if (p.total_rows <= kInt4NarrowRows * hit || narrow_items <= num_sms())
    return swiglu ? launch_int4_gemm<T, GROUP, true, true>(maps, p, hit, st)
                  : launch_int4_gemm<T, GROUP, false, true>(maps, p, hit, st);
  return swiglu ? launch_int4_gemm<T, GROUP, true, false>(maps, p, hit, st)
                : launch_int4_gemm<T, GROUP, false, false>(maps, p, hit, st);
}

template <typename T>
int launch_int4_group(int group, bool swiglu, const Int4Maps& maps, const Int4Params& p, int64_t hit,
                      cudaStream_t st) {
  if (group == 128) return launch_int4_shape<T, 128>(swiglu, maps, p, hit, st);
  if (group == 64) return launch_int4_shape<T, 64>(swiglu, maps, p, hit, st);
  return launch_int4_shape<T, 32>(swiglu, maps, p, hit, st);
}

// 4-bit words of all experts: boxes of 64 bytes (128 k) by `box_rows` rows.
int make_tmap_words(CUtensorMap* m, const void* ptr, uint64_t row_bytes, uint64_t rows, uint32_t box_rows) {
  cuuint64_t dims[2] = {row_bytes, rows};
  cuuint64_t strides[1] = {row_bytes};
  cuuint32_t box[2] = {(cuuint32_t)Q4_RAW_ROW, box_rows};
  CUresult r;
  MOE_TRY(encode_tiled(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, ptr, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_64B, &r));
  if (r != CUDA_SUCCESS)
    return set_error(MOE_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d) for %llu x %llu 4-bit words", (int)r,
                     (unsigned long long)rows, (unsigned long long)row_bytes);
  return MOE_OK;
}

}  // namespace

bool int4_gemm_fits(int64_t rows, int64_t n_out, int64_t w_rows, int E) {
  const int64_t items = (ceil_div(rows, Int4Shape<true>::kRows) + E) * ceil_div(n_out, Q4_FEAT / 2);
  return rows < (int64_t(1) << 31) - 256 && (int64_t)E * w_rows < (int64_t(1) << 31) - 256 &&
         items < (int64_t(1) << 31) - 65536;
}

int int4_gemm(const void* x, int dtype, int64_t rows, int64_t k, const uint8_t* w, const void* scale, int group, int E,
              int64_t n_out, bool swiglu, const void* counts, int counts_is64, void* out, bool out_f32,
              cudaStream_t st) {
  const int64_t w_rows = swiglu ? 2 * n_out : n_out;
  const int64_t hit = std::min<int64_t>(E, rows);
  Int4Maps maps;
  MOE_TRY(make_tmap_words(&maps.w, w, (uint64_t)k / 2, (uint64_t)E * w_rows, swiglu ? Q4_FEAT / 2 : Q4_FEAT));
  for (int b = 0; b < Q4_BOXES; ++b)
    MOE_TRY(make_tmap(&maps.x[b], x, dtype, (uint64_t)k, (uint64_t)rows, 16u << b));
  Int4Params p{};
  p.E = E;
  p.K = (int)k;
  p.n_out = (int)n_out;
  p.nf = (int)ceil_div(n_out, swiglu ? Q4_FEAT / 2 : Q4_FEAT);
  p.w_rows = (int)w_rows;
  p.scale = scale;
  p.counts = counts;
  p.counts_is64 = counts_is64;
  p.total_rows = rows;
  p.out = out;
  p.out_f32 = out_f32;
  p.idesc_m = make_idesc(dtype, Q4_FEAT) & ~(0x3Fu << 17);
  if (dtype == MOE_BF16) return launch_int4_group<__nv_bfloat16>(group, swiglu, maps, p, hit, st);
  return launch_int4_group<__half>(group, swiglu, maps, p, hit, st);
}

}  // namespace moe
