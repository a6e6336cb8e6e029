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
// cores take 16-bit operands: eight or twelve warps turn the 4-bit words into
// (q - 8) s in shared memory while earlier blocks multiply. A weight is
// rounded to the activations' type there, by at most half a step: scaling
// after the product instead would read the accumulator once for every group.
//
// Roles (one CTA per SM, persistent):
//   warp 0        rows of x: TMA, 64 k by up to 256 rows a block, one or two
//                 boxes whose heights are powers of two
//   warp 1        TMEM, MMA issue into one of two accumulators
//   warp 2        4-bit words: TMA, 128 k by 128 weight rows a block
//   warps 3..6    epilogue
//   warps 7..     decoding: two or three sets of four warps take the blocks of
//                 words in turn, a thread to a weight row
// With SWIGLU a tile's rows alternate between 16 gate rows and the 16 up rows
// that go with them, so gate and up of a feature sit sixteen TMEM lanes apart
// in one warp, and a shuffle for every two tokens brings them together.
#include "int4.cuh"

namespace moe {
namespace {

constexpr int Q4_FIRST = 7;              // first decoding warp
constexpr int Q4_MAX_SETS = 3;           // sets of four decoding warps
constexpr int Q4_THREADS = 32 * (Q4_FIRST + 4 * Q4_MAX_SETS);
constexpr int Q4_FEAT = 128;             // weight rows of a tile (UMMA M)
constexpr int Q4_KB = 64;                // k of an MMA block (128 bytes of 16-bit type)
constexpr int Q4_RAW_ROW = 64;           // bytes of 4-bit words in a block of 128 k
constexpr uint32_t Q4_RAW_BYTES = Q4_FEAT * Q4_RAW_ROW;
constexpr uint32_t Q4_A_BYTES = Q4_FEAT * ROW_BYTES;
constexpr int Q4_MAX_STAGES = 6, Q4_MAX_RAW = 9;
constexpr int Q4_BOXES = 5;              // boxes of 16, 32, 64, 128 and 256 rows of x

// Rows of x of a tile and pipeline stages. Wide tiles for many rows an expert;
// narrow ones, with more stages, where the launch is bound by the weights.
//
// A wait on a barrier's parity cannot tell use u of a stage from use u - 2, so
// no set may come to a use before use u - 2 is over for certain. A set that
// has filled a stage has seen the stage's last use freed, and stages are freed
// in order; from the last stage of its last block to the first of its next lie
// at most 2 sets - 1 stages, so sets <= stages / 2 keeps it within one round.
// Words come in any order: raw is a multiple of sets, so the use before the
// one that a set waits for was its own.
struct Int4Shape {
  int nmax;    // rows of x of a tile at most (UMMA N, at most 256)
  int stages;  // blocks of decoded weights and rows of x
  int raw;     // blocks of words
  int sets;    // sets of decoding warps
};
constexpr bool shape_ok(const Int4Shape& s) {
  return s.sets <= Q4_MAX_SETS && s.stages <= Q4_MAX_STAGES && s.raw <= Q4_MAX_RAW && 2 * s.nmax <= TMEM_COLS &&
         2 * s.sets <= s.stages && s.raw % s.sets == 0;
}
constexpr Int4Shape kInt4Wide{256, 4, 4, 2}, kInt4WideManyExperts{256, 4, 2, 2}, kInt4Narrow{64, 6, 9, 3};
static_assert(shape_ok(kInt4Wide) && shape_ok(kInt4WideManyExperts) && shape_ok(kInt4Narrow), "ring depths");
constexpr size_t kMaxSmem = 227 * 1024;
constexpr int64_t kInt4NarrowRows = 48;  // narrow tiles up to this many rows an expert on average

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
  Int4Shape shape;
};

// A place in a ring of barriers.
struct Ring {
  int i = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void advance(int n, int size) {
    i += n;
    while (i >= size) {
      i -= size;
      phase ^= 1;
    }
  }
};

struct Int4Smem {
  uint64_t raw_full[Q4_MAX_RAW], raw_empty[Q4_MAX_RAW], full[Q4_MAX_STAGES], empty[Q4_MAX_STAGES];
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
    r[b] = Decode<T>::value((t & 0x000f000fu) | Decode<T>::kMagic, s2);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

template <typename T, int GROUP, bool SWIGLU>
__global__ void __launch_bounds__(Q4_THREADS, 1) int4_gemm_kernel(const __grid_constant__ Int4Maps maps,
                                                                  const Int4Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int stages = p.shape.stages, raws = p.shape.raw, nmax = p.shape.nmax;
  const uint32_t x_bytes = (uint32_t)nmax * ROW_BYTES;
  uint8_t* sA = smem;
  uint8_t* sX = sA + stages * Q4_A_BYTES;
  uint8_t* sR = sX + stages * x_bytes;
  Int4Smem& sm = *reinterpret_cast<Int4Smem*>(sR + raws * Q4_RAW_BYTES);
  int32_t* s_off = reinterpret_cast<int32_t*>(&sm + 1);  // [E + 1] first row of each expert
  int32_t* s_cum = s_off + p.E + 1;                      // [E + 1] row tiles before each expert
  volatile int* abort_flag = &sm.abort_flag;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int E = p.E;
  if (threadIdx.x == 0) {
    for (int i = 0; i < raws; ++i) {
      ptx::mbar_init(&sm.raw_full[i], 1);
      ptx::mbar_init(&sm.raw_empty[i], 4);  // the warps of a set
    }
    for (int i = 0; i < stages; ++i) {
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
  if (warp == 2) {
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
      tiles += (int)((end - first + nmax - 1) / nmax);
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
      trun += (s_off[e + 1] - s_off[e] + nmax - 1) / nmax;
    }
    if (lane == 31) s_cum[E] = tincl;
  }
  if (warp == 1) {
    ptx::tmem_alloc(&sm.tmem_slot, TMEM_COLS);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = sm.tmem_slot;
  const int total = s_cum[E] * p.nf;
  const int nkb = (p.K + Q4_KB - 1) / Q4_KB;          // MMA blocks of 64 k
  const int nraw = (p.K + 2 * Q4_KB - 1) / (2 * Q4_KB);  // word blocks of 128 k

  if (warp == 0) {
    // ------------------------------------------------------------ rows of x
    Ring ring;
    int filled = 0;
    bool ok = true;
    for (int item = blockIdx.x; ok && item < total; item += gridDim.x) {
      const Int4Item it = int4_item(item, s_cum, s_off, E, p.nf);
      // one box of at least the rows, or two where that would load a third too many
      const int up = it.rows <= 16 ? 4 : 32 - __clz(it.rows - 1);  // 2^up >= rows
      const bool two = 4 * it.rows <= 3 << up && up > 5;
      const int h0 = two ? up - 1 : up;
      const int rest = it.rows - (1 << h0);
      const int h1 = rest <= 16 ? 4 : 32 - __clz(rest - 1);
      const uint32_t bytes = ((1u << h0) + (two ? 1u << h1 : 0u)) * ROW_BYTES;
      const CUtensorMap* m0 = &maps.x[h0 - 4];
      const CUtensorMap* m1 = &maps.x[h1 - 4];
      for (int kb = 0; kb < nkb; ++kb) {
        ok = __all_sync(0xffffffffu, ptx::mbar_wait(&sm.empty[ring.i], ring.phase ^ 1, abort_flag));
        if (!ok) break;
        if (ptx::elect_one()) {
          uint64_t* bar = &sm.full[ring.i];
          uint8_t* dst = sX + ring.i * x_bytes;
          ptx::mbar_arrive_expect_tx(bar, bytes);
          ptx::tma_load_2d(dst, m0, bar, kb * Q4_KB, (int32_t)it.row);
          if (two) ptx::tma_load_2d(dst + (ROW_BYTES << h0), m1, bar, kb * Q4_KB, (int32_t)it.row + (1 << h0));
        }
        __syncwarp();
        ring.advance(1, stages);
        filled = min(filled + 1, stages);
      }
    }
    if (!ok && lane == 0) {
      raise_device_error(1);
      *abort_flag = 1;
      // copies in flight land before the CTA exits: the stages filled last, newest first
      volatile int never = 0;
      for (; filled > 0; --filled) {
        ring.i = ring.i == 0 ? stages - 1 : ring.i - 1;
        if (ring.i == stages - 1) ring.phase ^= 1;
        ptx::mbar_wait(&sm.full[ring.i], ring.phase, &never);
      }
    }
    __syncwarp();
  } else if (warp == 2) {
    // ------------------------------------------------------------ 4-bit words
    Ring ring;
    int filled = 0;
    bool ok = true;
    for (int item = blockIdx.x; ok && item < total; item += gridDim.x) {
      const Int4Item it = int4_item(item, s_cum, s_off, E, p.nf);
      const int wrow = it.e * p.w_rows + it.f * (SWIGLU ? Q4_FEAT / 2 : Q4_FEAT);
      for (int kb = 0; kb < nraw; ++kb) {
        ok = __all_sync(0xffffffffu, ptx::mbar_wait(&sm.raw_empty[ring.i], ring.phase ^ 1, abort_flag));
        if (!ok) break;
        if (ptx::elect_one()) {
          uint64_t* bar = &sm.raw_full[ring.i];
          uint8_t* dst = sR + ring.i * Q4_RAW_BYTES;
          ptx::mbar_arrive_expect_tx(bar, Q4_RAW_BYTES);
          ptx::tma_load_2d(dst, &maps.w, bar, kb * Q4_RAW_ROW, wrow);
          if constexpr (SWIGLU)
            ptx::tma_load_2d(dst + Q4_RAW_BYTES / 2, &maps.w, bar, kb * Q4_RAW_ROW, wrow + p.n_out);
        }
        __syncwarp();
        ring.advance(1, raws);
        filled = min(filled + 1, raws);
      }
    }
    if (!ok && lane == 0) {
      raise_device_error(1);
      *abort_flag = 1;
      volatile int never = 0;
      for (; filled > 0; --filled) {
        ring.i = ring.i == 0 ? raws - 1 : ring.i - 1;
        if (ring.i == raws - 1) ring.phase ^= 1;
        ptx::mbar_wait(&sm.raw_full[ring.i], ring.phase, &never);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    // The whole warp runs the loop and one lane issues: descriptors stay in
    // uniform registers. Issued from a single-lane branch the four MMAs of a
    // block took 350 cycles to issue, which bound the launch.
    Ring ring;
    int n = 0;
    bool ok = true;
    const uint64_t a_desc = ptx::smem_desc_k128(ptx::smem_u32(sA)), x_desc = ptx::smem_desc_k128(ptx::smem_u32(sX));
    for (int item = blockIdx.x; ok && item < total; item += gridDim.x, ++n) {
      const Int4Item it = int4_item(item, s_cum, s_off, E, p.nf);
      const int buf = n & 1;
      ok = __all_sync(0xffffffffu, ptx::mbar_wait(&sm.tempty[buf], ((n >> 1) & 1) ^ 1, abort_flag));
      if (!ok) break;
      ptx::tc_fence_after();
      const uint32_t idesc = p.idesc_m | ((uint32_t)((it.rows + 15) / 16 * 2) << 17);
      const uint32_t d = tmem_base + (uint32_t)(buf * nmax);
      for (int kb = 0; kb < nkb; ++kb) {
        ok = __all_sync(0xffffffffu, ptx::mbar_wait(&sm.full[ring.i], ring.phase, abort_flag));
        if (!ok) break;
        ptx::tc_fence_after();
        const uint64_t ad = a_desc + (uint64_t)(ring.i * (Q4_A_BYTES >> 4));
        const uint64_t xd = x_desc + (uint64_t)(ring.i * (x_bytes >> 4));
        if (ptx::elect_one()) {
#pragma unroll
          for (int k = 0; k < ROW_BYTES / 32; ++k)
            ptx::umma<0>(d, ad + 2 * k, xd + 2 * k, idesc, (kb > 0 || k > 0) ? 1u : 0u);
          ptx::umma_commit(&sm.empty[ring.i]);
          if (kb == nkb - 1) ptx::umma_commit(&sm.tfull[buf]);
        }
        __syncwarp();
        ring.advance(1, stages);
      }
    }
    if (!ok && lane == 0) {
      raise_device_error(2);
      *abort_flag = 1;
    }
    if (ptx::elect_one()) {
      ptx::umma_commit(&sm.drain);  // all MMAs complete before TMEM is released
      volatile int never = 0;
      if (!ptx::mbar_wait(&sm.drain, 0, &never)) raise_device_error(4);
    }
    __syncwarp();
  } else if (warp < Q4_FIRST) {
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3;  // TMEM lanes 32 q .. 32 q + 31
    bool ok = true;
    int n = 0;
    for (int item = blockIdx.x; item < total; item += gridDim.x, ++n) {
      const Int4Item it = int4_item(item, s_cum, s_off, E, p.nf);
      const int buf = n & 1;
      const bool w_ok = ptx::mbar_wait(&sm.tfull[buf], (n >> 1) & 1, abort_flag);
      if (!__all_sync(0xffffffffu, w_ok)) {
        ok = false;
        break;
      }
      ptx::tc_fence_after();
      const uint32_t tbase = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * nmax);
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
    for (int64_t i = n0 + (int64_t)blockIdx.x * 128 + (warp - 3) * 32 + lane; i < n1; i += (int64_t)gridDim.x * 128) {
      if (p.out_f32) static_cast<float*>(p.out)[i] = 0.f;
      else static_cast<uint16_t*>(p.out)[i] = 0;
    }
  } else {
    // ------------------------------------------------------------ decoding
    const int set = (warp - Q4_FIRST) >> 2;
    const int r = ((warp - Q4_FIRST) & 3) * 32 + lane;  // row of the tile
    // its row of the word block (gate rows first, then up rows)
    const int rr = SWIGLU ? ((r & 16) ? Q4_FEAT / 2 : 0) + (r >> 5) * 16 + (r & 15) : r;
    constexpr int NS = 128 / GROUP;  // groups of a block of words
    const int groups = p.K / GROUP;
    // this set's blocks of words: every sets-th of the run of all blocks
    struct Walk {
      int item, kb;
      __device__ __forceinline__ bool step(int n, int nraw) {  // true: another item
        kb += n;
        bool moved = false;
        while (kb >= nraw) {
          kb -= nraw;
          item += gridDim.x;
          moved = true;
        }
        return moved;
      }
    };
    auto scale_row = [&](int item) -> const T* {
      if (item >= total) return nullptr;
      const Int4Item it = int4_item(item, s_cum, s_off, E, p.nf);
      int wr;
      if (SWIGLU)
        wr = min(it.f * (Q4_FEAT / 2) + (r >> 5) * 16 + (r & 15), p.n_out - 1) + ((r & 16) ? p.n_out : 0);
      else
        wr = min(it.f * Q4_FEAT + r, p.n_out - 1);
      return static_cast<const T*>(p.scale) + ((int64_t)it.e * p.w_rows + wr) * groups;
    };
    // scales are read two of this set's blocks ahead; groups past K are 0
    auto load_scales = [&](const T* row, int kb, T (&s)[NS]) {
#pragma unroll
      for (int j = 0; j < NS; ++j) {
        const int g = kb * NS + j;
        s[j] = row != nullptr && g < groups ? row[g] : u4::Act<T>::from_float(0.f);
      }
    };
    Walk cur{(int)blockIdx.x, 0}, ahead;
    cur.step(set, nraw);
    ahead = cur;
    const int sets = p.shape.sets;
    T s0[NS], s1[NS], s2[NS];
    const T* row = scale_row(ahead.item);
    load_scales(row, ahead.kb, s0);
    if (ahead.step(sets, nraw)) row = scale_row(ahead.item);
    load_scales(row, ahead.kb, s1);
    Ring raw, ring;
    raw.advance(set, raws);
    // MMA blocks before this set's first block
    ring.advance((cur.item - (int)blockIdx.x) / (int)gridDim.x * nkb + 2 * cur.kb, stages);
    bool ok = true;
    while (ok && cur.item < total) {
      if (ahead.step(sets, nraw)) row = scale_row(ahead.item);
      load_scales(row, ahead.kb, s2);
      ok = ptx::mbar_wait(&sm.raw_full[raw.i], raw.phase, abort_flag);
      uint4 w[4];
      const uint8_t* src = sR + raw.i * Q4_RAW_BYTES + rr * Q4_RAW_ROW;
      if (ok)
#pragma unroll
        for (int c = 0; c < 4; ++c) w[c] = *reinterpret_cast<const uint4*>(src + ((c ^ ((rr >> 1) & 3)) << 4));
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&sm.raw_empty[raw.i]);
      raw.advance(sets, raws);
      const int halves = min(2, nkb - 2 * cur.kb);  // the last block may have one half
      Ring at = ring;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (h >= halves) break;
        ok = ok && ptx::mbar_wait(&sm.empty[at.i], at.phase ^ 1, abort_flag);
        if (ok) {
          uint8_t* dst = sA + at.i * Q4_A_BYTES + r * ROW_BYTES;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const T s = s0[(2 * h + c) * NS / 4];
            const uint32_t one = *reinterpret_cast<const uint16_t*>(&s);
            const uint4 q = w[2 * h + c];
            const uint32_t words[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int k = 0; k < 4; ++k)
              *reinterpret_cast<uint4*>(dst + (((4 * c + k) ^ (r & 7)) << 4)) =
                  decode_word<T>(words[k], one | (one << 16));
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&sm.full[at.i]);
        at.advance(1, stages);
      }
      ok = __all_sync(0xffffffffu, ok);
#pragma unroll
      for (int j = 0; j < NS; ++j) {
        s0[j] = s1[j];
        s1[j] = s2[j];
      }
      const Walk was = cur;
      cur.step(sets, nraw);
      ring.advance((cur.item - was.item) / (int)gridDim.x * nkb + 2 * (cur.kb - was.kb), stages);
    }
    if (!ok) {
      if (lane == 0) raise_device_error(3);
      *abort_flag = 1;
    }
  }

  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

size_t int4_gemm_smem(const Int4Shape& s, int E) {
  return 1024 + (size_t)s.stages * (Q4_A_BYTES + s.nmax * ROW_BYTES) + (size_t)s.raw * Q4_RAW_BYTES +
         sizeof(Int4Smem) + 2 * (size_t)(E + 1) * sizeof(int32_t);
}

template <typename T, int GROUP, bool SWIGLU>
int launch_int4_gemm(const Int4Maps& maps, const Int4Params& p, int64_t items_ub, cudaStream_t st) {
  const size_t smem = int4_gemm_smem(p.shape, p.E);
  auto kfn = int4_gemm_kernel<T, GROUP, SWIGLU>;
  MOE_CUDA_TRY(cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  const unsigned grid = (unsigned)std::min<int64_t>(num_sms(), items_ub);
  MOE_CUDA_TRY(launch_kernel(kfn, dim3(grid), dim3(32 * (Q4_FIRST + 4 * p.shape.sets)), smem, st, maps, p));
  MOE_LAUNCH_CHECK("int4_gemm_kernel");
  return MOE_OK;
}

template <typename T, bool SWIGLU>
int launch_int4_group(int group, const Int4Maps& maps, const Int4Params& p, int64_t items_ub, cudaStream_t st) {
  if (group == 128) return launch_int4_gemm<T, 128, SWIGLU>(maps, p, items_ub, st);
  if (group == 64) return launch_int4_gemm<T, 64, SWIGLU>(maps, p, items_ub, st);
  return launch_int4_gemm<T, 32, SWIGLU>(maps, p, items_ub, st);
}

// 4-bit words of all experts: boxes of 64 bytes (128 k) by `box_rows` rows.
int make_tmap_words(CUtensorMap* m, const void* ptr, uint64_t row_bytes, uint64_t rows, uint32_t box_rows) {
  EncodeTiledFn enc;
  MOE_TRY(get_encode(&enc));
  cuuint64_t dims[2] = {row_bytes, rows};
  cuuint64_t strides[1] = {row_bytes};
  cuuint32_t box[2] = {(cuuint32_t)Q4_RAW_ROW, box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return set_error(MOE_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d) for %llu x %llu 4-bit words", (int)r,
                     (unsigned long long)rows, (unsigned long long)row_bytes);
  return MOE_OK;
}

}  // namespace

bool int4_gemm_fits(int64_t rows, int64_t n_out, int64_t w_rows, int E) {
  const int64_t items = (ceil_div(rows, kInt4Narrow.nmax) + E) * ceil_div(n_out, Q4_FEAT / 2);
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
  p.shape = rows <= kInt4NarrowRows * hit ? kInt4Narrow : kInt4Wide;
  if (int4_gemm_smem(p.shape, E) > kMaxSmem) p.shape = kInt4WideManyExperts;
  const int64_t items_ub = (ceil_div(rows, p.shape.nmax) + hit) * p.nf;
  if (dtype == MOE_BF16)
    return swiglu ? launch_int4_group<__nv_bfloat16, true>(group, maps, p, items_ub, st)
                  : launch_int4_group<__nv_bfloat16, false>(group, maps, p, items_ub, st);
  return swiglu ? launch_int4_group<__half, true>(group, maps, p, items_ub, st)
                : launch_int4_group<__half, false>(group, maps, p, items_ub, st);
}

}  // namespace moe
