// What the attention kernels share (attention_kernels.hip over contiguous keys and
// values, paged_attention_kernels.hip over pages): matrix operands, tiles in LDS and the
// online softmax of a wave's rows.
//
// The products run on the matrix cores in 32x32 tiles (v_mfma_f32_32x32x16 for
// bf16, eight v_mfma_f32_32x32x2 for fp32), everything else in fp32.  A wave
// always forms the score tile with its own rows along the lanes: in the 32x32 result layout a
// lane holds one column and the rows 8a + 4h + b (a, b = 0..3, h = lane / 32),
// so the row statistics are a reduction over a lane's own registers and one
// exchange between lane halves.  The same registers are the next product's
// B operand as they stand: its 16-long k axis takes the rows in the order
// (h, j) -> 16 s + 8 (j / 4) + 4h + j % 4 that the lane already holds, and the
// A operand is read from LDS in that order (for bf16 with the transposing
// ds_read_b64_tr_b16: four rows of one column per lane), so probabilities
// never cross lanes or go through LDS.
//
// Tiles go from HBM to LDS directly (global_load_lds, 16 bytes per lane).  A tile row is held
// as 16-byte chunks, chunk c of row r at place c ^ g(r) with
// g = 2 (r % 8) + (r / 8) % 2 (rows of 8 chunks: 2 (r % 8 / 2) + (r / 8) % 2): 16
// rows of one chunk fall on distinct banks, so the row reads of a tile are free
// of conflicts, and so are fp32's column reads.  bf16's transposed reads are not:
// 32 lanes read four chunks of each of four rows, and rows r and r + 1 (r even)
// lie 32 bytes apart there, so that half of their chunks share banks.  Each
// such read takes two cycles more than it needs.
#ifndef KOTODAMA_AMD_ATTENTION_TILES_H
#define KOTODAMA_AMD_ATTENTION_TILES_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "lm_params.h"

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

#define LM_LDS __attribute__((address_space(3)))
#define LM_GLOBAL __attribute__((address_space(1)))

namespace {

constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kNegInf = -__builtin_inff();

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  bf16x2 r = {(__bf16)lo, (__bf16)hi};
  return __builtin_bit_cast(uint32_t, r);
}
__device__ __forceinline__ float bf_lo(uint32_t u) { return __builtin_bit_cast(float, u << 16); }
__device__ __forceinline__ float bf_hi(uint32_t u) { return __builtin_bit_cast(float, u & 0xffff0000u); }

// 2^x; v_exp_f32 gives 0 for -inf and flushes results under 2^-126.
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// The value of the lane 32 away.
__device__ __forceinline__ float other_half(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(((int)(threadIdx.x & 63) ^ 32) << 2,
                                                                __builtin_bit_cast(int, v)));
}

// ------------------------------------------------------------- fragments --
//
// Frag<T>: eight elements of an operand along k: A row (or B column) lane % 32,
// k = 8 (lane / 32) + j of a 16-long step.

struct Bf16 {
  static constexpr int kBytes = 2;
  struct Frag {
    u32x4 w;
  };
  static __device__ __forceinline__ f32x16 mma(const Frag& a, const Frag& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a.w), __builtin_bit_cast(bf16x8, b.w),
                                                   c, 0, 0, 0);
  }
  static __device__ __forceinline__ Frag zero() { return Frag{u32x4{0, 0, 0, 0}}; }
  static __device__ __forceinline__ Frag load(const char* p) { return Frag{*reinterpret_cast<const u32x4*>(p)}; }
  // Registers 8s .. 8s+7 of a result tile as the B operand of step s.  Rounded:
  // probabilities and score gradients are held in fp32 up to here, but the
  // matrix instructions take both operands in one type, and in fp32 they run at
  // a sixteenth of bf16's rate.  With this rounding (and delta's,
  // see attention_bwd_dq) results are off by 2.0e-3 to 2.4e-3 of their norm,
  // against 1.7e-3 for 32-bit products rounded once at the end.
  static __device__ __forceinline__ Frag from_acc(const f32x16& c, int s) {
    Frag f;
#pragma unroll
    for (int i = 0; i < 4; ++i) f.w[i] = pack_bf16(c[8 * s + 2 * i], c[8 * s + 2 * i + 1]);
    return f;
  }
  static __device__ __forceinline__ float get(const Frag& f, int j) {
    return (j & 1) ? bf_hi(f.w[j >> 1]) : bf_lo(f.w[j >> 1]);
  }
};

struct F32 {
  static constexpr int kBytes = 4;
  struct Frag {
    f32x4 lo, hi;
  };
  static __device__ __forceinline__ f32x16 mma(const Frag& a, const Frag& b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.lo[j], b.lo[j], c, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.hi[j], b.hi[j], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ Frag zero() { return Frag{f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}}; }
  static __device__ __forceinline__ Frag load(const char* p) {
    return Frag{*reinterpret_cast<const f32x4*>(p), *reinterpret_cast<const f32x4*>(p + 16)};
  }
  static __device__ __forceinline__ Frag from_acc(const f32x16& c, int s) {
    Frag f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f.lo[i] = c[8 * s + i];
      f.hi[i] = c[8 * s + 4 + i];
    }
    return f;
  }
  static __device__ __forceinline__ float get(const Frag& f, int j) { return j < 4 ? f.lo[j] : f.hi[j - 4]; }
};

// ------------------------------------------------------------- LDS tiles --

// A tile of R rows of DP elements in LDS (layout in the head comment), loaded
// by WAVES waves.
template <typename T, int DP, int R, int WAVES = LM_ATTN_WAVES>
struct Tile {
  static constexpr int kRowBytes = DP * T::kBytes;
  static constexpr int kChunks = kRowBytes / 16;  // per row
  static constexpr int kRows = R;
  static constexpr int kBytes = R * kRowBytes;

  static __device__ __forceinline__ int place(int row) {
    if constexpr (kChunks >= 16) return ((row << 1) & 14) | ((row >> 3) & 1);
    return ((row & 6) | ((row >> 3) & 1));  // 8 chunks: row r and r + 1 share 256 bytes
  }

  using Mine = Tile<T, DP, 32, 1>;  // 32 of its rows, loaded by the wave that reads them
  // Round i, of kRound rows, is one wave-wide load per wave.
  static constexpr int kRound = WAVES * 64 / kChunks;
  static constexpr int kRounds = R / kRound;
  static_assert(kRounds * kRound == R, "whole rounds");

  // This lane's row within a round, and the offset within the round of its part.
  static __device__ __forceinline__ int round_row(int wave, int lane) { return (wave * 64 + lane) / kChunks; }
  static __device__ __forceinline__ uint32_t chunk_offset(int round, int wave, int lane, int chunks) {
    const int c = (lane % kChunks) ^ place(round * kRound + round_row(wave, lane));
    return 16 * (uint32_t)(c < chunks ? c : chunks - 1);  // chunks past the row's end repeat its last
  }

  // Request rows row0 .. row0+R-1 of `src` into `lds`.  Rows past `last` (at
  // least row0) repeat it.  The base is uniform and the offset 32 bits wide; the
  // places of rows 16 apart are the same, so that rounds of 16 rows or more
  // share one offset.
  static __device__ __forceinline__ void request(char* lds, const char* src, int64_t stride, int row0, int last,
                                                 int chunks, int wave, int lane) {
    const char* base = src + (int64_t)row0 * stride;
    if (row0 + R - 1 <= last) {
      const uint32_t row = (uint32_t)round_row(wave, lane) * (uint32_t)stride;
#pragma unroll
      for (int i = 0; i < kRounds; ++i)
        load_lds(lds + (i * WAVES + wave) * 1024, base + (int64_t)(i * kRound) * stride,
                 row + chunk_offset(i, wave, lane, chunks));
    } else {
#pragma unroll
      for (int i = 0; i < kRounds; ++i) {
        int row = i * kRound + round_row(wave, lane);
        row = row < last - row0 ? row : last - row0;
        load_lds(lds + (i * WAVES + wave) * 1024, base,
                 (uint32_t)row * (uint32_t)stride + chunk_offset(i, wave, lane, chunks));
      }
    }
  }
  static __device__ __forceinline__ void load_lds(char* lds, const char* base, uint32_t off) {
    __builtin_amdgcn_global_load_lds((const LM_GLOBAL void*)(base + off), (LM_LDS void*)lds, 16, 0, 0);
  }

  // Lane offsets of the reads below.  A step's or a column block's place in the
  // tile differs from the first's by an exclusive or, and rows 16 further down
  // by a constant, so one offset serves a whole tile.
  static __device__ __forceinline__ int row_at(int lane) {
    const int row = lane & 31, h = lane >> 5;
    return row * kRowBytes + (((T::kBytes == 2 ? h : 2 * h) ^ place(row)) << 4);
  }
  static __device__ __forceinline__ int col_at(int lane) {
    const int h = lane >> 5;
    if constexpr (T::kBytes == 2) {
      const int s = lane & 15;
      const int r = 4 * h + (s >> 2);
      const int c = 2 * ((lane >> 4) & 1) + ((s & 3) >> 1);
      return r * kRowBytes + ((c ^ place(r)) << 4) + ((s & 1) << 3);
    } else {
      const int d = lane & 31;
      return 4 * h * kRowBytes + ((d >> 2) << 4) + ((d & 3) << 2);
    }
  }

  // Row row0 + lane % 32 (row0 a multiple of 32), elements 16 step + 8h .. + 7:
  // an A operand with rows along m.  `at`: row_at(lane).
  static __device__ __forceinline__ typename T::Frag row_frag(const char* lds, int row0, int step, int at) {
    const char* p = lds + row0 * kRowBytes;
    typename T::Frag f;
    if constexpr (T::kBytes == 2) {
      f.w = *reinterpret_cast<const u32x4*>(p + (at ^ (step << 5)));
    } else {
      f.lo = *reinterpret_cast<const f32x4*>(p + (at ^ (step << 6)));
      f.hi = *reinterpret_cast<const f32x4*>(p + (at ^ (step << 6) ^ 16));
    }
    return f;
  }

  // Column 32 dt + lane % 32 over the rows row0 + 8 (j / 4) + 4h + j % 4, j = 0..7 (an A
  // operand with columns along m and a step's 16 rows along k); row0 a multiple of 16.
  // `at`: col_at(lane).
  static __device__ __forceinline__ typename T::Frag col_frag(const char* lds, int row0, int dt, int at, int lane) {
    const char* p = lds + row0 * kRowBytes;
    typename T::Frag f;
    if constexpr (T::kBytes == 2) {
      // rows 8 further down: place() differs in its lowest bit
      const int a = at ^ (dt << 6);
      const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LM_LDS i16x4*)(p + a)));
      const u32x2 hi = __builtin_bit_cast(
          u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LM_LDS i16x4*)(p + 8 * kRowBytes + (a ^ 16))));
      f.w = u32x4{lo[0], lo[1], hi[0], hi[1]};
    } else {
      const int h4 = (lane >> 5) << 2;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int a = at ^ (dt << 7);
        f.lo[j] = *reinterpret_cast<const float*>(p + j * kRowBytes + (a ^ (place(h4 + j) << 4)));
        f.hi[j] = *reinterpret_cast<const float*>(p + (j + 8) * kRowBytes + (a ^ (place(h4 + j + 8) << 4)));
      }
    }
    return f;
  }
};

// A global row as B operands: elements 16 step + 8h .. + 7; zero past `dim` or
// where the row does not exist.
template <typename T, int DC>
__device__ __forceinline__ void load_rows(typename T::Frag (&f)[DC / 16], const char* row, int dim, int h, bool live) {
#pragma unroll
  for (int s = 0; s < DC / 16; ++s) {
    const int d = 16 * s + 8 * h;
    f[s] = (live && d < dim) ? T::load(row + d * T::kBytes) : T::zero();
  }
}

// Four consecutive elements of an output row.
template <typename T>
__device__ __forceinline__ void store4(char* p, float a, float b, float c, float d) {
  if constexpr (T::kBytes == 2) {
    *reinterpret_cast<u32x2*>(p) = u32x2{pack_bf16(a, b), pack_bf16(c, d)};
  } else {
    *reinterpret_cast<f32x4*>(p) = f32x4{a, b, c, d};
  }
}

// A wave's 32 rows x DC result held as its transpose (lane: row lane % 32,
// registers: columns), scaled and stored; only columns under dim.
template <typename T, int DC>
__device__ __forceinline__ void store_rows(char* row, const f32x16 (&acc)[DC / 32], float scale, int dim, int h) {
#pragma unroll
  for (int dt = 0; dt < DC / 32; ++dt) {
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int d = 32 * dt + 8 * a + 4 * h;
      if (d < dim)
        store4<T>(row + d * T::kBytes, acc[dt][4 * a] * scale, acc[dt][4 * a + 1] * scale, acc[dt][4 * a + 2] * scale,
                  acc[dt][4 * a + 3] * scale);
    }
  }
}

// ------------------------------------------------------------- schedules --

// Orders the matrix instructions of the code before it (in its basic block): `ahead` LDS
// reads, then N times one matrix instruction and the next reads, so that a
// product waits for reads requested several products ago.  (Left to itself the
// compiler reads one operand, waits, and multiplies.)  VALU: other vector
// instructions placed behind each of the first VN products.
template <int AHEAD, int N, int READS, int VN, int VALU>
__device__ __forceinline__ void interleave() {
  __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if (AHEAD + (i + 1) * READS <= N * READS) __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    if (i < VN) __builtin_amdgcn_sched_group_barrier(0x002, VALU, 0);
  }
}

__device__ __forceinline__ int64_t index_at(const void* p, int i, int is64) {
  return is64 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}

// Where row `r` of a sequence's key head lies in a (batch, heads, tokens, dim) tensor.
__device__ __forceinline__ int64_t row_offset(const lm_strides& s, int b, int head, int64_t i) {
  return (int64_t)b * s.b + (int64_t)head * s.h + i * s.t;
}

// ---------------------------------------------------------- online softmax --

// The waves that share rows or keys add their results: part 0 receives.  `x`
// holds 64 lanes x DC/2 floats per pair; every wave of the workgroup calls this.
template <int DC>
__device__ __forceinline__ void put(float* x, const f32x16 (&acc)[DC / 32], int lane) {
#pragma unroll
  for (int dt = 0; dt < DC / 32; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) x[(dt * 16 + i) * 64 + lane] = acc[dt][i];
}
template <int DC>
__device__ __forceinline__ void add(const float* x, f32x16 (&acc)[DC / 32], int lane, float mine, float theirs) {
#pragma unroll
  for (int dt = 0; dt < DC / 32; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i)
      acc[dt][i] = __builtin_fmaf(x[(dt * 16 + i) * 64 + lane], theirs, acc[dt][i] * mine);
}

// One tile's part in the online softmax of a wave's 32 rows (along the lanes): NB blocks of 32 keys
// from key `key0`, rows `first` on of the tiles `kc` and `vc`.  m: the reference maximum (of scores
// times log2 e), l: this lane's part of the sum, acc: the result's transpose.  A row sees the keys
// under `lim`, all rows those under `all`.
template <typename T, typename KT, int DC, int NB>
__device__ __forceinline__ void attend(const char* kc, const char* vc, int first, int key0, int all, int lim,
                                       const typename T::Frag (&qf)[DC / 16], f32x16 (&acc)[DC / 32], float& m, float& l,
                                       float scale_log2, int row_at, int col_at, int lane, int h) {
  f32x16 s[NB];
  __builtin_amdgcn_s_setprio(1);
#pragma unroll
  for (int kb = 0; kb < NB; ++kb) {
    s[kb] = zero16();
#pragma unroll
    for (int st = 0; st < DC / 16; ++st)
      s[kb] = T::mma(KT::row_frag(kc, first + 32 * kb, st, row_at), qf[st], s[kb]);
  }
  if constexpr (T::kBytes == 2) interleave<4, NB * DC / 16, 1, 0, 0>();
  __builtin_amdgcn_s_setprio(0);
  if (key0 + 32 * NB > all) {
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = key0 + 32 * kb + 8 * (i >> 2) + 4 * h + (i & 3);
        s[kb][i] = key < lim ? s[kb][i] : kNegInf;
      }
  }
  float top = s[0][0];
#pragma unroll
  for (int kb = 0; kb < NB; ++kb)
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, s[kb][i]);
  top = fmaxf(top, other_half(top)) * scale_log2;
  // The reference only has to be near the maximum: probabilities up to
  // 2^8 are as exact.  Most tiles after the first leave it, and so the
  // accumulators, as they are.
  if (__any(top > m + 8.f)) {
    const float mn = fmaxf(m, top);
    const float fade = mn == kNegInf ? 1.f : exp2_fast(m - mn);
    m = mn;
    l *= fade;
#pragma unroll
    for (int dt = 0; dt < DC / 32; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[dt][i] *= fade;
  }
  const float ref = m == kNegInf ? 0.f : m;
#pragma unroll
  for (int kb = 0; kb < NB; ++kb)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[kb][i] = exp2_fast(__builtin_fmaf(s[kb][i], scale_log2, -ref));
      l += s[kb][i];
    }
#pragma unroll
  for (int kb = 0; kb < NB; ++kb)
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const typename T::Frag p = T::from_acc(s[kb], st);
#pragma unroll
      for (int dt = 0; dt < DC / 32; ++dt)
        acc[dt] = T::mma(KT::col_frag(vc, first + 32 * kb + 16 * st, dt, col_at, lane), p, acc[dt]);
    }
  if constexpr (T::kBytes == 2) interleave<8, NB * DC / 16, 2, (NB == 2 ? DC / 16 : 0), 7>();
}

// Joins the online softmax of the KS waves that share their rows, one part after another to part 0,
// which rescales both to their common maximum.  x: 64 x DC / 2 floats, xm: 128; every wave of the
// workgroup calls this.
template <int DC, int KS>
__device__ __forceinline__ void join_waves(float* x, float* xm, int part, f32x16 (&acc)[DC / 32], float& m, float& l,
                                           int lane) {
#pragma unroll
  for (int o = 1; o < KS; ++o) {
    __syncthreads();
    if (part == o) {
      put<DC>(x, acc, lane);
      xm[lane] = m;
      xm[64 + lane] = l;
    }
    __syncthreads();
    if (part == 0) {
      const float om = xm[lane], ol = xm[64 + lane];
      const float mn = fmaxf(m, om);
      const float a = m == kNegInf ? 0.f : exp2_fast(m - mn), c = om == kNegInf ? 0.f : exp2_fast(om - mn);
      add<DC>(x, acc, lane, a, c);
      l = l * a + ol * c;
      m = mn;
    }
  }
}

}  // namespace

#endif  // KOTODAMA_AMD_ATTENTION_TILES_H
