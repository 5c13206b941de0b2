// Causal attention of a ragged batch over a paged KV cache (keys and values [page, kv head, slot, D], both
// row-major): the step kernel for few rows a sequence, the tile kernel for prompts, both in one launch for a
// prefix that the sequences share, and the joins of their parts. For row t at position p of its sequence,
//   out = sum_j 2^(s_j - m) v_j / l,  m = max_j s_j,  l = sum_j 2^(s_j - m),  p - window < j <= p,
// in one pass over the keys: s in log2 units, m, l and the sums in fp32, moved along when m grows; parts of
// the keys join by the same formula. bf16 rounds each weight 2^(s - m) once, as an operand of the matrix
// cores, and the outputs.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "paged.hpp"

namespace tl {

// A block of a sequence's rows (row r: token r / g, query head r % g of the kv head's), from `row` on, and
// the chunks that they see: chunk0 .. chunk0 + chunks - 1, which lie from `at` on on the line. The sequence's
// tokens begin at row row0 of the batch and at position base; it has n rows.
struct __attribute__((aligned(32))) PagedTile {
  int seq, row, chunk0, chunks, at, row0, base, n;
};

// Where a workgroup's run of the lines begins: at `place` of them all, in block `tile` of kv head `head`.
struct __attribute__((aligned(16))) PagedRun {
  int place, head, tile, unused;
};

struct PagedAttn {
  PagedBatch b;
  const void* q;
  const void* k;
  const void* v;
  void* out;
  int64_t ld_q, ld_out;
  int g;              // query heads of a kv head
  int max_q, window;  // window 0: none
  int shared, skip;   // positions that the sequences share, and those of them that another kernel takes
  float scale;                // of score() to log2 units
  float cap_in;               // of a product to score()'s argument; 0: no cap
  // the step kernel's parts, [slot][group rows]: outputs [D] and (max, sum)
  float* part_o;
  float2* part_ml;
  int workers;
  // the shared prefix: its chunks cut into `splits` for each of row_blocks blocks of the batch's rows
  float* pre_o;
  float2* pre_ml;
  int splits, row_blocks;  // (without a prefix: most blocks of 16 rows that a sequence has)
  // the tile kernel's plan: row blocks of the batch, in order; per kv head they are one line of chunks
  PagedTile* tiles;
  PagedRun* runs;  // [workers + 1]
  int most_tiles;
};

typedef const __attribute__((address_space(4))) int32_t* ConstInts;
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ const void* uniform(const void* p) {
  const uint64_t x = (uint64_t)(uintptr_t)p;
  return (const void*)(((uint64_t)(uint32_t)uniform((int)(x >> 32)) << 32) | (uint32_t)uniform((int)x));
}
__device__ __forceinline__ ConstInts const_ints(const int32_t* p) { return (ConstInts)(uintptr_t)p; }

// ---------------------------------------------------------------------------------------
// keys and values in LDS
// ---------------------------------------------------------------------------------------
// Rows of a chunk lie in LDS one after another as 16-byte pieces. The pieces of a row are permuted by
// an XOR with a number made from the row (applied to the source address of the direct load, which
// writes linearly), so that the lanes that read LDS together meet different banks:
//   keys: 16 lanes read the same piece of 16 rows;
//   values (bf16): 16 lanes read 32 bytes of each of 4 rows, transposed; two such groups a phase.
template <typename T, int D>
struct Rows {
  static constexpr int kVec = 16 / (int)sizeof(T);
  static constexpr int kPieces = D / kVec;        // of a row
  static constexpr int kBytes = D * (int)sizeof(T);
  static constexpr int kPerLoad = 64 / kPieces;   // rows that one direct load of a wave covers
  static_assert(kPieces <= 64 && kPerLoad <= 16, "row size");
  __device__ __forceinline__ static int key_swizzle(int row) {
    return kPieces >= 16 ? row & 15 : (row / (16 / (kPieces < 16 ? kPieces : 16))) & (kPieces - 1);
  }
  __device__ __forceinline__ static int value_swizzle(int row) {
    constexpr int kSegs = kPieces / 2;  // of 32 bytes
    if (sizeof(T) == 4) return 0;
    return 2 * (kSegs >= 8 ? row & 7 : (row / (8 / (kSegs < 8 ? kSegs : 8))) & (kSegs - 1));
  }
};

// N direct loads of a wave, 16 bytes a lane each: load i takes base + 1024 i + offset[i] (per lane) to LDS at
// lds + 1024 i + 16 lane (the instruction's offset counts on both sides). M0 holds the LDS address; it must
// have been written one wait state before it is used.
template <int N>
__device__ __forceinline__ void dma_load16_rows(const void* base, const uint32_t* offset, uint32_t lds) {
  static_assert(N == 1 || N == 2 || N == 4, "loads at a time");
  uint32_t saved;
  if constexpr (N == 1)
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %3, %2\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(saved)
        : "s"(lds), "s"(base), "v"(offset[0])
        : "memory");
  else if constexpr (N == 2)
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %3, %2\n\t"
        "global_load_lds_dwordx4 %4, %2 offset:1024\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(saved)
        : "s"(lds), "s"(base), "v"(offset[0]), "v"(offset[1])
        : "memory");
  else
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %3, %2\n\t"
        "global_load_lds_dwordx4 %4, %2 offset:1024\n\t"
        "global_load_lds_dwordx4 %5, %2 offset:2048\n\t"
        "global_load_lds_dwordx4 %6, %2 offset:3072\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(saved)
        : "s"(lds), "s"(base), "v"(offset[0]), "v"(offset[1]), "v"(offset[2]), "v"(offset[3])
        : "memory");
}
// Waits until at most n direct loads of the wave are in flight (n is uniform, a multiple of STEP).
template <int STEP, int MOST>
__device__ __forceinline__ void wait_loads(int n) {
  if constexpr (MOST == 0) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  } else {
    if (n >= MOST) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(MOST) : "memory");
    else wait_loads<STEP, MOST - STEP>(n);
  }
}

// Queues the 16 rows of one 16-position block of a page (uniform address) to LDS.
template <typename T, int D, bool KEYS>
__device__ __forceinline__ void load_block16(const void* src, uint32_t lds, int lane) {
  using R = Rows<T, D>;
  constexpr int kLoads = 16 / R::kPerLoad, N = kLoads < 4 ? kLoads : 4;
  const int rr = lane / R::kPieces, c = lane % R::kPieces;
#pragma unroll
  for (int i = 0; i < kLoads; i += N) {
    uint32_t offset[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int row = (i + k) * R::kPerLoad + rr;
      offset[k] = (uint32_t)(rr * R::kBytes + ((c ^ (KEYS ? R::key_swizzle(row) : R::value_swizzle(row))) << 4));
    }
    dma_load16_rows<N>((const unsigned char*)src + i * 1024, offset, lds + i * 1024);
  }
}

// ---------------------------------------------------------------------------------------
// tile arithmetic: 16 rows of queries (columns of S^T and O^T) by 16-key tiles
// ---------------------------------------------------------------------------------------
// S^T = K Q^T: lane l of the wave holds the scores of query row l % 16 at keys 16 j + 4 (l / 16) + r.
// O^T += V^T P^T takes those probabilities as its B operand where they are: bf16, 32 keys a step, in
// the key order that the lanes hold; fp32, 4 keys a step, one of each lane group.
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

template <typename T, int D>
struct Tile16 {
  using R = Rows<T, D>;
  static constexpr bool kBf = sizeof(T) == 2;
  static constexpr int KS = R::kPieces / 4;          // steps of 4 pieces over D
  static constexpr int DT = D / 16;                  // output tiles
  static constexpr int E = DT < 4 ? DT : 4;          // fp32: consecutive outputs that one read feeds

  // Scores of KT tiles of 16 keys of a chunk against RG groups of 16 queries: q[group][KS] to
  // s[tile][group]. The reads of a few fragments run ahead of the products that take them.
  template <int KT, int RG>
  __device__ __forceinline__ static void scores(const unsigned char* keys, const uint4* q, f32x4* s, int fr, int fg) {
    const int sw = R::key_swizzle(fr);
    // fp32: a sum of D products in up to 4 chains of 32 or 64, whose roundings are smaller than those of one
    // (D 256, 54 to 326 keys: outputs off by 3.0e-7, 1.2e-6 in one)
    constexpr int C = kBf || D == 32 ? 1 : D == 64 ? 2 : 4;
    f32x4 part[C][KT * RG];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < KT * RG; ++i) part[c][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int j = 0; j < KT; ++j) {
        const uint4 k = *reinterpret_cast<const uint4*>(keys + (16 * j + fr) * R::kBytes + (((4 * ks + fg) ^ sw) << 4));
#pragma unroll
        for (int i = 0; i < RG; ++i) {
          if constexpr (kBf) {
            f32x4& x = part[0][j * RG + i];
            x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k),
                                                        __builtin_bit_cast(bf16x8, q[i * KS + ks]), x, 0, 0, 0);
          } else {
            const f32x4 a = __builtin_bit_cast(f32x4, k), b = __builtin_bit_cast(f32x4, q[i * KS + ks]);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              part[e % C][j * RG + i] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], part[e % C][j * RG + i], 0, 0, 0);
          }
        }
      }
#pragma unroll
    for (int i = 0; i < KT * RG; ++i) {
      s[i] = part[0][i];
      if constexpr (C == 2) s[i] += part[1][i];
      if constexpr (C == 4) s[i] = (part[0][i] + part[1][i]) + (part[2][i] + part[3][i]);
    }
    pipeline<KT * KS, KT * KS < 6 ? KT * KS : 6, kBf ? RG : 4 * RG, 1>();
    __builtin_amdgcn_sched_barrier(0);
  }
  // The order of a region of `reads` x PER LDS reads that feed MFMAS products each: AHEAD of them first,
  // then one (PER reads) for every MFMAS products.
  template <int READS, int AHEAD, int MFMAS, int PER>
  __device__ __forceinline__ static void pipeline() {
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * PER, 0);
#pragma unroll
    for (int i = 0; i < READS - AHEAD; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x8, MFMAS, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, AHEAD * MFMAS, 0);
  }
  // The bf16 operand V^T[16 t .. +15][32 keys] of keys 4 fg .. +3 and 16 + 4 fg .. +3 of `half`
  __device__ __forceinline__ static bf16x8 value_frag(const unsigned char* values, int half, int t, int lane) {
    const int sub = lane & 15, row = 32 * half + 4 * (lane >> 4) + (sub >> 2);
    const int piece = 2 * t + ((sub >> 1) & 1), at = (sub & 1) * 8;
    const unsigned char* lo = values + row * R::kBytes + ((piece ^ R::value_swizzle(row)) << 4) + at;
    const unsigned char* hi = values + (row + 16) * R::kBytes + ((piece ^ R::value_swizzle(row + 16)) << 4) + at;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)lo);
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)hi);
    return __builtin_shufflevector(__builtin_bit_cast(bf16x4, a), __builtin_bit_cast(bf16x4, b), 0, 1, 2, 3, 4, 5, 6, 7);
  }
  // The bf16 operand P^T of a group's two tiles of 16 keys, s[0] and s[RG]
  template <int RG>
  __device__ __forceinline__ static bf16x8 weights(const f32x4* s) {
    bf16x8 p;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      p[r] = (__bf16)s[0][r];
      p[4 + r] = (__bf16)s[RG][r];
    }
    return p;
  }
  // The same for OT output tiles from tile t0 on and operands p[2][RG] of 64 keys (bf16)
  template <int RG, int OT>
  __device__ __forceinline__ static void values_of(const unsigned char* vals, int t0, const bf16x8* p, f32x4* o, int lane) {
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int t = 0; t < OT; ++t) {
        const bf16x8 vf = value_frag(vals, c, t0 + t, lane);
#pragma unroll
        for (int i = 0; i < RG; ++i)
          o[i * OT + t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, p[c * RG + i], o[i * OT + t], 0, 0, 0);
      }
    pipeline<2 * OT, 5, RG, 2>();
    __builtin_amdgcn_sched_barrier(0);
  }
  // O^T += V^T P^T over KT tiles of 16 keys: s[tile][group], o[group][DT]
  template <int KT, int RG>
  __device__ __forceinline__ static void values(const unsigned char* vals, const f32x4* s, f32x4* o, int lane) {
    if constexpr (kBf) {
#pragma unroll
      for (int c = 0; c < KT / 2; ++c) {
        bf16x8 pf[RG];
#pragma unroll
        for (int i = 0; i < RG; ++i) pf[i] = weights<RG>(s + 2 * c * RG + i);
#pragma unroll
        for (int t = 0; t < DT; ++t) {
          const bf16x8 vf = value_frag(vals, c, t, lane);
#pragma unroll
          for (int i = 0; i < RG; ++i)
            o[i * DT + t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[i], o[i * DT + t], 0, 0, 0);
        }
      }
      pipeline<KT / 2 * DT, KT / 2 * DT < 5 ? KT / 2 * DT : 5, RG, 2>();
    } else {
      const int fr = lane & 15, fg = lane >> 4;
#pragma unroll
      for (int j = 0; j < KT; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const unsigned char* row = vals + (16 * j + 4 * fg + r) * R::kBytes + fr * (4 * E);
#pragma unroll
          for (int t = 0; t < DT / E; ++t) {
            float a[E];
            if constexpr (E == 4) *reinterpret_cast<f32x4*>(a) = *reinterpret_cast<const f32x4*>(row + t * 64 * E);
            else *reinterpret_cast<f32x2*>(a) = *reinterpret_cast<const f32x2*>(row + t * 64 * E);
#pragma unroll
            for (int i = 0; i < RG; ++i)
#pragma unroll
              for (int e = 0; e < E; ++e)
                o[i * DT + t * E + e] =
                    __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], s[j * RG + i][r], o[i * DT + t * E + e], 0, 0, 0);
          }
        }
      pipeline<KT * 4 * (DT / E), 4, E * RG, 1>();
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  // The output that element r of the lane's tile t is
  __device__ __forceinline__ static int column(int t, int r, int fg) {
    return kBf ? 16 * t + 4 * fg + r : 16 * E * (t / E) + 4 * E * fg + E * r + t % E;
  }
  // Calls f(d, x) for runs of 4 consecutive outputs x of the lane's query row, at d .. d + 3 (fp32 at
  // D = 32: 2 runs of 4 all the same).
  template <typename F>
  __device__ __forceinline__ static void each_run(const f32x4* o, int fg, F f) {
    if constexpr (kBf) {
#pragma unroll
      for (int t = 0; t < DT; ++t) f(16 * t + 4 * fg, o[t]);
    } else if constexpr (E == 4) {
#pragma unroll
      for (int t = 0; t < DT / 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          f(64 * t + 16 * fg + 4 * r, f32x4{o[4 * t][r], o[4 * t + 1][r], o[4 * t + 2][r], o[4 * t + 3][r]});
    } else {
#pragma unroll
      for (int r = 0; r < 4; r += 2) f(8 * fg + 2 * r, f32x4{o[0][r], o[1][r], o[0][r + 1], o[1][r + 1]});
    }
  }
};

__device__ __forceinline__ void store_run(float* p, f32x4 x) { *reinterpret_cast<f32x4*>(p) = x; }
__device__ __forceinline__ void store_run(bf16_t* p, f32x4 x) {
  *reinterpret_cast<uint2*>(p) = make_uint2((uint32_t)f2bf(x[0]) | ((uint32_t)f2bf(x[1]) << 16),
                                            (uint32_t)f2bf(x[2]) | ((uint32_t)f2bf(x[3]) << 16));
}

// What `scale` turns into a score in log2 units, up to a constant of all a row's, in the same fma that takes
// the maximum off (one rounding, at the size of the difference): a product of a query and a key, or where
// scores are capped as c tanh(s / c), the tanh (fp32), or, as tanh x = 2 / (1 + e^(-2 x)) - 1, the fraction.
// That is off by a few fp32 roundings of c: up to c = 4096, the most that bf16 is served with, by some 2^-10,
// as a bf16 weight is by its own rounding.
template <typename T, bool CAP>
__device__ __forceinline__ float score(const PagedAttn& p, float s) {
  if constexpr (!CAP) return s;
  if constexpr (sizeof(T) == 4) return tanhf(s * p.cap_in);
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s * p.cap_in));
}
__device__ __forceinline__ float weight(const PagedAttn& p, float s, float m) {
  return __builtin_amdgcn_exp2f(__builtin_fmaf(s, p.scale, -m));
}

// The scores of KT x 16 keys from k0 on of one group (every RG-th of s), those of positions outside lo .. hi
// at -inf unless all are inside (`whole`, uniform); returns the lane's largest, in log2 units.
template <typename T, bool CAP, int KT, int RG>
__device__ __forceinline__ float mask_scores(const PagedAttn& p, f32x4* s, bool whole, int first, int lo, int hi) {
  float mx = -INFINITY;
  if (whole) {
#pragma unroll
    for (int j = 0; j < KT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[j * RG][r] = score<T, CAP>(p, s[j * RG][r]);
        mx = fmaxf(mx, s[j * RG][r]);
      }
  } else {
    // the lane's key 16 j + r of the chunk is position first + 16 j + r
    const int a = lo - first, n = hi - lo;
#pragma unroll
    for (int j = 0; j < KT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float y = score<T, CAP>(p, s[j * RG][r]);
        s[j * RG][r] = hi >= lo && (uint32_t)(16 * j + r - a) <= (uint32_t)n ? y : -INFINITY;
        mx = fmaxf(mx, s[j * RG][r]);
      }
  }
  return mx * p.scale;
}

// Outputs that are NaN although the row's sum l is not: a position that another row of the wave sees, and this
// one may not, holds an infinite or NaN value, and its weight 0 times that is NaN. (Or one that it may see does,
// and then they stay what they are.) The lane's OT tiles from tile t0 on are summed again, key by key from memory
// over positions from .. to - 1, without those outside lo .. pos. Slow, and not on any path of finite values.
template <typename T, int D, bool CAP, int OT>
__device__ __forceinline__ void mend(const PagedAttn& p, ConstInts table, int h, const uint4* q, f32x4* o, float l,
                                     float m_run, int from, int to, int lo, int pos, int t0, int fg) {
  using M = Tile16<T, D>;
  using R = Rows<T, D>;
  bool mine = false;
#pragma unroll
  for (int t = 0; t < OT; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) mine |= o[t][r] != o[t][r];
  mine = mine && l == l;
  if (!__any(mine)) return;
  const float m = m_run == -INFINITY ? 0.f : m_run;
#pragma unroll
  for (int t = 0; t < OT; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) o[t][r] = mine ? 0.f : o[t][r];
#pragma unroll 1
  for (int j = from; j < to; ++j) {
    const int id = uniform(table[min(j >> p.b.page_shift, p.b.cols - 1)]);
    const int slot = j & ((1 << p.b.page_shift) - 1);
    const int64_t at = ((((int64_t)((uint32_t)id < (uint32_t)p.b.n_pages ? id : 0) * p.b.Hkv + h) << p.b.page_shift) + slot) * D;
    float s = 0.f;
#pragma unroll
    for (int ks = 0; ks < M::KS; ++ks) {
      float a[R::kVec], b[R::kVec];
      Elem<T>::unpack(q[ks], a);
      Elem<T>::unpack(*reinterpret_cast<const uint4*>((const T*)p.k + at + (4 * ks + fg) * R::kVec), b);
#pragma unroll
      for (int e = 0; e < R::kVec; ++e) s = __builtin_fmaf(a[e], b[e], s);
    }
    s += __shfl_xor(s, 16, 64);
    s += __shfl_xor(s, 32, 64);
    const bool see = mine && j >= lo && j <= pos;
    const float w = weight(p, score<T, CAP>(p, s), m);
    const T* v = (const T*)p.v + at;
#pragma unroll
    for (int t = 0; t < OT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float x = Elem<T>::load(v + M::column(t0 + t, r, fg));
        o[t][r] = see ? __builtin_fmaf(w, x, o[t][r]) : o[t][r];
      }
  }
}

// ---------------------------------------------------------------------------------------
// the step kernel
// ---------------------------------------------------------------------------------------
// Few rows a sequence (kv head's query heads and tokens together), in blocks of 16: every key and value read
// is used by one MFMA operand, so memory is the bound. The keys of all sequences and kv heads,
// in chunks of KC, are one line that is cut into equal runs, one for each wave of the chip (a
// workgroup), whatever the sequences' lengths are; a wave streams its run through an LDS ring of its
// own (ST chunks, direct loads, no barrier), across the sequences' borders. A (sequence, kv head)
// inside one run is finished there; the parts of one that is cut are joined by the second kernel.
// Where the tables hold a few chunks a sequence at most, a wave takes one (sequence, kv head) whole
// (WHOLE), and there is no second launch. Measured: 6 single tokens behind 20001 to 60000 positions, 32 / 4
// heads at D 128, 107 us with the join, 5.2 TB/s (a 1 GiB copy: 5.16); 48 behind 500 to 2048, 8 / 1 heads at D
// 256, 22 us for 65 MB, where the first loads' latency and the second launch weigh.

// What a sequence's rows see: positions lo .. hi - 1, token i those up to base + i. `blocks`: of 16 rows.
struct StepSeq {
  int row0, n, base, lo, hi, blocks;
};
__device__ __forceinline__ StepSeq step_seq(const PagedAttn& p, int row0, int n, int len) {
  StepSeq s;
  s.row0 = row0;
  s.n = min(n, p.max_q);
  s.base = len - n;
  s.lo = max(p.skip, p.window > 0 ? s.base - p.window + 1 : 0);
  s.hi = s.base + s.n;
  s.blocks = (s.n * p.g + 15) >> 4;
  if (s.n <= 0 || s.hi <= s.lo) s.lo = s.hi = 0;
  return s;
}
template <int KC>
__device__ __forceinline__ int step_chunks(const StepSeq& s) {
  return s.hi > 0 ? (s.hi + KC - 1) / KC - s.lo / KC : 0;
}
// The length of the runs that `total` chunks are cut into: one for each worker, but no sequence of `most`
// chunks in more than kMostParts, whose join would take longer than the waves spared (one sequence of 30000
// positions, 2 heads at D 128: 24.3 us, 30.8 in as many parts as workers).
constexpr int kMostParts = 64;
__device__ __forceinline__ int step_run(const PagedAttn& p, int total, int most) {
  return max((int)(((uint32_t)total + p.workers - 1) / (uint32_t)p.workers), (most + kMostParts - 1) / kMostParts);
}
__device__ __forceinline__ int wave_max_int(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o, 64));
  return v;
}
__device__ __forceinline__ int wave_sum_int(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// The sequence at which a wave stands (uniform): read through the scalar cache, whose waits leave the
// direct loads alone.
__device__ __forceinline__ StepSeq step_seq_at(const PagedAttn& p, int s) {
  ConstInts start = const_ints(p.b.q_start), len = const_ints(p.b.kv_len);
  const int a = uniform(start[s]), e = uniform(start[s + 1]), l = uniform(len[s]);
  const int row0 = min(max(a, 0), p.b.n_rows);
  return step_seq(p, row0, min(max(e, row0), p.b.n_rows) - row0, min(max(l, 0), p.b.cols << p.b.page_shift));
}

template <int KC>
struct StepCursor {
  int s, h, rb, c;  // sequence, kv head, block of rows, chunk
  StepSeq q;
  __device__ __forceinline__ void next(const PagedAttn& p) {
    if (++c < (q.hi + KC - 1) / KC) return;
    if (++rb == q.blocks) {
      rb = 0;
      ++h;
    }
    if (h == p.b.Hkv) {
      h = 0;
      do {
        if (++s >= p.b.n_seqs) return;
        q = step_seq_at(p, s);
      } while (q.hi == 0);
    }
    c = q.lo / KC;
  }
};

template <typename T, int D, int KC, int ST, bool CAP, bool WHOLE>
__device__ __forceinline__ void step_wave(const PagedAttn& p, const int w, unsigned char* ring) {
  using R = Rows<T, D>;
  using M = Tile16<T, D>;
  constexpr int KT = KC / 16, kHalf = KC * R::kBytes, kStage = 2 * kHalf;
  constexpr int kLoads = kHalf / 1024;  // direct loads for a chunk's keys, and for its values
  const int lane = threadIdx.x & 63, fr = lane & 15, fg = lane >> 4;
  const int g = p.g;

  StepCursor<KC> ld;
  int begin, end;
  if constexpr (WHOLE) {
    const int item = w / p.row_blocks;
    ld.rb = w - item * p.row_blocks;
    ld.s = item / p.b.Hkv;
    ld.h = item - ld.s * p.b.Hkv;
    const PagedSeq raw = paged_seq(p.b, ld.s, ld.h == 0 && ld.rb == 0 && lane == 0);
    ld.q = step_seq(p, uniform(raw.row0), uniform(raw.n), uniform(raw.len));
    if (raw.n > p.max_q && lane == 0) latch(p.b.status, kBadSequence);
    if (ld.rb >= ld.q.blocks) return;
    ld.c = ld.q.lo / KC;
    begin = 0;
    end = step_chunks<KC>(ld.q);
    if (end == 0) {
      // rows that see nothing
      const int h = ld.h, r0 = ld.rb * 16;
      for (int x = lane; x < min(16, ld.q.n * g - r0) * (D / 4); x += 64) {
        const int r = r0 + x / (D / 4), token = r / g;
        store_run((T*)p.out + (int64_t)(ld.q.row0 + token) * p.ld_out + (h * g + r - token * g) * D + 4 * (x % (D / 4)),
                  f32x4{0.f, 0.f, 0.f, 0.f});
      }
      return;
    }
  } else {
    // this wave's run [begin, end) of the line of chunks, and where it begins
    int total = 0, most = 0, mine = 0;
    PagedSeq raw = {};
    for (int s = lane; s < p.b.n_seqs; s += 64) {
      raw = paged_seq(p.b, s, false);
      const StepSeq q = step_seq(p, raw.row0, raw.n, raw.len);
      most = max(most, step_chunks<KC>(q));
      mine = step_chunks<KC>(q) * q.blocks;
      total += mine;
    }
    total = uniform(wave_sum_int(total) * p.b.Hkv);
    const int per = step_run(p, total, uniform(wave_max_int(most)));
    begin = uniform(w * per);
    end = min(total, begin + uniform(per));
    if (begin >= end) return;
    {
      int before = 0, s0 = 0, incl;
      while (true) {
        if (p.b.n_seqs > 64) {
          mine = 0;
          if (s0 + lane < p.b.n_seqs) {
            raw = paged_seq(p.b, s0 + lane, false);
            const StepSeq q = step_seq(p, raw.row0, raw.n, raw.len);
            mine = step_chunks<KC>(q) * q.blocks;
          }
        }
        incl = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const int x = __shfl_up(incl, o, 64);
          if (lane >= o) incl += x;
        }
        const uint64_t past = __ballot((before + incl) * p.b.Hkv > begin);
        if (past) {
          const int at = __ffsll((unsigned long long)past) - 1;
          ld.s = uniform(s0 + at);
          before = uniform(before + __shfl(incl - mine, at, 64));
          ld.q = step_seq(p, uniform(__shfl(raw.row0, at, 64)), uniform(__shfl(raw.n, at, 64)), uniform(__shfl(raw.len, at, 64)));
          break;
        }
        before += uniform(__shfl(incl, 63, 64));
        s0 += 64;
        if (s0 >= p.b.n_seqs) return;  // not reached: begin < total
      }
      const int off = begin - before * p.b.Hkv, chunks = step_chunks<KC>(ld.q);
      const int block = uniform(off / chunks);
      ld.h = ld.q.blocks == 1 ? block : block / ld.q.blocks;
      ld.rb = block - ld.h * ld.q.blocks;
      ld.c = ld.q.lo / KC + off - block * chunks;
    }
  }
  StepCursor<KC> cp = ld;

  const uint32_t ring0 = lds_offset(ring);
  const int count = end - begin;
  int queued = 0;
  // the pages of the chunk to be queued next, looked up a chunk ahead; a block of 16 positions without a
  // visible one is read from page 0: its scores are masked, its values zeroed
  int id[KT];
  bool bad = false;
  auto look_up = [&]() {
    ConstInts row = const_ints(p.b.table) + (int64_t)ld.s * p.b.ld_table;
#pragma unroll
    for (int j = 0; j < KT; ++j) id[j] = uniform(row[min((ld.c * KC + 16 * j) >> p.b.page_shift, p.b.cols - 1)]);
  };
  auto issue = [&](int stage) {
    const int k0 = ld.c * KC;
#pragma unroll
    for (int j = 0; j < KT; ++j) {
      const int pos = k0 + 16 * j;
      const bool use = pos < ld.q.hi && pos + 16 > ld.q.lo, ok = (uint32_t)id[j] < (uint32_t)p.b.n_pages;
      bad |= use && !ok;
      id[j] = use && ok ? id[j] : 0;
    }
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      const unsigned char* base = (const unsigned char*)(v ? p.v : p.k);
#pragma unroll
      for (int j = 0; j < KT; ++j) {
        const int slot = (k0 + 16 * j) & ((1 << p.b.page_shift) - 1);
        const unsigned char* src = base + ((((int64_t)id[j] * p.b.Hkv + ld.h) << p.b.page_shift) + slot) * R::kBytes;
        const int lds = (int)ring0 + stage * kStage + v * kHalf + j * 16 * R::kBytes;
        if (v) load_block16<T, D, false>(uniform(src), uniform(lds), lane);
        else load_block16<T, D, true>(uniform(src), uniform(lds), lane);
      }
    }
    ld.next(p);
    ++queued;
    if (queued < count) look_up();
  };

  look_up();
#pragma unroll
  for (int st = 0; st < ST; ++st)
    if (queued < count) issue(st);

  uint4 qf[M::KS];
  f32x4 o[M::DT];
  float m_run = -INFINITY, l_part = 0.f;
  bool fresh = true, first_item = true;
  int c_first = cp.c, stage = 0, token = 0, head = 0, row = 0;
  for (int it = 0; it < count; ++it) {
    if (fresh) {
      // the lane's row: token row / g, query head row % g of the kv head's; the columns past them repeat the first
      row = cp.rb * 16 + fr;
      const bool row_ok = row < cp.q.n * g;
      token = row_ok ? row / g : 0;
      head = cp.h * g + (row_ok ? row - token * g : 0);
      const T* qr = (const T*)p.q + (int64_t)(cp.q.row0 + token) * p.ld_q + head * D;
#pragma unroll
      for (int ks = 0; ks < M::KS; ++ks) qf[ks] = *reinterpret_cast<const uint4*>(qr + (4 * ks + fg) * R::kVec);
      // waited for here, once an item: at their first use the compiler would wait in every chunk, for the
      // direct loads in flight too
#pragma unroll
      for (int ks = 0; ks < M::KS; ++ks) asm volatile("" : "+v"(qf[ks].x), "+v"(qf[ks].y), "+v"(qf[ks].z), "+v"(qf[ks].w));
#pragma unroll
      for (int t = 0; t < M::DT; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
      m_run = -INFINITY;
      l_part = 0.f;
      c_first = cp.c;
      fresh = false;
    }
    const int ahead = (queued - it - 1) * 2 * kLoads;  // loads queued after this chunk's
    const unsigned char* keys = ring + stage * kStage;
    unsigned char* vals = ring + stage * kStage + kHalf;
    wait_loads<kLoads, (2 * ST - 1) * kLoads>(ahead + kLoads);
    f32x4 s[KT];
    M::template scores<KT, 1>(keys, qf, s, fr, fg);

    const int k0 = cp.c * KC;
    const int pos = cp.q.base + token;
    const int lo = max(p.skip, p.window > 0 ? pos - p.window + 1 : 0);
    const bool whole = k0 >= max(p.skip, p.window > 0 ? cp.q.hi - p.window : 0) && k0 + KC <= cp.q.base + 1;
    float mx = mask_scores<T, CAP, KT, 1>(p, s, whole, k0 + 4 * fg, lo, pos);
    // the reference maximum moves only when a score passes it by more than 2^8, and only then the
    // row's four lanes are asked (unnormalised probabilities stay below 2^8)
    if (__any(mx > m_run + 8.f)) {
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float m_new = mx > m_run + 8.f ? mx : m_run;
      const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
      l_part *= alpha;
#pragma unroll
      for (int t = 0; t < M::DT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[t][r] *= alpha;
      m_run = m_new;
    }
    const float m_ref = m_run == -INFINITY ? 0.f : m_run;
#pragma unroll
    for (int j = 0; j < KT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[j][r] = weight(p, s[j][r], m_ref);
        l_part += s[j][r];
      }
    wait_loads<kLoads, (2 * ST - 2) * kLoads>(ahead);
    if (k0 < cp.q.lo || k0 + KC > cp.q.hi) {
      // positions that no row sees may hold anything, and 0 times a NaN would be one
      for (int x = lane; x < KC * R::kPieces; x += 64) {
        const int key = k0 + x / R::kPieces;
        if (key < cp.q.lo || key >= cp.q.hi) *reinterpret_cast<uint4*>(vals + x * 16) = make_uint4(0, 0, 0, 0);
      }
    }
    M::template values<KT, 1>(vals, s, o, lane);
    // the stage is free once its reads have returned
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (queued < count) issue(stage);
    stage = stage + 1 == ST ? 0 : stage + 1;

    const bool last = cp.c + 1 == (cp.q.hi + KC - 1) / KC;
    if (last || it + 1 == count) {
      float l = l_part + __shfl_xor(l_part, 16, 64);
      l += __shfl_xor(l, 32, 64);
      const bool all = last && c_first == cp.q.lo / KC;
      if (cp.q.n > 1)  // (the rows of one token see the same)
        mend<T, D, CAP, M::DT>(p, const_ints(p.b.table) + (int64_t)cp.s * p.b.ld_table, cp.h, qf, o, l, m_run,
                               max(c_first * KC, cp.q.lo), min(k0 + KC, cp.q.hi), lo, pos, 0, fg);
      if (row < cp.q.n * g) {
        if (all && p.skip == 0) {
          T* orow = (T*)p.out + (int64_t)(cp.q.row0 + token) * p.ld_out + head * D;
          const float inv = l > 0.f ? 1.f / l : 0.f;
          M::each_run(o, fg, [&](int d, f32x4 x) { store_run(orow + d, x * inv); });
        } else {
          // a run has at most two items that it does not hold whole: the one it begins in, and its last;
          // whole ones that the prefix is still to be joined to come after those of all runs
          const int rows = min(p.max_q * g, 16);
          const int64_t slot = all ? (int64_t)2 * p.workers * rows + (int64_t)(cp.q.row0 + token) * p.b.Hq + head
                                   : (int64_t)(2 * w + (first_item ? 0 : 1)) * rows + fr;
          float* orow = p.part_o + slot * D;
          M::each_run(o, fg, [&](int d, f32x4 x) { store_run(orow + d, x); });
          if (fg == 0) p.part_ml[slot] = make_float2(m_run, l);
        }
      }
      fresh = true;
      first_item = false;
    }
    cp.next(p);
  }
  if (bad && lane == 0) latch(p.b.status, kBadPage);
}

template <typename T, int D, int KC, int ST, bool CAP, bool WHOLE>
__global__ __launch_bounds__(64) void paged_step_kernel(PagedAttn p) {
  __shared__ __attribute__((aligned(1024))) unsigned char ring[ST * 2 * KC * Rows<T, D>::kBytes];
  step_wave<T, D, KC, ST, CAP, WHOLE>(p, blockIdx.x, ring);
}

// Joins the parts of a row's query heads of one kv head: out = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i,
// m the largest m_i. Also what the step kernel has no chunk for: zeros for rows that see nothing, and the
// report of bounds that are out of range. Every workgroup finds its parts from the lengths, as the step
// kernel found its runs; the parts are taken in a fixed order, so results repeat bit for bit.
template <typename T, int D, int KC, int PBQ>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttn p) {
  constexpr int kLanes = D / 4, kGroups = 256 / kLanes;  // threads of a part, groups of them
  constexpr int kPhases = 4, kHeads = kGroups / kPhases;  // a head's parts go round four groups
  __shared__ int sums[4][3];
  __shared__ int found;
  __shared__ f32x4 acc[kGroups][kLanes];
  __shared__ float2 accml[kGroups];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int t = blockIdx.x, hk = blockIdx.z, g = p.g;
  const bool reports = blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0;
  // the row's sequence, and the chunks of all and of those before it
  if (tid == 0) found = -1;
  __syncthreads();
  int all = 0, most = 0, mine = 0;
  for (int s = tid; s < p.b.n_seqs; s += 256) {
    const PagedSeq x = paged_seq(p.b, s, reports);
    const StepSeq q = step_seq(p, x.row0, x.n, x.len);
    most = max(most, step_chunks<KC>(q));
    mine = step_chunks<KC>(q) * q.blocks;
    all += mine;
    if (x.row0 <= t && t < x.row0 + x.n) atomicMax(&found, s);
  }
  __syncthreads();
  const int sq = found;
  if (sq < 0) return;
  int before = 0;
  if (p.b.n_seqs <= 256) {
    before = tid < sq ? mine : 0;
  } else {
    for (int s = tid; s < sq; s += 256) {
      const PagedSeq x = paged_seq(p.b, s, false);
      const StepSeq q = step_seq(p, x.row0, x.n, x.len);
      before += step_chunks<KC>(q) * q.blocks;
    }
  }
  all = wave_sum_int(all);
  before = wave_sum_int(before);
  most = wave_max_int(most);
  if (lane == 0) {
    sums[wave][2] = most;
    sums[wave][0] = all;
    sums[wave][1] = before;
  }
  const PagedSeq raw = paged_seq(p.b, sq, false);
  const StepSeq q = step_seq(p, raw.row0, raw.n, raw.len);
  const int i = t - raw.row0;
  if (hk == 0 && blockIdx.y == 0 && i == 0 && wave == 0 && p.shared > 0) check_shared(p.b, sq, raw, p.shared, lane);
  if (i >= q.n) {
    if (tid == 0) latch(p.b.status, kBadSequence);
    return;
  }
  __syncthreads();
  all = (sums[0][0] + sums[1][0] + sums[2][0] + sums[3][0]) * p.b.Hkv;
  before = sums[0][1] + sums[1][1] + sums[2][1] + sums[3][1];
  most = max(max(sums[0][2], sums[1][2]), max(sums[2][2], sums[3][2]));
  const int chunks = step_chunks<KC>(q);
  const int grp = tid / kLanes, at = tid % kLanes;
  const int h = blockIdx.y * kHeads + grp / kPhases, phase = grp % kPhases;
  const int row = i * g + min(h, g - 1), prow = t * g + min(h, g - 1);  // of the sequence's, of the batch's
  int own = 0, wa = 0;  // parts of the row's own chunks
  bool at_start = false;
  if (chunks > 0) {
    const int per = step_run(p, all, most);
    const int a = before * p.b.Hkv + (hk * q.blocks + row / 16) * chunks;
    wa = a / per;
    own = (a + chunks - 1) / per - wa + 1;
    at_start = a == wa * per;
  }
  const bool done = own == 1 && p.skip == 0;  // finished by the step kernel
  if (done && q.blocks == 1) return;
  const int rows = min(p.max_q * g, 16), parts = done ? 0 : own + (p.skip > 0 ? p.splits : 0);
  const int64_t whole = (int64_t)2 * p.workers * rows + (int64_t)t * p.b.Hq + hk * g + h;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  if (h < g) {
#pragma unroll 4
    for (int k = phase; k < parts; k += kPhases) {
      const bool pre = k >= own;  // the prefix's
      const int64_t mine_at = own == 1 ? whole : (int64_t)(2 * (wa + k) + (k > 0 || at_start ? 0 : 1)) * rows + row % 16;
      const int64_t pre_at = ((int64_t)(hk * p.splits + k - own) * p.row_blocks + prow / PBQ) * PBQ + prow % PBQ;
      const int64_t s = pre ? pre_at : mine_at;
      const float2 ml = (pre ? p.pre_ml : p.part_ml)[s];
      const f32x4 x = *reinterpret_cast<const f32x4*>((pre ? p.pre_o : p.part_o) + s * D + 4 * at);
      const float m_new = fmaxf(m, ml.x), ref = m_new == -INFINITY ? 0.f : m_new;
      const float e0 = __builtin_amdgcn_exp2f(m - ref), e1 = __builtin_amdgcn_exp2f(ml.x - ref);
      l = e0 * l + e1 * ml.y;
      o = e0 * o + e1 * x;
      m = m_new;
    }
  }
  acc[grp][at] = o;
  if (at == 0) accml[grp] = make_float2(m, l);
  __syncthreads();
  if (phase == 0 && h < g && !done) {
    float top = m;
#pragma unroll
    for (int k = 1; k < kPhases; ++k) top = fmaxf(top, accml[grp + k].x);
    const float ref = top == -INFINITY ? 0.f : top, e0 = __builtin_amdgcn_exp2f(m - ref);
    l *= e0;
    o *= e0;
#pragma unroll
    for (int k = 1; k < kPhases; ++k) {
      const float e = __builtin_amdgcn_exp2f(accml[grp + k].x - ref);
      l += e * accml[grp + k].y;
      o += e * acc[grp + k][at];
    }
    store_run((T*)p.out + (int64_t)t * p.ld_out + (hk * g + h) * D + 4 * at, o * (l > 0.f ? 1.f / l : 0.f));
  }
}

// ---------------------------------------------------------------------------------------
// the tile kernel
// ---------------------------------------------------------------------------------------
// Prompts: blocks of NW x RG x 16 rows (tokens x the kv head's query heads, so that they share its keys
// and values) against chunks of KC positions in LDS, double-buffered by direct loads. A plan made on the
// device lists the blocks of all sequences and the chunks that each sees; per kv head they are one line,
// the lines one after another, cut into equal runs for as many workgroups as are resident: neither
// unequal lengths nor the causal triangle leave a workgroup idle. A block takes kTileStart places on the
// line before its chunks, for what starting and ending it costs (without them the run with the many short
// blocks of a prompt's first rows took 202 us beside 118 of the others, four prompts of 2048 at D 256). A
// block cut by a run's border leaves parts, which a third launch joins; writing and reading one's outputs in 32
// bits takes as long as some four chunks, so a border within kTileSnap of a block's edge moves there (but by an
// eighth of a run at most), and a sequence's long blocks and short ones alternate: two of them together are
// alike long, and more borders meet edges. Measured: a plan of 6 us, then 3 sequences of 1000 to 4000 rows and
// 4000 to 8001 keys, 32 / 4 heads at D 128: 974 us with capped scores (782 TFLOP/s; two exp2 and a reciprocal a
// score bound it), 870 without a cap; 4 prompts of 2048, 8 / 1 heads at D 256: 105 us (654 TFLOP/s).
constexpr int kTileStart = 2, kTileSnap = 4;

template <int BQ, int KC>
__global__ __launch_bounds__(1024) void paged_plan_kernel(PagedAttn p, int* total) {
  constexpr int kKeep = 2048, kKeepTiles = 4096;
  __shared__ int wsum[16];
  __shared__ int carry;
  __shared__ int keep[kKeep];
  __shared__ int keep_at[kKeepTiles];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = p.g;
  // inclusive sum over the workgroup plus what went before; all threads call it
  auto scan = [&](int x) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(x, o, 64);
      if (lane >= o) x += y;
    }
    if (lane == 63) wsum[wave] = x;
    __syncthreads();
    int add = carry, all = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      add += i < wave ? wsum[i] : 0;
      all += wsum[i];
    }
    __syncthreads();
    if (tid == 0) carry += all;
    __syncthreads();
    return x + add;
  };
  if (tid == 0) carry = 0;
  __syncthreads();
  // each sequence's first block in the list; all others follow from them
  int* first = p.b.n_seqs <= kKeep ? keep : total + 2;
  for (int s0 = 0; s0 < p.b.n_seqs; s0 += 1024) {
    const int s = s0 + tid;
    int n = 0;
    if (s < p.b.n_seqs) {
      const PagedSeq q = paged_seq(p.b, s, true);
      if (q.n > p.max_q) latch(p.b.status, kBadSequence);
      n = (min(q.n, p.max_q) * g + BQ - 1) / BQ;
    }
    const int end = scan(n);
    if (s < p.b.n_seqs) first[s] = end - n;
  }
  const int tiles = min(carry, p.most_tiles);
  __threadfence_block();
  __syncthreads();
  if (tid == 0) carry = 0;
  __syncthreads();
  for (int t0 = 0; t0 < tiles; t0 += 1024) {
    const int t = t0 + tid;
    PagedTile x = {};
    if (t < tiles) {
      int lo = 0, hi = p.b.n_seqs;  // the last s with first[s] <= t
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= t) lo = mid;
        else hi = mid;
      }
      const PagedSeq q = paged_seq(p.b, lo, false);
      x.seq = lo;
      x.row0 = q.row0;
      x.base = q.len - q.n;
      x.n = min(q.n, p.max_q) * g;
      const int i = t - first[lo], blocks = (x.n + BQ - 1) / BQ;
      x.row = ((i & 1) ? i >> 1 : blocks - 1 - (i >> 1)) * BQ;
      const int a = max(0, p.window > 0 ? x.base + x.row / g - p.window + 1 : 0);
      const int e = x.base + (min(x.row + BQ, x.n) - 1) / g + 1;
      x.chunk0 = a / KC;
      x.chunks = e > a ? (e + KC - 1) / KC - x.chunk0 : 0;
    }
    const int len = x.chunks > 0 ? x.chunks + kTileStart : 0;
    x.at = scan(len) - len + kTileStart;
    if (t < tiles) {
      p.tiles[t] = x;
      if (tiles <= kKeepTiles) keep_at[t] = x.at;
    }
  }
  const int line = carry;
  if (tid == 0) {
    total[0] = line;
    total[1] = tiles;
  }
  __threadfence_block();
  __syncthreads();
  // the runs
  const int places = line * p.b.Hkv, per = max((int)(((uint32_t)places + p.workers - 1) / (uint32_t)p.workers), 1);
  const int snap = min(kTileSnap, per / 8);
  auto start = [&](int t) { return t == tiles ? line : (tiles <= kKeepTiles ? keep_at[t] : p.tiles[t].at) - kTileStart; };
  for (int w = tid; w <= p.workers; w += 1024) {
    PagedRun r = {places, p.b.Hkv, 0, 0};
    if ((int64_t)w * per < places) {
      r.head = w * per / line;
      int off = w * per - r.head * line, lo = 0, hi = tiles;  // the last block that starts at or before off
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start(mid) <= off) lo = mid;
        else hi = mid;
      }
      const int a = start(lo), e = start(lo + 1);
      if (min(off - a, e - off) <= snap) {
        if (off - a <= e - off) {
          off = a;
        } else {
          off = e;
          ++lo;
        }
      }
      r.place = r.head * line + off;
      if (lo == tiles) {
        lo = 0;  // the line's end is the next one's start
        ++r.head;
      }
      r.tile = lo;
    }
    p.runs[w] = r;
  }
  if (p.shared > 0)
    for (int s = wave; s < p.b.n_seqs; s += 16) check_shared(p.b, s, paged_seq(p.b, s, false), p.shared, lane);
}

// The same for a shared prefix (PREFIX): all rows of the batch as one sequence that sees positions 0 ..
// skip - 1 whole, each workgroup one part of them for one block of rows; always parts, which the step
// kernel's join takes in.
//
// PAIR (bf16 at D 256): two waves share RG x 16 rows. Each takes the scores of one half of a chunk's keys and
// the outputs of one half of D, so that a key or value read from LDS serves two groups of rows without the
// outputs of both over all of D in one wave's registers (which leave no room for a second wave on the SIMD).
// They exchange their probabilities through LDS. LDS reads, 128 bytes a cycle, are what bounds the products:
// with 16 rows a wave they took 4000 of a chunk's 7000 cycles.
template <typename T, int D, int NW, int RG, int KC, bool PAIR>
struct TileLds {
  unsigned char ring[2][2 * KC * Rows<T, D>::kBytes];
  uint4 swap_p[PAIR ? NW * RG * 64 : 1];
  float swap_m[PAIR ? NW : 1][RG][16], swap_l[PAIR ? NW : 1][RG][16];
};

template <typename T, int D, int NW, int RG, int KC, bool CAP, bool PREFIX, bool PAIR>
__device__ __forceinline__ void tile_group(const PagedAttn& p, const int* total, const int block, const int blocks,
                                           TileLds<T, D, NW, RG, KC, PAIR>& lds) {
  using R = Rows<T, D>;
  using M = Tile16<T, D>;
  constexpr int KT = KC / 16, BQ = 16 * RG * (PAIR ? NW / 2 : NW), kHalf = KC * R::kBytes;
  constexpr int KTW = PAIR ? KT / 2 : KT, OT = PAIR ? M::DT / 2 : M::DT;  // a wave's key tiles and output tiles
  static_assert(!PAIR || (KT == 4 && M::kBf), "pairs take 64 keys in bf16");
  auto& ring = lds.ring;
  auto& swap_p = lds.swap_p;
  auto& swap_m = lds.swap_m;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), fr = lane & 15, fg = lane >> 4;
  const int g = p.g;
  const int row_wave = PAIR ? wave % (NW / 2) : wave, half = PAIR ? wave / (NW / 2) : 0;  // a pair's are on one SIMD
  const int other = PAIR ? wave ^ (NW / 2) : wave;
  // workgroups go round the 8 XCDs; neighbouring runs read the same keys, so each XCD takes a stretch of them
  const int w = block % 8 * (blocks / 8) + block / 8;
  const uint32_t ring0 = lds_offset(ring);

  // the part of a block's chunks that the run holds: chunks c0 .. c0 + count - 1 of kv head h
  struct Item {
    int h, c0, count, chunks, seq, row0, base, n, row, hi_pos, lo_pos;
  };
  int at = w, stop = min(w + 1, p.b.Hkv * p.splits * p.row_blocks), line = 1, tiles = 0, tile = 0, head = 0;
  typedef const __attribute__((address_space(4))) PagedTile* ConstTiles;
  ConstTiles list = (ConstTiles)(uintptr_t)p.tiles;
  // goes to the first block from (head, tile) on that sees anything, and `at` to its first chunk
  auto seek = [&]() {
    if constexpr (!PREFIX) {
      while (true) {
        if (tile == tiles) {
          tile = 0;
          ++head;
        }
        if (head == p.b.Hkv || uniform(list[tile].chunks) > 0) break;
        ++tile;
      }
      at = head == p.b.Hkv ? stop : head * line + uniform(list[tile].at);
    }
  };
  // the item there, of which the run holds the chunks from place `begin` on; goes on to the next one
  auto item = [&](int begin) {
    Item x;
    if constexpr (PREFIX) {
      x.h = at / (p.splits * p.row_blocks);
      const int split = at / p.row_blocks % p.splits, all = (p.skip + KC - 1) / KC;
      x.c0 = (int)((int64_t)split * all / p.splits);
      x.count = (int)((int64_t)(split + 1) * all / p.splits) - x.c0;
      x.chunks = x.seq = x.row0 = x.lo_pos = 0;
      x.row = at % p.row_blocks * BQ;
      x.n = p.b.n_rows * g;
      x.base = p.skip - 1;
      x.hi_pos = p.skip;
      at += 1;
    } else {
      begin = max(begin, at);
      x.h = head;
      x.chunks = uniform(list[tile].chunks);
      x.c0 = uniform(list[tile].chunk0) + begin - at;
      x.count = min(at + x.chunks, stop) - begin;
      x.seq = uniform(list[tile].seq);
      x.row0 = uniform(list[tile].row0);
      x.base = uniform(list[tile].base);
      x.n = uniform(list[tile].n);
      x.row = uniform(list[tile].row);
      x.hi_pos = x.base + (min(x.row + BQ, x.n) - 1) / g + 1;
      x.lo_pos = max(0, p.window > 0 ? x.base + x.row / g - p.window + 1 : 0);
      ++tile;
      seek();
    }
    return x;
  };
  int begin = at;
  if constexpr (!PREFIX) {
    ConstInts tot = const_ints(total);
    line = uniform(tot[0]);
    tiles = uniform(tot[1]);
    typedef const __attribute__((address_space(4))) PagedRun* ConstRuns;
    ConstRuns run = (ConstRuns)(uintptr_t)p.runs + w;
    begin = uniform(run[0].place);
    stop = uniform(run[1].place);
    head = uniform(run[0].head);
    tile = uniform(run[0].tile);
    if (begin >= stop) return;
    seek();
  }
  if (at >= stop) return;

  // Pages: a lane holds one entry of the item's row of the table, 64 from entry `first` on, from which the
  // wave picks. `pages` looks ahead for the item whose chunks are queued next.
  struct Pages {
    int first, entry;
  };
  auto look_up = [&](const Item& x, int c) {
    Pages t;
    t.first = (c * KC) >> p.b.page_shift;
    t.entry = p.b.table[(int64_t)x.seq * p.b.ld_table + min(t.first + lane, p.b.cols - 1)];
    asm volatile("" : "+v"(t.entry));  // waited for here, not at each use, where the direct loads would be too
    return t;
  };
  // Queues chunk c of an item: the wave's blocks of 16 positions (keys' blocks, then values'). One that no
  // row of the block of rows sees is read from page 0 (masked, and zeroed).
  constexpr int kMine = (2 * KT + NW - 1) / NW;
  bool bad = false;
  auto issue = [&](const Item& x, int c, int stage, const Pages& t) {
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int blk = i * NW + wave;
      if (2 * KT % NW != 0 && blk >= 2 * KT) break;
      const int j = blk % KT, pos = c * KC + 16 * j;
      const int id = __builtin_amdgcn_readlane(t.entry, (pos >> p.b.page_shift) - t.first);
      const bool use = pos < x.hi_pos && pos + 16 > x.lo_pos, ok = (uint32_t)id < (uint32_t)p.b.n_pages;
      bad |= use && !ok;
      const int slot = pos & ((1 << p.b.page_shift) - 1);
      const int64_t from = ((((int64_t)(use && ok ? id : 0) * p.b.Hkv + x.h) << p.b.page_shift) + slot) * R::kBytes;
      const int lds = (int)ring0 + stage * 2 * kHalf + (blk / KT) * kHalf + j * 16 * R::kBytes;
      if (blk < KT) load_block16<T, D, true>(uniform((const unsigned char*)p.k + from), uniform(lds), lane);
      else load_block16<T, D, false>(uniform((const unsigned char*)p.v + from), uniform(lds), lane);
    }
  };

  // chunks follow one another through the two buffers, across the items' borders too
  Item x = item(begin);
  int stage = 0;
  bool first_item = true;
  Pages pages = look_up(x, x.c0);
  issue(x, x.c0, 0, pages);
  while (true) {
    const bool more = at < stop;
    Item next = x;
    if (more) next = item(at);
    const int h = x.h, n = x.n;
    // the position of the block's row r
    auto position = [&](int r) { return PREFIX ? x.base : x.base + r / g; };

    // this wave's rows
    uint4 qf[RG * M::KS];
    int pos_r[RG], lo_r[RG];
    f32x4 o[RG * OT];
    float m_run[RG], l_part[RG];
    const int wrow = x.row + row_wave * 16 * RG;
#pragma unroll
    for (int i = 0; i < RG; ++i) {
      const int r = min(wrow + 16 * i + fr, n - 1), token = r / g;
      const T* qr = (const T*)p.q + (int64_t)(x.row0 + token) * p.ld_q + (h * g + r - token * g) * D;
#pragma unroll
      for (int ks = 0; ks < M::KS; ++ks)
        qf[i * M::KS + ks] = *reinterpret_cast<const uint4*>(qr + (4 * ks + fg) * R::kVec);
      pos_r[i] = position(r);
      lo_r[i] = p.window > 0 ? max(0, pos_r[i] - p.window + 1) : 0;
#pragma unroll
      for (int t = 0; t < OT; ++t) o[i * OT + t] = f32x4{0.f, 0.f, 0.f, 0.f};
      m_run[i] = -INFINITY;
      l_part[i] = 0.f;
    }
    Pages next_pages = pages;
    if (more) next_pages = look_up(next, next.c0);
#pragma unroll
    for (int k = 0; k < RG * M::KS; ++k)
      asm volatile("" : "+v"(qf[k].x), "+v"(qf[k].y), "+v"(qf[k].z), "+v"(qf[k].w));
    // what all, and what any, of the wave's rows see
    const int pos_first = position(min(wrow, n - 1)), pos_last = position(min(wrow + 16 * RG - 1, n - 1));
    const int lo_last = p.window > 0 ? max(0, pos_last - p.window + 1) : 0;
    const int lo_first = p.window > 0 ? max(0, pos_first - p.window + 1) : 0;
    const bool rows_here = wrow < n;

    for (int ch = 0; ch < x.count; ++ch) {
      const int k0 = (x.c0 + ch) * KC;
      const unsigned char* keys = ring[stage];
      unsigned char* vals = ring[stage] + kHalf;
      stage ^= 1;
      dma_stage_sync<0>();  // this chunk has landed, and every wave is done with the other buffer
      // the next chunk's loads. They leave a CU at 64 bytes a cycle, and who queues them waits for that: of a
      // pair one queues its own before the scores, one after them
      auto queue = [&]() {
        if (ch + 1 < x.count) {
          if (((k0 + 2 * KC - 1) >> p.b.page_shift) - pages.first >= 64) pages = look_up(x, x.c0 + ch + 1);
          issue(x, x.c0 + ch + 1, stage, pages);
        } else if (more) {
          issue(next, next.c0, stage, next_pages);
        }
      };
      if (half == 0) queue();
      if (k0 < x.lo_pos || k0 + KC > x.hi_pos) {
        // positions that no row of the block sees may hold anything, and 0 times a NaN would be one
        for (int y = tid; y < KC * R::kPieces; y += 64 * NW) {
          const int key = k0 + y / R::kPieces;
          if (key < x.lo_pos || key >= x.hi_pos) *reinterpret_cast<uint4*>(vals + y * 16) = make_uint4(0, 0, 0, 0);
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      }
      const bool sees = rows_here && k0 <= pos_last && k0 + KC > lo_first;
      if (!sees) {
        if (half) queue();
        if constexpr (PAIR) asm volatile("s_barrier" ::: "memory");  // the one of the exchange below
        continue;
      }
      const int kw = k0 + half * 16 * KTW;  // the wave's keys
      f32x4 s[KTW * RG];
      M::template scores<KTW, RG>(keys + half * 16 * KTW * R::kBytes, qf, s, fr, fg);
      if (half) queue();
      const bool whole = kw >= lo_last && kw + 16 * KTW <= pos_first + 1;
      float mx[RG];
      bool grow = false;
#pragma unroll
      for (int i = 0; i < RG; ++i) {
        mx[i] = mask_scores<T, CAP, KTW, RG>(p, s + i, whole, kw + 4 * fg, lo_r[i], pos_r[i]);
        grow |= mx[i] > m_run[i] + 8.f;
      }
      if (__any(grow)) {
#pragma unroll
        for (int i = 0; i < RG; ++i) {
          float v = fmaxf(mx[i], __shfl_xor(mx[i], 16, 64));
          v = fmaxf(v, __shfl_xor(v, 32, 64));
          if constexpr (PAIR) v = ceilf(v);  // a whole power of two scales bf16 exactly, below
          const float m_new = v > m_run[i] + 8.f ? v : m_run[i];
          const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run[i] - m_new);
          l_part[i] *= alpha;
#pragma unroll
          for (int t = 0; t < OT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[i * OT + t][r] *= alpha;
          m_run[i] = m_new;
        }
      }
#pragma unroll
      for (int i = 0; i < RG; ++i) {
        const float m_ref = m_run[i] == -INFINITY ? 0.f : m_run[i];
#pragma unroll
        for (int j = 0; j < KTW; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float y = weight(p, s[j * RG + i][r], m_ref);
            s[j * RG + i][r] = y;
            l_part[i] += y;
          }
      }
      if constexpr (!PAIR) {
        M::template values<KT, RG>(vals, s, o, lane);
      } else {
        bf16x8 pw[2 * RG];  // of both halves' keys
#pragma unroll
        for (int i = 0; i < RG; ++i) {
          const bf16x8 mine = M::template weights<RG>(s + i);
          swap_p[(wave * RG + i) * 64 + lane] = __builtin_bit_cast(uint4, mine);
          if (fg == 0) swap_m[wave][i][fr] = m_run[i];
          pw[i] = pw[RG + i] = mine;
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        float m_other[RG];
        bool differ = false;
#pragma unroll
        for (int i = 0; i < RG; ++i) {
          const bf16x8 theirs = __builtin_bit_cast(bf16x8, swap_p[(other * RG + i) * 64 + lane]);
          if (half) pw[i] = theirs;
          else pw[RG + i] = theirs;
          m_other[i] = swap_m[other][i][fr];
          differ |= m_other[i] != m_run[i];
        }
        if (__any(differ)) {
          // one of the two moved its maximum (rarely, once a row has seen a chunk): both go by the larger
#pragma unroll
          for (int i = 0; i < RG; ++i) {
            const float m_new = fmaxf(m_run[i], m_other[i]), ref = m_new == -INFINITY ? 0.f : m_new;
            const float mine = __builtin_amdgcn_exp2f(m_run[i] - ref), theirs = __builtin_amdgcn_exp2f(m_other[i] - ref);
            const float first = half ? theirs : mine, second = half ? mine : theirs;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              pw[i][e] = (__bf16)((float)pw[i][e] * first);
              pw[RG + i][e] = (__bf16)((float)pw[RG + i][e] * second);
            }
            l_part[i] *= mine;
#pragma unroll
            for (int t = 0; t < OT; ++t)
#pragma unroll
              for (int r = 0; r < 4; ++r) o[i * OT + t][r] *= mine;
            m_run[i] = m_new;
          }
        }
        M::template values_of<RG, OT>(vals, half * OT, pw, o, lane);
      }
    }
    auto each_run = [&](int i, auto f) {
      if constexpr (PAIR) {
#pragma unroll
        for (int t = 0; t < OT; ++t) f(16 * (half * OT + t) + 4 * fg, o[i * OT + t]);
      } else {
        M::each_run(o + i * OT, fg, f);
      }
    };
    const bool all = x.count == x.chunks;
    const int64_t slot = (PREFIX ? (int64_t)w : (int64_t)2 * w + (first_item ? 0 : 1)) * BQ;
    float* part_o = PREFIX ? p.pre_o : p.part_o;
    float2* part_ml = PREFIX ? p.pre_ml : p.part_ml;
    if constexpr (PAIR) {
      // the row's sum over both halves of the keys (not by way of swap_p or swap_m, which the other wave may
      // still be reading for the last chunk)
#pragma unroll
      for (int i = 0; i < RG; ++i) {
        l_part[i] += __shfl_xor(l_part[i], 16, 64);
        l_part[i] += __shfl_xor(l_part[i], 32, 64);
        if (fg == 0) lds.swap_l[wave][i][fr] = l_part[i];
      }
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
      for (int i = 0; i < RG; ++i) l_part[i] += lds.swap_l[other][i][fr];
    }
#pragma unroll
    for (int i = 0; i < RG; ++i) {
      float l = l_part[i];
      if constexpr (!PAIR) {
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
      }
      const int r = wrow + 16 * i + fr, token = r / g;
      if constexpr (!PREFIX)
        mend<T, D, CAP, OT>(p, const_ints(p.b.table) + (int64_t)x.seq * p.b.ld_table, h, qf + i * M::KS, o + i * OT, l,
                            m_run[i], max(x.c0 * KC, x.lo_pos), min((x.c0 + x.count) * KC, x.hi_pos), lo_r[i], pos_r[i],
                            half * OT, fg);
      if (r >= n) continue;
      if (!PREFIX && all) {
        T* orow = (T*)p.out + (int64_t)(x.row0 + token) * p.ld_out + (h * g + r - token * g) * D;
        const float inv = l > 0.f ? 1.f / l : 0.f;
        each_run(i, [&](int d, f32x4 y) { store_run(orow + d, y * inv); });
      } else {
        const int64_t at_row = slot + r - x.row;
        each_run(i, [&](int d, f32x4 y) { store_run(part_o + at_row * D + d, y); });
        if (fg == 0 && half == 0) part_ml[at_row] = make_float2(m_run[i], l);
      }
    }
    first_item = false;
    if (!more) break;
    x = next;
    pages = next_pages;
  }
  if (bad && lane == 0) latch(p.b.status, kBadPage);
}

template <typename T, int D, int NW, int RG, int KC, bool CAP, bool PAIR>
__global__ __launch_bounds__(64 * NW) void paged_tile_kernel(PagedAttn p, const int* total) {
  __shared__ __attribute__((aligned(1024))) TileLds<T, D, NW, RG, KC, PAIR> lds;
  tile_group<T, D, NW, RG, KC, CAP, false, PAIR>(p, total, blockIdx.x, gridDim.x, lds);
}

// A shared prefix and the sequences' own parts in one launch: the first is bound by the matrix cores, the
// second by memory. Eight workgroups (one an XCD) of each kind take turns in the grid; one of the second
// kind holds as many waves of the step kernel as its LDS has room for.
template <typename T, int D, int NW, int RG, int KC, bool PAIR, int SKC, bool CAP>
__global__ __launch_bounds__(64 * NW) void paged_shared_kernel(PagedAttn p, int prefix_blocks, int step_blocks) {
  using Lds = TileLds<T, D, NW, RG, KC, PAIR>;
  constexpr int kRing = 2 * 2 * SKC * Rows<T, D>::kBytes;  // two chunks
  __shared__ __attribute__((aligned(1024))) unsigned char lds[sizeof(Lds) > kRing ? sizeof(Lds) : kRing];
  constexpr int kWaves = sizeof(lds) / kRing < NW ? sizeof(lds) / kRing : NW;
  const int round = blockIdx.x / 8, pre = prefix_blocks / 8, step = step_blocks / 8, both = min(pre, step);
  const bool tile = round < 2 * both ? (round & 1) == 0 : pre > step;
  const int block = (round < 2 * both ? round / 2 : round - both) * 8 + blockIdx.x % 8;
  if (tile) {
    tile_group<T, D, NW, RG, KC, CAP, true, PAIR>(p, nullptr, block, prefix_blocks, *reinterpret_cast<Lds*>(lds));
  } else {
    const int wave = uniform(threadIdx.x >> 6);
    if (wave < kWaves && block * kWaves + wave < p.workers)
      step_wave<T, D, SKC, 2, CAP, false>(p, block * kWaves + wave, lds + wave * kRing);
  }
}

// Joins the parts of blocks that runs' borders cut (8 to 17 us for the 67 MB of 512 runs' parts), and writes zeros for blocks that see nothing. A workgroup
// belongs to a border and 16 rows of the block that it cuts; where a block is cut more than once the borders
// share its rows, so that many parts have many workgroups.
template <typename T, int D, int BQ>
__global__ __launch_bounds__(256) void paged_tile_join_kernel(PagedAttn p, const int* total) {
  constexpr int kLanes = D / 4, kGroups = 256 / kLanes;
  __shared__ f32x4 acc[kGroups][kLanes];
  __shared__ float2 accml[kGroups];
  const int tid = threadIdx.x, g = p.g, at = tid % kLanes, grp = tid / kLanes, lane = tid & 63;
  const int line = total[0], tiles = total[1], w = blockIdx.x + 1;
  auto out_row = [&](const PagedTile& x, int h, int r) {
    const int token = r / g;
    return (T*)p.out + (int64_t)(x.row0 + token) * p.ld_out + (h * g + r - token * g) * D + 4 * at;
  };
  for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
    if (p.tiles[t].chunks > 0) continue;
    const PagedTile x = p.tiles[t];
    for (int h = 0; h < p.b.Hkv; ++h)
      for (int i = grp; i < 16; i += kGroups) {
        const int r = x.row + blockIdx.y * 16 + i;
        if (r < x.n) store_run(out_row(x, h, r), f32x4{0.f, 0.f, 0.f, 0.f});
      }
  }
  const PagedRun b = p.runs[w];
  if (b.place >= line * p.b.Hkv) return;
  const PagedTile x = p.tiles[b.tile];
  const int a = b.head * line + x.at, end = a + x.chunks;
  if (b.place <= a || b.place >= end) return;
  // borders of the same block before and after this one
  int before = 0, after = 0;
  while (true) {
    const int i = w - 1 - before - lane;
    const int n = __popcll(__ballot(i >= 0 && p.runs[max(i, 0)].place > a));
    before += n;
    if (n < 64) break;
  }
  while (true) {
    const int i = w + 1 + after + lane;
    const int n = __popcll(__ballot(i <= p.workers && p.runs[min(i, p.workers)].place < end));
    after += n;
    if (n < 64) break;
  }
  const int first = w - before, borders = before + 1 + after, parts = borders + 1;
  // the first part is its run's first item if no earlier block has chunks there; the others are
  const int64_t part0 = (int64_t)(2 * (first - 1) + (p.runs[first - 1].place >= a - kTileStart ? 0 : 1)) * BQ;
  auto take = [&](int k, int r, f32x4& o, float& m, float& l) {
    const int64_t s = (k == 0 ? part0 : (int64_t)2 * (first + k - 1) * BQ) + r - x.row;
    const float2 ml = p.part_ml[s];
    const f32x4 y = *reinterpret_cast<const f32x4*>(p.part_o + s * D + 4 * at);
    const float m_new = fmaxf(m, ml.x), ref = m_new == -INFINITY ? 0.f : m_new;
    const float e0 = __builtin_amdgcn_exp2f(m - ref), e1 = __builtin_amdgcn_exp2f(ml.x - ref);
    l = e0 * l + e1 * ml.y;
    o = e0 * o + e1 * y;
    m = m_new;
  };
  if (parts <= (kGroups >= 8 ? kGroups / 2 : 3)) {
    // a row a group, its parts one after another
#pragma unroll
    for (int i0 = 0; i0 < 16; i0 += kGroups) {
      const int i = i0 + grp, r = x.row + blockIdx.y * 16 + i;
      if (i >= 16 || r >= x.n || i % borders != before) continue;
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
      float l = 0.f, m = -INFINITY;
      take(0, r, o, m, l);
      take(1, r, o, m, l);
#pragma unroll 2
      for (int k = 2; k < parts; ++k) take(k, r, o, m, l);
      store_run(out_row(x, b.head, r), o * (l > 0.f ? 1.f / l : 0.f));
    }
    return;
  }
  for (int i = before; i < 16; i += borders) {
    // a row, its parts round the groups
    const int r = x.row + blockIdx.y * 16 + i;
    if (r >= x.n) break;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f, m = -INFINITY;
#pragma unroll 4
    for (int k = grp; k < parts; k += kGroups) take(k, r, o, m, l);
    acc[grp][at] = o;
    if (at == 0) accml[grp] = make_float2(m, l);
    __syncthreads();
    if (grp == 0) {
      float top = m;
      for (int k = 1; k < kGroups; ++k) top = fmaxf(top, accml[k].x);
      const float ref = top == -INFINITY ? 0.f : top, e0 = __builtin_amdgcn_exp2f(m - ref);
      l *= e0;
      o *= e0;
      for (int k = 1; k < kGroups; ++k) {
        const float e = __builtin_amdgcn_exp2f(accml[k].x - ref);
        l += e * accml[k].y;
        o += e * acc[k][at];
      }
      store_run(out_row(x, b.head, r), o * (l > 0.f ? 1.f / l : 0.f));
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------
// Chunks and ring of the step kernel: 16 KB of keys and values a chunk (32 KB at the widest rows), as many
// waves on a CU as its 160 KB of LDS hold.
template <typename T, int D>
struct StepShape {
  static constexpr int kRow = D * (int)sizeof(T);
  static constexpr int KC = kRow <= 128 ? 64 : kRow <= 512 ? 32 : 16;
  static constexpr int ST = kRow * KC * 2 > 16384 ? 2 : 3;
  static constexpr int kLds = ST * 2 * KC * kRow;
  static constexpr int kPerCu = (160 * 1024) / kLds < 8 ? (160 * 1024) / kLds : 8;
  // Chunks that one wave takes whole rather than share them out and join the parts, when there are few
  // sequences and when there is one for each CU (us, whole / shared out: 65 keys x 4 heads fp32 at D 32 6.9 /
  // 10.3; bf16, 2 heads at D 128: 16 x 128 to 256 keys 10.2 / 9.7, 128 x 64 to 256 11.1 / 14.5; 64 x 12 heads x 300
  // to 512 at D 64 17.8 / 23.1; fp32's chunks take twice as long: 4 of 16 keys at D 256 13.7 / 11.7).
  static constexpr int kWholeFew = sizeof(T) == 4 && D >= 128 ? 2 : 4, kWholeMany = 2 * kWholeFew;
};

// Blocks of the tile kernel: 128 rows, two 16-row groups a wave while their outputs fit the registers of
// two waves a SIMD; fp32 64 rows. As many workgroups as LDS and registers hold at a time.
template <typename T, int D>
struct TileShape {
  static constexpr bool kBf = sizeof(T) == 2;
  static constexpr int NW = kBf && D == 256 ? 8 : 4, RG = kBf ? 2 : 1, KC = kBf ? 64 : 32;
  static constexpr bool kPair = kBf && D == 256;
  static constexpr int BQ = 16 * RG * (kPair ? NW / 2 : NW);
  static constexpr int kLds = 4 * KC * D * (int)sizeof(T);
  static constexpr int kPerCu = std::min(160 * 1024 / kLds, kBf ? (D <= 32 ? 4 : D == 64 ? 3 : 2) : D <= 64 ? 4 : 2);
};

static size_t aligned256(size_t x) { return (x + 255) & ~(size_t)255; }

template <typename T, int D>
static int launch_step(tl_ctx* ctx, PagedAttn p) {
  using S = StepShape<T, D>;
  using P = TileShape<T, D>;
  const int64_t g = p.g, rows = std::min<int64_t>(p.max_q * g, 16), heads = (int64_t)p.b.n_rows * p.b.Hq;
  const int64_t blocks16 = (p.max_q * g + 15) / 16;
  const int64_t most = blocks16 * p.b.Hkv * p.b.n_seqs * ((((int64_t)p.b.cols << p.b.page_shift) + S::KC - 1) / S::KC);
  TL_REQUIRE(most < (1LL << 30), "batch too large: sequences x kv heads x table positions");
  const int64_t items = blocks16 * p.b.Hkv * p.b.n_seqs;
  const int cus = ctx->num_cus > 0 ? ctx->num_cus : 256;
  const int whole = items >= cus ? S::kWholeMany : S::kWholeFew;
  if (p.shared == 0 && items < (1LL << 26) && ((int64_t)p.b.cols << p.b.page_shift) <= whole * S::KC) {
    p.skip = 0;
    p.row_blocks = (int)blocks16;
    if (p.cap_in != 0.f) paged_step_kernel<T, D, S::KC, S::ST, true, true><<<(unsigned)items, 64, 0, ctx->stream>>>(p);
    else paged_step_kernel<T, D, S::KC, S::ST, false, true><<<(unsigned)items, 64, 0, ctx->stream>>>(p);
    return TL_OK;
  }
  p.workers = (int)std::max<int64_t>(1, std::min<int64_t>(most, (int64_t)S::kPerCu * cus));
  p.skip = p.shared;
  p.row_blocks = p.splits = 0;
  int64_t blocks = 0, step_blocks = 0;
  constexpr int kRing = 2 * 2 * S::KC * S::kRow, kBlockLds = P::kLds > kRing ? P::kLds : kRing;
  constexpr int kStepWaves = std::min(kBlockLds / kRing, P::NW);  // of a workgroup
  if (p.skip > 0) {
    // The prefix's chunks are split for as many workgroups as are resident, two chunks each at least (us, 64
    // rows x 8 heads x 2048 positions at D 256, with the join: one chunk each 24.6, two 21.3)
    p.row_blocks = (int)((p.b.n_rows * g + P::BQ - 1) / P::BQ);
    const int64_t lines = (int64_t)p.row_blocks * p.b.Hkv, chunks = (p.skip + P::KC - 1) / P::KC;
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(chunks / 2, (int64_t)P::kPerCu * cus / lines));
    blocks = lines * p.splits;
    TL_REQUIRE(blocks < (1LL << 22), "batch too large: row blocks x kv heads");
    const int64_t slots = std::max(1, 160 * 1024 / kBlockLds / 2) * (int64_t)cus;  // half of the chip
    p.workers = (int)std::min<int64_t>(p.workers, slots * kStepWaves);
    step_blocks = (p.workers + kStepWaves - 1) / kStepWaves;
  }
  const int64_t slots = 2LL * p.workers * rows + (p.skip > 0 ? heads : 0), pre = blocks * P::BQ;
  const size_t obytes = aligned256((size_t)slots * D * sizeof(float)), mbytes = aligned256((size_t)slots * sizeof(float2));
  const size_t pbytes = aligned256((size_t)pre * D * sizeof(float));
  void* ws;
  const int rc = workspace(ctx, obytes + mbytes + pbytes + (size_t)pre * sizeof(float2), &ws);
  if (rc) return rc;
  p.part_o = (float*)ws;
  p.part_ml = (float2*)((char*)ws + obytes);
  p.pre_o = (float*)((char*)ws + obytes + mbytes);
  p.pre_ml = (float2*)((char*)ws + obytes + mbytes + pbytes);
  if (p.skip > 0) {
    const int n = (int)((blocks + 7) / 8 * 8), m = (int)((step_blocks + 7) / 8 * 8);
    if (p.cap_in != 0.f)
      paged_shared_kernel<T, D, P::NW, P::RG, P::KC, P::kPair, S::KC, true><<<n + m, 64 * P::NW, 0, ctx->stream>>>(p, n, m);
    else
      paged_shared_kernel<T, D, P::NW, P::RG, P::KC, P::kPair, S::KC, false><<<n + m, 64 * P::NW, 0, ctx->stream>>>(p, n, m);
  } else if (p.cap_in != 0.f) {
    paged_step_kernel<T, D, S::KC, S::ST, true, false><<<p.workers, 64, 0, ctx->stream>>>(p);
  } else {
    paged_step_kernel<T, D, S::KC, S::ST, false, false><<<p.workers, 64, 0, ctx->stream>>>(p);
  }
  const dim3 join((unsigned)p.b.n_rows, (unsigned)((g + 256 / D - 1) / (256 / D)), (unsigned)p.b.Hkv);
  paged_join_kernel<T, D, S::KC, P::BQ><<<join, 256, 0, ctx->stream>>>(p);
  return TL_OK;
}

template <typename T, int D>
static int launch_tiles(tl_ctx* ctx, PagedAttn p) {
  using S = TileShape<T, D>;
  const int64_t g = p.g;
  const int64_t most = std::min<int64_t>(p.b.n_seqs, p.b.n_rows) + (int64_t)p.b.n_rows * g / S::BQ;
  const int64_t line = most * ((((int64_t)p.b.cols << p.b.page_shift) + S::KC - 1) / S::KC + kTileStart);
  // (the second also when the bounds are wrong and sequences claim the same rows)
  TL_REQUIRE(line * p.b.Hkv < (1LL << 30) && p.b.n_seqs * ((p.max_q * g + S::BQ - 1) / S::BQ) < (1LL << 31),
             "batch too large: row blocks x kv heads x table positions");
  const int cus = ctx->num_cus > 0 ? ctx->num_cus : 256;
  p.workers = (int)std::max<int64_t>(8, (int64_t)S::kPerCu * cus / 8 * 8);
  p.most_tiles = (int)most;
  const size_t obytes = aligned256((size_t)p.workers * 2 * S::BQ * D * sizeof(float));
  const size_t mbytes = aligned256((size_t)p.workers * 2 * S::BQ * sizeof(float2));
  const size_t tbytes = aligned256((size_t)most * sizeof(PagedTile));
  void* ws;
  const size_t rbytes = aligned256((size_t)(p.workers + 1) * sizeof(PagedRun));
  const int rc = workspace(ctx, obytes + mbytes + tbytes + rbytes + ((size_t)p.b.n_seqs + 2) * sizeof(int), &ws);
  if (rc) return rc;
  p.part_o = (float*)ws;
  p.part_ml = (float2*)((char*)ws + obytes);
  p.tiles = (PagedTile*)((char*)ws + obytes + mbytes);
  p.runs = (PagedRun*)((char*)ws + obytes + mbytes + tbytes);
  int* total = (int*)((char*)ws + obytes + mbytes + tbytes + rbytes);
  paged_plan_kernel<S::BQ, S::KC><<<1, 1024, 0, ctx->stream>>>(p, total);
  if (p.cap_in != 0.f)
    paged_tile_kernel<T, D, S::NW, S::RG, S::KC, true, S::kPair><<<p.workers, 64 * S::NW, 0, ctx->stream>>>(p, total);
  else
    paged_tile_kernel<T, D, S::NW, S::RG, S::KC, false, S::kPair><<<p.workers, 64 * S::NW, 0, ctx->stream>>>(p, total);
  paged_tile_join_kernel<T, D, S::BQ>
      <<<dim3((unsigned)p.workers, S::BQ / 16), 256, 0, ctx->stream>>>(p, total);
  return TL_OK;
}

// The step kernel reads a sequence's keys once for each 16 rows, the tile kernel once for 128, after a plan and
// with a join that costs more. Up to kStepRows rows the first is taken while what it reads again is little (us,
// step / tile: 24 rows, 2000 keys, D 256 16.6 / 70.7; 48 sequences x 32 rows, 500 to 2048 keys 32.6 / 41.8, 64
// rows 52.0 / 48.5; 6 x 4 heads x 32 rows, 20000 to 60000 keys, D 128 174 / 139). Lengths are not known here:
// what the tables hold stands for them.
constexpr int kStepRows = 128;
constexpr int64_t kStepAgain = 100 << 20;

template <typename T, int D>
static int launch_attention(tl_ctx* ctx, PagedAttn p) {
  const int64_t g = p.g;
  const int64_t rows = p.max_q * g, again = (rows + 15) / 16 - 1;
  const int64_t bytes = ((int64_t)p.b.n_seqs * p.b.cols << p.b.page_shift) * p.b.Hkv * D * 2 * (int64_t)sizeof(T);
  if (rows <= 16 || (rows <= kStepRows && bytes <= kStepAgain / again)) return launch_step<T, D>(ctx, p);
  p.skip = 0;
  return launch_tiles<T, D>(ctx, p);
}

}  // namespace tl

using namespace tl;

extern "C" int tl_paged_attention(tl_ctx* ctx, const tl_paged_desc* desc, const void* q, int64_t ld_q,
                                  void* out, int64_t ld_out, int64_t max_q, float divisor, float softcap,
                                  int64_t window, int64_t shared) {
  int rc = enter(ctx);
  if (rc) return rc;
  PagedAttn p;
  rc = paged_batch(ctx, desc, &p.b);
  if (rc) return rc;
  TL_REQUIRE(divisor > 0.f && divisor < INFINITY, "divisor must be positive and finite");
  TL_REQUIRE(softcap >= 0.f && softcap < INFINITY, "softcap must be 0 or positive and finite");
  TL_REQUIRE(softcap <= 4096.f || desc->dtype != TL_BF16, "a softcap above 4096 is served in fp32 only");
  TL_REQUIRE(max_q > 0, "max_q must be positive");
  TL_REQUIRE(window >= 0, "negative window");
  TL_REQUIRE(shared >= 0 && shared % desc->page_size == 0 && shared <= desc->table_cols * desc->page_size,
             "shared must be whole pages of the table");
  TL_REQUIRE(shared == 0 || window == 0, "a window and a shared prefix exclude each other");
  if (desc->n_rows == 0 || desc->n_seqs == 0) return TL_OK;
  const int64_t D = desc->head_dim, wq = desc->n_heads_q * D;
  rc = paged_rows(desc, q, ld_q, wq, "q");
  if (rc) return rc;
  rc = paged_rows(desc, out, ld_out, wq, "out");
  if (rc) return rc;
  p.q = q; p.k = desc->k_pages; p.v = desc->v_pages; p.out = out;
  p.ld_q = ld_q; p.ld_out = ld_out;
  p.g = p.b.Hq / p.b.Hkv;
  p.max_q = (int)std::min<int64_t>(max_q, desc->n_rows);
  p.window = (int)std::min<int64_t>(window, 1LL << 30);
  p.shared = (int)shared;
  const double log2e = 1.4426950408889634;
  const bool capped = softcap > 0.f, wide = desc->dtype == TL_F32;
  p.scale = (float)(capped ? (wide ? 1.0 : 2.0) * log2e * softcap : log2e / divisor);
  p.cap_in = capped ? (float)((wide ? 1.0 : -2.0 * log2e) / ((double)divisor * softcap)) : 0.f;
  TL_REQUIRE(p.scale >= FLT_MIN && p.scale < INFINITY && std::fabs(p.cap_in) < INFINITY &&
             (!capped || std::fabs(p.cap_in) >= FLT_MIN), "divisor or softcap out of fp32's range");
  p.part_o = nullptr; p.part_ml = nullptr; p.workers = 0;
  const double es = (double)dtype_size(desc->dtype);
  // lengths are known on the device only: the profiler is told of the queries and outputs alone
  LaunchScope ls(ctx, TL_KF_ATTENTION, 0, 2.0 * es * desc->n_rows * wq);
  rc = TL_OK;
  for_head_dim(D, [&](auto dim) {
    constexpr int DD = decltype(dim)::value;
    rc = desc->dtype == TL_F32 ? launch_attention<float, DD>(ctx, p) : launch_attention<bf16_t, DD>(ctx, p);
  });
  if (rc) return rc;
  return ls.finish("paged_attention");
}
