// Ragged serving over a paged KV cache: the append of a QKV product's rows to the pages, and the
// attention that reads them.
#include <algorithm>

#include "paged.hpp"

namespace tl {

// ---------------------------------------------------------------------------------------
// batches
// ---------------------------------------------------------------------------------------
int paged_batch(tl_ctx* ctx, const tl_paged_desc* d, PagedBatch* b) {
  TL_REQUIRE(d, "null descriptor");
  TL_REQUIRE(dtype_is_float(d->dtype), "a paged cache holds fp32 or bf16");
  TL_REQUIRE(d->n_seqs >= 0 && d->n_rows >= 0 && d->n_pages >= 0, "negative size");
  TL_REQUIRE(d->n_heads_q > 0 && d->n_heads_kv > 0 && d->n_heads_q % d->n_heads_kv == 0,
             "bad head configuration");
  if (!(d->head_dim == 32 || d->head_dim == 64 || d->head_dim == 128 || d->head_dim == 256))
    return fail(TL_ERR_UNSUPPORTED, "a paged cache supports head_dim 32, 64, 128, 256");
  int shift = 4;
  while (shift < 12 && (1LL << shift) < d->page_size) ++shift;
  TL_REQUIRE((1LL << shift) == d->page_size, "page_size must be a power of two from 16 to 4096");
  TL_REQUIRE(d->n_heads_q <= 4096, "more than 4096 heads");
  TL_REQUIRE(d->n_rows < (1LL << 24) && d->n_seqs < (1LL << 20) && d->n_rows * d->n_heads_q < (1LL << 30),
             "batch too large");
  TL_REQUIRE(d->n_pages < (1LL << 31), "too many pages");
  TL_REQUIRE(d->table_cols >= 0 && d->table_cols <= d->ld_table && d->table_cols * d->page_size <= (1LL << 30),
             "bad page table shape");
  if (d->n_seqs > 0 && d->n_rows > 0) {
    TL_REQUIRE(d->k_pages && d->v_pages && d->page_table && d->q_start && d->kv_len, "null pointer");
    TL_REQUIRE(d->n_pages > 0 && d->table_cols > 0, "no pages");
    TL_REQUIRE((((uintptr_t)d->k_pages | (uintptr_t)d->v_pages) & 15u) == 0, "pages must be 16-byte aligned");
    TL_REQUIRE((((uintptr_t)d->page_table | (uintptr_t)d->q_start | (uintptr_t)d->kv_len) & 3u) == 0,
               "tables must be 4-byte aligned");
  }
  b->table = d->page_table; b->q_start = d->q_start; b->kv_len = d->kv_len;
  b->ld_table = d->ld_table; b->cols = (int)d->table_cols; b->n_seqs = (int)d->n_seqs;
  b->n_rows = (int)d->n_rows; b->n_pages = (int)d->n_pages; b->page_shift = shift;
  b->Hq = (int)d->n_heads_q; b->Hkv = (int)d->n_heads_kv;
  b->status = ctx->status;
  return TL_OK;
}

// A tensor of d->n_rows rows: 16-byte aligned rows that do not overlap.
static int check_rows(const tl_paged_desc* d, const void* p, int64_t ld, int64_t cols, const char* what) {
  TL_REQUIRE(p, "null pointer");
  TL_REQUIRE(ld >= cols, "row pitch of %s smaller than its %lld columns", what, (long long)cols);
  const int64_t vec = 16 / (int64_t)dtype_size(d->dtype);
  TL_REQUIRE(((uintptr_t)p & 15u) == 0 && (d->n_rows == 1 || ld % vec == 0), "rows of %s must be 16-byte aligned",
             what);
  TL_REQUIRE(ld < (1LL << 31), "row pitch of %s too large", what);
  return TL_OK;
}

// ---------------------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------------------
// The sequence that row t belongs to, by a whole wave: the last s with q_start[s] <= t, found by
// 64 probes a round (one round up to 64 sequences, two up to 4096). n_seqs for a row of none.
__device__ __forceinline__ int seq_of_row(const PagedBatch& b, int t, int lane) {
  int lo = 0, n = b.n_seqs;  // q_start[lo] <= t as far as probed; the answer is in [lo, lo + n)
  int hits = 0;
  while (true) {
    const int step = (n + 63) >> 6;
    const int at = lo + (lane + 1) * step;
    const bool hit = at <= lo + n && at <= b.n_seqs && b.q_start[at] <= t;
    hits = __popcll(__ballot(hit));
    if (step == 1) break;
    lo += hits * step;
    n = min(step, b.n_seqs - lo);
    if (n <= 0) break;
  }
  return min(lo + (n > 0 ? hits : 0), b.n_seqs);
}

// Rows of a workgroup; each wave finds the place of one row of four.
constexpr int kAppendRows = 4;

// One thread per 16-byte chunk of a head's first half and its partner in the second half: it
// rotates both by the row's position, or copies them (values, and keys without a table).
template <typename T, int D>
__global__ __launch_bounds__(256) void kv_append_kernel(PagedBatch b, const T* __restrict__ qkv, int64_t ld,
                                                        T* __restrict__ k_pages, T* __restrict__ v_pages,
                                                        T* __restrict__ q_out, int64_t ld_q,
                                                        const float* __restrict__ rope, int rope_rows) {
  constexpr int VEC = Elem<T>::kVec, HALF = D / 2, CH = HALF / VEC;  // chunk pairs per head
  __shared__ int64_t place[kAppendRows];  // offset of the row's slot in head 0 of its page, -1: nowhere
  __shared__ int posn[kAppendRows];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  {
    const int t = blockIdx.x * kAppendRows + wave;
    int64_t at = -1;
    int pos = 0;
    if (t < b.n_rows) {
      const int s = seq_of_row(b, t, lane);
      if (s < b.n_seqs) {
        const PagedSeq q = paged_seq(b, s, lane == 0);
        pos = q.len - q.n + (t - q.row0);
        if (t >= q.row0 && t < q.row0 + q.n && pos >= 0) {
          if (rope && pos >= rope_rows) {
            if (lane == 0) latch(b.status, kBadPosition);
          } else {
            const int id = b.table[s * b.ld_table + (pos >> b.page_shift)];
            if ((uint32_t)id < (uint32_t)b.n_pages)
              at = ((((int64_t)id * b.Hkv) << b.page_shift) + (pos & ((1 << b.page_shift) - 1))) * D;
            else if (lane == 0) latch(b.status, kBadPage);
          }
        }
      }
    }
    if (lane == 0) {
      place[wave] = at;
      posn[wave] = pos;
    }
  }
  __syncthreads();
  const int first = rope ? 0 : b.Hq;  // queries that are not rotated stay where they are
  const int units = (b.Hq + 2 * b.Hkv - first) * CH;
  for (int u = tid; u < kAppendRows * units; u += 256) {
    const int r = u / units, x = u - r * units;
    const int h = first + x / CH, c = (x % CH) * VEC;
    const int64_t at = place[r];
    if (at < 0) continue;
    const int64_t t = (int64_t)blockIdx.x * kAppendRows + r;
    const T* src = qkv + t * ld + h * D + c;
    uint4 lo = *reinterpret_cast<const uint4*>(src), hi = *reinterpret_cast<const uint4*>(src + HALF);
    T* dst;
    if (h < b.Hq) dst = q_out + t * ld_q + h * D;
    else if (h < b.Hq + b.Hkv) dst = k_pages + at + ((int64_t)(h - b.Hq) << b.page_shift) * D;
    else dst = v_pages + at + ((int64_t)(h - b.Hq - b.Hkv) << b.page_shift) * D;
    if (rope && h < b.Hq + b.Hkv) {
      const float* cs = rope + (int64_t)posn[r] * HALF + c;
      float a[VEC], e[VEC], ra[VEC], re[VEC];
      Elem<T>::unpack(lo, a);
      Elem<T>::unpack(hi, e);
#pragma unroll
      for (int i = 0; i < VEC; i += 4) {
        const float4 co = *reinterpret_cast<const float4*>(cs + i);
        const float4 si = *reinterpret_cast<const float4*>(cs + (int64_t)rope_rows * HALF + i);
        const float cv[4] = {co.x, co.y, co.z, co.w}, sv[4] = {si.x, si.y, si.z, si.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          ra[i + j] = a[i + j] * cv[j] - e[i + j] * sv[j];
          re[i + j] = e[i + j] * cv[j] + a[i + j] * sv[j];
        }
      }
      lo = Elem<T>::pack(ra);
      hi = Elem<T>::pack(re);
    }
    *reinterpret_cast<uint4*>(dst + c) = lo;
    *reinterpret_cast<uint4*>(dst + c + HALF) = hi;
  }
}

__global__ void i32_add_kernel(int32_t* x, int64_t n, int32_t delta) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n) x[i] += delta;
}

// ---------------------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------------------
struct PagedAttn {
  PagedBatch b;
  const void* q;
  const void* k;
  const void* v;
  void* out;
  int64_t ld_q, ld_out;
  int max_q, window, shared;  // window 0: none
  float divisor, cap;
};

// One wave per (row, query head): each lane takes a key of 64, then an element of the output.
template <typename T, int D>
__global__ __launch_bounds__(64) void paged_attention_simple_kernel(PagedAttn p) {
  __shared__ float qs[D];
  const int lane = threadIdx.x;
  const int t = blockIdx.x / p.b.Hq, h = blockIdx.x % p.b.Hq;
  const int s = seq_of_row(p.b, t, lane);
  if (s >= p.b.n_seqs) return;
  const PagedSeq q = paged_seq(p.b, s, lane == 0);
  const int i = t - q.row0;
  if (i < 0 || i >= q.n) return;
  if (p.shared > 0) check_shared(p.b, s, q, p.shared, lane);
  if (i >= p.max_q) {
    if (lane == 0) latch(p.b.status, kBadSequence);
    return;
  }
  const int pos = q.len - q.n + i;
  const int first = p.window > 0 ? max(0, pos - p.window + 1) : 0;
  const int32_t* row = p.b.table + s * p.b.ld_table;
  const T* qr = (const T*)p.q + t * p.ld_q + h * D;
  for (int d = lane; d < D; d += 64) qs[d] = Elem<T>::load(qr + d);
  __syncthreads();
  const int hk = h / (p.b.Hq / p.b.Hkv), mask = (1 << p.b.page_shift) - 1;
  constexpr int E = (D + 63) / 64;
  float o[E] = {}, m = -INFINITY, l = 0.f;
  for (int j0 = first; j0 <= pos; j0 += 64) {
    const int j = j0 + lane;
    float sc = -INFINITY;
    int64_t at = 0;
    if (j <= pos) {
      const int64_t page = paged_page(p.b, row, j, true);
      at = (((page * p.b.Hkv + hk) << p.b.page_shift) + (j & mask)) * D;
      float a = 0.f;
      for (int d = 0; d < D; ++d) a += qs[d] * Elem<T>::load((const T*)p.k + at + d);
      sc = a / p.divisor;
      if (p.cap > 0.f) sc = p.cap * tanhf(sc / p.cap);
    }
    const float mn = fmaxf(m, wave_max(sc));
    const float e = expf(sc - mn), al = expf(m - mn);
    l = l * al + wave_sum(e);
    m = mn;
#pragma unroll
    for (int x = 0; x < E; ++x) o[x] *= al;
    const int n = min(64, pos + 1 - j0);
    for (int y = 0; y < n; ++y) {
      const float w = __shfl(e, y, 64);
      const int64_t a = (int64_t)__shfl((long long)at, y, 64);
#pragma unroll
      for (int x = 0; x < E; ++x)
        if (x * 64 + lane < D) o[x] += w * Elem<T>::load((const T*)p.v + a + x * 64 + lane);
    }
  }
  T* orow = (T*)p.out + t * p.ld_out + h * D;
#pragma unroll
  for (int x = 0; x < E; ++x)
    if (x * 64 + lane < D) Elem<T>::store(orow + x * 64 + lane, l > 0.f ? o[x] / l : 0.f);
}

}  // namespace tl

using namespace tl;

// Calls f with a D of the descriptor's head_dim as a type.
template <int D>
struct HeadDim {
  static constexpr int value = D;
};
template <typename F>
static void for_head_dim(int64_t d, F f) {
  switch (d) {
    case 32: f(HeadDim<32>{}); break;
    case 64: f(HeadDim<64>{}); break;
    case 128: f(HeadDim<128>{}); break;
    default: f(HeadDim<256>{}); break;
  }
}

extern "C" int tl_kv_append(tl_ctx* ctx, const tl_paged_desc* desc, const void* qkv, int64_t ld_qkv,
                            void* q_out, int64_t ld_q, const void* rope_table, int64_t rope_rows) {
  int rc = enter(ctx);
  if (rc) return rc;
  PagedBatch b;
  rc = paged_batch(ctx, desc, &b);
  if (rc) return rc;
  const int64_t D = desc->head_dim, wq = desc->n_heads_q * D, w = wq + 2 * desc->n_heads_kv * D;
  if (desc->n_rows == 0 || desc->n_seqs == 0) return TL_OK;
  rc = check_rows(desc, qkv, ld_qkv, w, "qkv");
  if (rc) return rc;
  const double es = (double)dtype_size(desc->dtype);
  if (rope_table) {
    TL_REQUIRE(rope_rows > 0 && rope_rows <= (1LL << 30), "bad RoPE table length");
    TL_REQUIRE(((uintptr_t)rope_table & 15u) == 0, "the RoPE table must be 16-byte aligned");
    rc = check_rows(desc, q_out, ld_q, wq, "q_out");
    if (rc) return rc;
    const uintptr_t x = (uintptr_t)qkv, y = (uintptr_t)q_out;
    const uintptr_t xe = x + (uintptr_t)(((desc->n_rows - 1) * ld_qkv + w) * es);
    const uintptr_t ye = y + (uintptr_t)(((desc->n_rows - 1) * ld_q + wq) * es);
    TL_REQUIRE(xe <= y || ye <= x, "q_out overlaps qkv");
  } else {
    TL_REQUIRE(!q_out && rope_rows == 0, "queries are written only with a RoPE table");
  }
  const double moved = (double)desc->n_rows * ((rope_table ? wq : 0) + 2 * desc->n_heads_kv * D);
  LaunchScope ls(ctx, TL_KF_ROPE, 0, 2.0 * es * moved);
  const unsigned grid = (unsigned)((desc->n_rows + kAppendRows - 1) / kAppendRows);
  for_head_dim(D, [&](auto dim) {
    constexpr int DD = decltype(dim)::value;
    if (desc->dtype == TL_F32)
      kv_append_kernel<float, DD><<<grid, 256, 0, ctx->stream>>>(
          b, (const float*)qkv, ld_qkv, (float*)desc->k_pages, (float*)desc->v_pages, (float*)q_out, ld_q,
          (const float*)rope_table, (int)rope_rows);
    else
      kv_append_kernel<bf16_t, DD><<<grid, 256, 0, ctx->stream>>>(
          b, (const bf16_t*)qkv, ld_qkv, (bf16_t*)desc->k_pages, (bf16_t*)desc->v_pages, (bf16_t*)q_out, ld_q,
          (const float*)rope_table, (int)rope_rows);
  });
  return ls.finish("kv_append");
}

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
  TL_REQUIRE(max_q > 0, "max_q must be positive");
  TL_REQUIRE(window >= 0, "negative window");
  TL_REQUIRE(shared >= 0 && shared % desc->page_size == 0 && shared <= desc->table_cols * desc->page_size,
             "shared must be whole pages of the table");
  TL_REQUIRE(shared == 0 || window == 0, "a window and a shared prefix exclude each other");
  if (desc->n_rows == 0 || desc->n_seqs == 0) return TL_OK;
  const int64_t D = desc->head_dim, wq = desc->n_heads_q * D;
  rc = check_rows(desc, q, ld_q, wq, "q");
  if (rc) return rc;
  rc = check_rows(desc, out, ld_out, wq, "out");
  if (rc) return rc;
  p.q = q; p.k = desc->k_pages; p.v = desc->v_pages; p.out = out;
  p.ld_q = ld_q; p.ld_out = ld_out;
  p.max_q = (int)std::min<int64_t>(max_q, desc->n_rows);
  p.window = (int)std::min<int64_t>(window, 1LL << 30);
  p.shared = (int)shared;
  p.divisor = divisor; p.cap = softcap;
  const double es = (double)dtype_size(desc->dtype);
  // lengths are known on the device only: the profiler is told of the queries and outputs alone
  LaunchScope ls(ctx, TL_KF_ATTENTION, 0, 2.0 * es * desc->n_rows * wq);
  const unsigned grid = (unsigned)(desc->n_rows * desc->n_heads_q);
  for_head_dim(D, [&](auto dim) {
    constexpr int DD = decltype(dim)::value;
    if (desc->dtype == TL_F32) paged_attention_simple_kernel<float, DD><<<grid, 64, 0, ctx->stream>>>(p);
    else paged_attention_simple_kernel<bf16_t, DD><<<grid, 64, 0, ctx->stream>>>(p);
  });
  return ls.finish("paged_attention");
}

extern "C" int tl_i32_add(tl_ctx* ctx, int32_t* x, int64_t n, int32_t delta) {
  int rc = enter(ctx);
  if (rc) return rc;
  TL_REQUIRE(n >= 0 && n < (1LL << 31), "bad size");
  if (n == 0) return TL_OK;
  TL_REQUIRE(x && ((uintptr_t)x & 3u) == 0, "null or unaligned pointer");
  LaunchScope ls(ctx, TL_KF_MISC, 0, 8.0 * n);
  i32_add_kernel<<<(unsigned)((n + 255) / 256), 256, 0, ctx->stream>>>(x, n, delta);
  return ls.finish("i32_add");
}
