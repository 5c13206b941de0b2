// The append of a ragged batch's QKV rows to a paged KV cache.
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

int paged_rows(const tl_paged_desc* d, const void* p, int64_t ld, int64_t cols, const char* what) {
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
// Rows of a workgroup; each wave finds the place of one row of four.
constexpr int kAppendRows = 4;

// One thread per 16-byte chunk of a head's first half and its partner in the second half: it
// rotates both by the row's position, or copies them (values, and keys without a table). HBM is the bound:
// 9151 rows, 8 / 1 heads at D 256 in bf16, 21 us (4.6 TB/s), fp32 without a table 8.7 us (5.1 TB/s); 32 rows
// take 5 us, a launch and two reads one after the other before the rows.
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

}  // namespace tl

using namespace tl;

extern "C" int tl_kv_append(tl_ctx* ctx, const tl_paged_desc* desc, const void* qkv, int64_t ld_qkv,
                            void* q_out, int64_t ld_q, const void* rope_table, int64_t rope_rows) {
  int rc = enter(ctx);
  if (rc) return rc;
  PagedBatch b;
  rc = paged_batch(ctx, desc, &b);
  if (rc) return rc;
  const int64_t D = desc->head_dim, wq = desc->n_heads_q * D, w = wq + 2 * desc->n_heads_kv * D;
  if (desc->n_rows == 0 || desc->n_seqs == 0) return TL_OK;
  rc = paged_rows(desc, qkv, ld_qkv, w, "qkv");
  if (rc) return rc;
  const double es = (double)dtype_size(desc->dtype);
  if (rope_table) {
    TL_REQUIRE(rope_rows > 0 && rope_rows <= (1LL << 30), "bad RoPE table length");
    TL_REQUIRE(((uintptr_t)rope_table & 15u) == 0, "the RoPE table must be 16-byte aligned");
    rc = paged_rows(desc, q_out, ld_q, wq, "q_out");
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
