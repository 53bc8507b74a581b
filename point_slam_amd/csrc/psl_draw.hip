// Draws of indices from rows of scores: temperature, top-k, top-p, min-p, and the caller's random numbers (psl_draw_indices).
//
// With M the largest allowed score of a row, an entry weighs w = exp((s - M) / T).  Entries are ordered by (score descending,
// index ascending); top-k and top-p keep prefixes of that order, so both are ONE threshold on the 64-bit number
// (ordered bits of the score, ~index): an entry is kept iff its number is at least the threshold, and w >= min_p.  A draw
// is the lowest index whose running sum of kept weights, in index order, passes u * (sum of all).
//
// Which index a u selects is decided by sums of up to a million weights: weights and sums are fp64, and every sum has one
// fixed order (or is a sum of integers), so that a call's answer does not depend on the schedule.
#include "psl_common.h"

namespace psl {

typedef unsigned long long u64;

struct DrawArgs {
  int n_rows, n_cols, n_draws;
  const void* scores; long long stride;
  const unsigned char* mask; long long mask_stride;
  const float* temperature; const int* top_k; const float* top_p; const float* min_p;
  double t_all, p_all, m_all; int k_all;
  const float* u; long long u_stride;
  int* idx; float* prob;
  // workspace
  struct DrawState* state;     // [n_rows]
  double* chunk_sum;           // [n_rows][n_chunks]
  double* block_incl;          // [n_rows][n_chunks * chunk / 16]: running sums inside a chunk, at the end of each 16 entries
  int n_chunks, chunk;         // entries of a chunk (a multiple of kTile)
};
struct DrawState {
  u64 thr;                     // kept: number(entry) >= thr
  float M; int any;            // largest allowed score; whether there is one
};

constexpr int kBlock = 16;     // entries to a stored running sum: one 64-byte line of fp32 scores
constexpr int kTile = 4096;    // entries that a workgroup of k_draw_sums takes per step
constexpr int kMaxChunks = 1024;

// ---- an entry's order: excluded entries (masked, NaN, -inf) are 0, everything else grows with the score; -0 == +0
__device__ __forceinline__ unsigned key_of(float s) {
  if (!(s > -__builtin_inff())) return 0u;
  const unsigned b = __float_as_uint(s + 0.f);
  return (b >> 31) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float score_of(unsigned key) { return __uint_as_float((key >> 31) ? (key & 0x7fffffffu) : ~key); }
__device__ __forceinline__ u64 number_of(unsigned key, int i) { return ((u64)key << 32) | (unsigned)~i; }

template <int DT> __device__ __forceinline__ float load_score(const void* p, long long i) {
  if constexpr (DT == PSL_F32) return ((const float*)p)[i];
  else if constexpr (DT == PSL_BF16) return __uint_as_float((unsigned)((const unsigned short*)p)[i] << 16);
  else return (float)((const _Float16*)p)[i];
}
struct RowView { const void* s; const unsigned char* m; };
template <int DT> __device__ __forceinline__ RowView row_view(const DrawArgs& a, int r) {
  constexpr int es = DT == PSL_F32 ? 4 : 2;
  return RowView{(const char*)a.scores + (long long)r * a.stride * es, a.mask ? a.mask + (long long)r * a.mask_stride : nullptr};
}
template <int DT> __device__ __forceinline__ unsigned entry_key(const RowView& v, int i) {
  if (v.m && !v.m[i]) return 0u;
  return key_of(load_score<DT>(v.s, i));
}

struct RowPar { double inv_t, p, m; int k; };      // k <= 0: no limit; p >= 1: no limit
__device__ __forceinline__ RowPar row_par(const DrawArgs& a, int r) {
  RowPar q;
  const double t = a.temperature ? (double)a.temperature[r] : a.t_all;
  q.k = a.top_k ? a.top_k[r] : a.k_all;
  q.p = a.top_p ? (double)a.top_p[r] : a.p_all;
  q.m = a.min_p ? (double)a.min_p[r] : a.m_all;
  if (!(q.p < 1.0)) q.p = 1.0;
  if (!(q.m > 0.0)) q.m = 0.0;
  q.m = q.m > 1.0 ? 1.0 : q.m;
  // no temperature, or nothing but the first entry asked for: the first of the order, whatever the weights
  if (!(t > 0.0) || q.p <= 0.0) q.k = 1;
  q.inv_t = t > 0.0 ? 1.0 / t : 1.0;
  return q;
}
// weight of an allowed score; +inf among the scores takes all
__device__ __forceinline__ double weight_of(float s, float M, double inv_t) {
  if (s == M) return 1.0;
  if (M == __builtin_inff()) return 0.0;
  return exp(((double)s - (double)M) * inv_t);
}

__device__ __forceinline__ double shfl_up_d(double v, int o) { return __shfl_up(v, o); }

// ---------------------------------------------------------------- the threshold of a row, by radix selection
// 256 bins of (count, mass): masses are summed as integers, 32 bits before and 32 behind the point at 2^-32, so their sum has no order
struct RadixBins { unsigned cnt[256]; u64 hi[256], lo[256]; };
struct RadixPick { int bin; unsigned above, count; double mass_above, mass; };

__device__ __forceinline__ void radix_zero(RadixBins& b) {
  for (int j = threadIdx.x; j < 256; j += blockDim.x) { b.cnt[j] = 0; b.hi[j] = 0; b.lo[j] = 0; }
}
__device__ __forceinline__ double fixed_d(u64 hi, u64 lo) { return (double)hi * 0x1p-32 + (double)lo * 0x1p-64; }

// wavefront 0, all lanes: the first bin from the top where the running count (by_mass: mass) reaches `want`
__device__ __forceinline__ RadixPick radix_pick(const RadixBins& b, bool by_mass, unsigned want_n, double want_m) {
  const int lane = threadIdx.x & 63;
  unsigned c[4], cs = 0; double m[4], ms = 0.0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int bin = 255 - (4 * lane + j);
    c[j] = b.cnt[bin]; m[j] = fixed_d(b.hi[bin], b.lo[bin]);
    cs += c[j]; ms += m[j];
  }
  unsigned ci = cs; double mi = ms;
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned cu = __shfl_up(ci, o); const double mu = shfl_up_d(mi, o);
    if (lane >= o) { ci += cu; mi += mu; }
  }
  unsigned above = ci - cs; double mabove = __shfl_up(mi, 1);
  if (lane == 0) mabove = 0.0;
  int at = -1, last = -1;
  RadixPick mine{0, 0u, 0u, 0.0, 0.0}, tail{0, 0u, 0u, 0.0, 0.0};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const RadixPick here{255 - (4 * lane + j), above, c[j], mabove, m[j]};
    if (c[j]) { last = j; tail = here; }
    const bool hit = c[j] && (by_mass ? mabove + m[j] >= want_m : above + c[j] >= want_n);
    if (hit && at < 0) { at = j; mine = here; }
    above += c[j]; mabove += m[j];
  }
  const u64 hits = __ballot(at >= 0), some = __ballot(last >= 0);
  // rounding may leave the wanted mass a hair above the sum: then the last entry there is
  const int src = hits ? __ffsll((long long)hits) - 1 : some ? 63 - __clzll((long long)some) : 0;
  const RadixPick send = hits ? mine : tail;
  RadixPick r;
  r.bin = __shfl(send.bin, src); r.above = __shfl(send.above, src); r.count = __shfl(send.count, src);
  r.mass_above = __shfl(send.mass_above, src); r.mass = __shfl(send.mass, src);
  return r;
}

// One workgroup to a row.  Digits of eight bits of the entry's 64-bit number, from the top; a level counts the entries
// whose higher digits are the ones found so far.  Stops as soon as the bin found is taken whole.
template <int DT> __global__ __launch_bounds__(1024) void k_draw_select(DrawArgs a) {
  __shared__ RadixBins bins;
  __shared__ unsigned s_max[16], s_cnt[16];
  __shared__ RadixPick s_pick;
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const RowView v = row_view<DT>(a, r);
  const RowPar par = row_par(a, r);
  unsigned top = 0, cnt = 0;
  for (int i = tid; i < a.n_cols; i += 1024) {
    const unsigned k = entry_key<DT>(v, i);
    top = k > top ? k : top; cnt += k ? 1u : 0u;
  }
  for (int o = 32; o > 0; o >>= 1) { const unsigned t = __shfl_xor(top, o); top = t > top ? t : top; cnt += __shfl_xor(cnt, o); }
  if (lane == 0) { s_max[tid >> 6] = top; s_cnt[tid >> 6] = cnt; }
  __syncthreads();
  top = 0; cnt = 0;
  for (int j = 0; j < 16; ++j) { top = s_max[j] > top ? s_max[j] : top; cnt += s_cnt[j]; }
  const float M = score_of(top);
  u64 thr = 1ull << 32;                             // every allowed entry
  if (top && par.k > 0 && (unsigned)par.k < cnt) {
    unsigned want = (unsigned)par.k;
    u64 prefix = 0;
    for (int shift = 56; shift >= 0; shift -= 8) {
      __syncthreads(); radix_zero(bins); __syncthreads();
      for (int i = tid; i < a.n_cols; i += 1024) {
        const unsigned k = entry_key<DT>(v, i);
        const u64 num = number_of(k, i);
        if (k && (shift == 56 || (num >> (shift + 8)) == prefix)) atomicAdd(&bins.cnt[(num >> shift) & 255], 1u);
      }
      __syncthreads();
      if (tid < 64) { const RadixPick p = radix_pick(bins, false, want, 0.0); if (tid == 0) s_pick = p; }
      __syncthreads();
      const RadixPick p = s_pick;
      prefix = (prefix << 8) | (unsigned)p.bin;
      want -= p.above;
      thr = prefix << shift;
      if (want == p.count) break;
    }
  }
  const u64 thr_k = thr;
  if (top && par.p < 1.0 && par.k != 1) {
    double above = 0.0, want = 0.0;
    u64 prefix = 0;
    unsigned ties = 0;                              // > 0: inside entries of one score, counted instead of weighed
    for (int shift = 56; shift >= 0; shift -= 8) {
      __syncthreads(); radix_zero(bins); __syncthreads();
      for (int i = tid; i < a.n_cols; i += 1024) {
        const unsigned k = entry_key<DT>(v, i);
        const u64 num = number_of(k, i);
        if (k && num >= thr_k && (shift == 56 || (num >> (shift + 8)) == prefix)) {
          const int bin = (int)((num >> shift) & 255);
          atomicAdd(&bins.cnt[bin], 1u);
          if (shift >= 32) {
            const double w = weight_of(score_of(k), M, par.inv_t) * 0x1p32;
            const u64 hi = (u64)w;
            atomicAdd(&bins.hi[bin], hi);
            atomicAdd(&bins.lo[bin], (u64)((w - (double)hi) * 0x1p32));
          }
        }
      }
      __syncthreads();
      if (shift == 56) {
        u64 hi = 0, lo = 0;
        for (int j = 0; j < 256; ++j) { hi += bins.hi[j]; lo += bins.lo[j]; }
        want = par.p * fixed_d(hi, lo);
      }
      if (tid < 64) { const RadixPick p = radix_pick(bins, shift >= 32, ties, want - above); if (tid == 0) s_pick = p; }
      __syncthreads();
      const RadixPick p = s_pick;
      prefix = (prefix << 8) | (unsigned)p.bin;
      thr = prefix << shift;
      if (shift >= 32) {
        above += p.mass_above;
        if (p.count == 1) break;
        if (shift == 32) {
          // p.count entries of one score are left: as many of them as the mass still wants, at least one
          const double n = ceil((want - above) / weight_of(score_of((unsigned)prefix), M, par.inv_t));
          ties = n < 1.0 ? 1u : n < (double)p.count ? (unsigned)n : p.count;
          if (ties == p.count) break;
        }
      } else {
        ties -= p.above;
        if (ties == p.count) break;
      }
    }
  }
  // (the lower end of the bin found may lie below what top-k keeps)
  if (tid == 0) a.state[r] = DrawState{thr > thr_k ? thr : thr_k, M, top ? 1 : 0};
}

// ---------------------------------------------------------------- running sums of the kept weights
template <int DT> __device__ __forceinline__ double kept_weight(const RowView& v, int i, const DrawState& st, const RowPar& par) {
  const unsigned k = entry_key<DT>(v, i);
  if (number_of(k, i) < st.thr) return 0.0;
  const double w = weight_of(score_of(k), st.M, par.inv_t);
  return w >= par.m ? w : 0.0;
}

// One workgroup to a chunk: four entries to a lane, four lanes to a block of 16.
template <int DT> __global__ __launch_bounds__(256) void k_draw_sums(DrawArgs a) {
  __shared__ double blk[kTile / kBlock];
  __shared__ double wsum[4];
  const int r = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const RowView v = row_view<DT>(a, r);
  const DrawState st = a.state[r];
  const RowPar par = row_par(a, r);
  double carry = 0.0;
  const int per_chunk = a.chunk / kBlock;
  double* out = a.block_incl + ((long long)r * a.n_chunks + blockIdx.x) * per_chunk;
  for (int t0 = 0; t0 < a.chunk; t0 += kTile) {
    const long long base = (long long)blockIdx.x * a.chunk + t0;
    if (base >= a.n_cols) break;                    // (uniform; nothing reads the sums behind the row's end)
    for (int j = 0; j < kTile / 1024; ++j) {
      const long long e = base + j * 1024 + tid * 4;
      double w = 0.0;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (e + q < a.n_cols) w += kept_weight<DT>(v, (int)(e + q), st, par);
      w += __shfl_xor(w, 1);
      w += __shfl_xor(w, 2);
      if ((tid & 3) == 0) blk[j * 64 + (tid >> 2)] = w;
    }
    __syncthreads();
    // inclusive sums over the tile's 256 blocks, one to a thread
    double s = blk[tid];
    for (int o = 1; o < 64; o <<= 1) { const double t = shfl_up_d(s, o); if (lane >= o) s += t; }
    if (lane == 63) wsum[tid >> 6] = s;
    __syncthreads();
    double before = carry;
    for (int j = 0; j < (tid >> 6); ++j) before += wsum[j];
    s += before;
    out[t0 / kBlock + tid] = s;
    carry = ((((carry + wsum[0]) + wsum[1]) + wsum[2]) + wsum[3]);
    __syncthreads();
  }
  if (tid == 0) a.chunk_sum[(long long)r * a.n_chunks + blockIdx.x] = carry;
}

// ---------------------------------------------------------------- the draws: a thread to a draw
template <int DT> __global__ __launch_bounds__(256) void k_draw_pick(DrawArgs a) {
  __shared__ double incl[kMaxChunks];
  __shared__ double wsum[4];
  const int r = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const long long d = (long long)blockIdx.x * 256 + tid;
  const DrawState st = a.state[r];
  const int nc = a.n_chunks;
  if (!st.any) {
    if (d < a.n_draws) { a.idx[(long long)r * a.n_draws + d] = -1; if (a.prob) a.prob[(long long)r * a.n_draws + d] = 0.f; }
    return;
  }
  // running sums over the row's chunks, four to a thread
  double c[4], s = 0.0;
#pragma unroll
  for (int j = 0; j < 4; ++j) { const int k = 4 * tid + j; c[j] = k < nc ? a.chunk_sum[(long long)r * nc + k] : 0.0; s += c[j]; c[j] = s; }
  double t = s;
  for (int o = 1; o < 64; o <<= 1) { const double x = shfl_up_d(t, o); if (lane >= o) t += x; }
  double before = __shfl_up(t, 1);
  if (lane == 0) before = 0.0;
  if (lane == 63) wsum[tid >> 6] = t;
  __syncthreads();
  for (int j = 0; j < (tid >> 6); ++j) before += wsum[j];
#pragma unroll
  for (int j = 0; j < 4; ++j) incl[4 * tid + j] = before + c[j];
  __syncthreads();
  if (d >= a.n_draws) return;
  const double total = incl[kMaxChunks - 1];
  double u = (double)a.u[(long long)r * a.u_stride + d];
  u = u > 0.0 ? (u < 1.0 ? u : 1.0 - 0x1p-24) : 0.0;
  const double target = u * total;
  // first chunk whose running sum passes the target (the last one that adds anything, should rounding leave none)
  int lo = 0, hi = nc - 1;
  while (lo < hi) { const int mid = (lo + hi) >> 1; if (incl[mid] > target || incl[mid] >= total) hi = mid; else lo = mid + 1; }
  const double in_chunk = target - (lo ? incl[lo - 1] : 0.0);
  const int per_chunk = a.chunk / kBlock;
  const double* bi = a.block_incl + ((long long)r * nc + lo) * per_chunk;
  const long long first = (long long)lo * a.chunk;
  const long long left = a.n_cols - first;
  const int nb = (int)(((left < a.chunk ? left : a.chunk) + kBlock - 1) / kBlock);
  const double chunk_total = a.chunk_sum[(long long)r * nc + lo];
  int b0 = 0, b1 = nb - 1;
  while (b0 < b1) { const int mid = (b0 + b1) >> 1; const double x = bi[mid]; if (x > in_chunk || x >= chunk_total) b1 = mid; else b0 = mid + 1; }
  const double in_block = in_chunk - (b0 ? bi[b0 - 1] : 0.0);
  const RowView v = row_view<DT>(a, r);
  const RowPar par = row_par(a, r);
  const int i0 = (int)(first + (long long)b0 * kBlock);
  double acc = 0.0, w_at = 0.0;
  int at = -1;
  for (int j = 0; j < kBlock; ++j) {
    const int i = i0 + j;
    if (i >= a.n_cols) break;
    const double w = kept_weight<DT>(v, i, st, par);
    if (w > 0.0) { at = i; w_at = w; }
    acc += w;
    if (acc > in_block && w > 0.0) break;
  }
  a.idx[(long long)r * a.n_draws + d] = at;
  if (a.prob) a.prob[(long long)r * a.n_draws + d] = (float)(w_at / total);
}

// ---------------------------------------------------------------- host side
struct DrawLayout { int chunk, n_chunks; size_t state, chunk_sum, block_incl, total; };
static DrawLayout draw_layout(long long n_rows, long long n_cols) {
  DrawLayout l;
  // chunks of one tile; of more where a row would have over kMaxChunks of them
  const long long tiles = n_cols > 0 ? (n_cols + kTile - 1) / kTile : 1;
  const long long per = (tiles + kMaxChunks - 1) / kMaxChunks;
  l.chunk = (int)(per * kTile);
  l.n_chunks = n_cols > 0 ? (int)((n_cols + l.chunk - 1) / l.chunk) : 1;
  size_t o = 0;
  auto take = [&o](size_t bytes) { const size_t at = o; o += (bytes + 255) & ~(size_t)255; return at; };
  l.state = take(sizeof(DrawState) * n_rows);
  l.chunk_sum = take(sizeof(double) * n_rows * l.n_chunks);
  l.block_incl = take(sizeof(double) * n_rows * l.n_chunks * (l.chunk / kBlock));
  l.total = o;
  return l;
}
template <int DT> static void launch_draw(const DrawArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(k_draw_select<DT>, dim3(a.n_rows), dim3(1024), 0, s, a);
  hipLaunchKernelGGL(k_draw_sums<DT>, dim3(a.n_chunks, a.n_rows), dim3(256), 0, s, a);
  hipLaunchKernelGGL(k_draw_pick<DT>, dim3((unsigned)(((long long)a.n_draws + 255) / 256), a.n_rows), dim3(256), 0, s, a);
}

}  // namespace psl
using namespace psl;

extern "C" int64_t psl_draw_ws_bytes(int32_t n_rows, int32_t n_cols) {
  if (n_rows < 0 || n_cols < 0 || n_rows > 65535 || n_cols > 0x7ffff000) { set_error("psl_draw_ws_bytes: %d rows of %d", n_rows, n_cols); return PSL_ERR_ARG; }
  return (int64_t)draw_layout(n_rows, n_cols).total;
}

extern "C" int psl_draw_indices(const psl_draw_args* q, void* stream) {
#define PSL_BAD(...) do { set_error(__VA_ARGS__); return PSL_ERR_ARG; } while (0)
  if (!q) PSL_BAD("psl_draw_indices: null argument");
  if (q->dtype < PSL_F32 || q->dtype > PSL_F16) PSL_BAD("psl_draw_indices: unknown dtype %d", q->dtype);
  if (q->n_rows < 0 || q->n_rows > 65535 || q->n_cols < 0 || q->n_cols > 0x7ffff000 || q->n_draws < 0)
    PSL_BAD("psl_draw_indices: %d rows (up to 65535) of %d entries, %d draws", q->n_rows, q->n_cols, q->n_draws);
  if (q->n_rows == 0 || q->n_draws == 0) return PSL_OK;
  if ((!q->scores && q->n_cols) || !q->u || !q->idx || !q->ws) PSL_BAD("psl_draw_indices: missing pointer");
  const int es = q->dtype == PSL_F32 ? 4 : 2;
  const long long big = 1ll << 40;
  if (q->score_stride < 0 || q->mask_stride < 0 || q->u_stride < 0 || q->score_stride > big || q->mask_stride > big || q->u_stride > big)
    PSL_BAD("psl_draw_indices: bad stride");
  if ((uintptr_t)q->scores % es || (uintptr_t)q->u % 4 || (uintptr_t)q->idx % 4 || (uintptr_t)q->prob % 4 || (uintptr_t)q->ws % 256 ||
      (uintptr_t)q->temperature % 4 || (uintptr_t)q->top_k % 4 || (uintptr_t)q->top_p % 4 || (uintptr_t)q->min_p % 4)
    PSL_BAD("psl_draw_indices: misaligned pointer (the workspace needs 256 bytes)");
  if ((!q->temperature && q->temperature_all != q->temperature_all) || (!q->top_p && q->top_p_all != q->top_p_all) ||
      (!q->min_p && q->min_p_all != q->min_p_all))
    PSL_BAD("psl_draw_indices: NaN parameter");
  const DrawLayout l = draw_layout(q->n_rows, q->n_cols);
  if (q->ws_bytes < (int64_t)l.total) PSL_BAD("psl_draw_indices: workspace of %lld bytes, %lld needed", (long long)q->ws_bytes, (long long)l.total);
  DrawArgs a;
  a.n_rows = q->n_rows; a.n_cols = q->n_cols; a.n_draws = q->n_draws;
  a.scores = q->scores; a.stride = q->score_stride; a.mask = q->mask; a.mask_stride = q->mask_stride;
  a.temperature = q->temperature; a.top_k = q->top_k; a.top_p = q->top_p; a.min_p = q->min_p;
  a.t_all = q->temperature_all; a.p_all = q->top_p_all; a.m_all = q->min_p_all; a.k_all = q->top_k_all;
  a.u = q->u; a.u_stride = q->u_stride; a.idx = q->idx; a.prob = q->prob;
  char* w = (char*)q->ws;
  a.state = (DrawState*)(w + l.state); a.chunk_sum = (double*)(w + l.chunk_sum); a.block_incl = (double*)(w + l.block_incl);
  a.n_chunks = l.n_chunks; a.chunk = l.chunk;
  hipStream_t s = (hipStream_t)stream;
  if (q->dtype == PSL_F32) launch_draw<PSL_F32>(a, s);
  else if (q->dtype == PSL_BF16) launch_draw<PSL_BF16>(a, s);
  else launch_draw<PSL_F16>(a, s);
  PSL_LAUNCH_CHECK();
  return PSL_OK;
#undef PSL_BAD
}
