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
  int cuts;                    // whether any row may have a limit (else the launches that find thresholds are left out)
  int n_parts, part_len;       // pieces of a row in the launches before k_draw_sums
  struct DrawState* state;     // [n_rows]
  struct DrawCut* cut;         // [n_rows]
  unsigned* part_max; unsigned* part_min;       // [n_rows][n_parts] keys
  unsigned* tops; int top_lanes, n_tops;       // [n_rows][n_tops] keys: the largest of every top_lanes lanes of a part's workgroup
  int listed_draws;            // whether k_draw_cut may draw from a row's list
  unsigned* bin_cnt; unsigned long long* bin_mass;       // [n_rows][kBins]
  double* bin_excl;            // [n_rows][kBins]: running sums in front of the bins; those behind them replace bin_mass
  unsigned long long* list_a; unsigned long long* list_b; int list_cap;      // [n_rows][list_cap] numbers of candidate entries
  double* chunk_sum;           // [n_rows][n_chunks]
  struct DrawGroup* group;     // [n_rows][n_chunks * chunk / kGroup]
  double* group_incl;          // [n_rows][n_chunks * chunk / kGroup]: a group's last running sum once more, packed
  int n_chunks, chunk;         // entries of a chunk (a multiple of kTile)
  int pick_wgs, place_groups; long long pick_len;       // k_draw_pick: workgroups and draws to a workgroup; groups between places in LDS
};
struct DrawState {
  u64 thr;                     // kept: number(entry) >= thr
  double inv_t, m;             // 1 / temperature, min-p
  float M; int any;            // largest allowed score; whether there is one
  unsigned n_a, n_b;           // fill of the two lists
  int drawn;                   // k_draw_cut has drawn for this row
};

struct DrawCut {
  float M; int any;                // as in DrawState
  double inv_t, p;                 // 1 / temperature, top-p (1: off)
  float scale; unsigned want;      // bins per unit of score; entries of k_bin that top-k keeps
  int k_bin, p_lo, p_hi;           // k_bin = kBins: top-k keeps all; top-p's bin lies in [p_lo, p_hi], or is k_bin
  unsigned n_a;                    // entries of k_bin
  unsigned n_all;                  // entries up to the last bin that a limit can fall into, if they are all drawn from one list (else 0)
  double above_k, total;           // mass of the bins before k_bin; of all
};

// Eight blocks of 16 entries, one 128-byte line: the running sums inside their chunk at the end of each block, and which of
// a block's entries are kept.
struct alignas(128) DrawGroup { double incl[8]; unsigned short kept[8]; };

constexpr int kBlock = 16;     // entries to a stored running sum: one 64-byte line of fp32 scores
constexpr int kGroup = 8 * kBlock;
constexpr int kTile = 4096;    // entries that a workgroup of k_draw_sums takes per step
constexpr int kMaxChunks = 1024;
constexpr int kMaxParts = 256;
constexpr int kBins = 1024;
constexpr double kRange = 48.0;
constexpr int kSorted = 1024;  // numbers that a workgroup sorts, one to a thread

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
  q.inv_t = t > 0.0 ? fmin(1.0 / t, 1e300) : 1.0;       // (finite: no difference times it stays 0)
  return q;
}
// exp(-x) for x >= 0 to about one unit of the last place, in 14 fp64 instructions and one LDS read (the library's takes about
// 35, and the weights of a pass are what it computes): x = (n + f) ln2 / 64 with |f| <= 1/2, 2^(-(n mod 64) / 64) from a table of
// 64, e^-r = 1 - r + r^2/2 - r^3/6 + r^4/24 - r^5/120 for the rest |r| <= ln2 / 128 (the next term is below 4e-17), 2^-(n / 64)
// into the exponent.  Beyond x = 1100 the result is 0; a NaN counts as that.
struct ExpTable { double t[64]; };
__device__ __forceinline__ void exp_table_init(ExpTable& e) { if (threadIdx.x < 64) e.t[threadIdx.x] = exp2(-(double)threadIdx.x / 64.0); }
// a constant that stays in a scalar register (the compiler would write it into two vector registers for every use)
__device__ __forceinline__ double resident(double c) { asm("" : "+s"(c)); return c; }
__device__ __forceinline__ double exp_neg(double x, const ExpTable& e) {
  x = fmin(x, 1100.0);
  const double n = rint(x * resident(92.332482616893656));          // 64 / ln2
  double r = fma(n, resident(-0x1.62e42fefa39efp-7), x);            // ln2 / 64, and what that number leaves of it
  r = fma(n, resident(-0x1.abc9e3b39803fp-62), r);
  const int k = (int)n;
  double p = fma(r, resident(-1.0 / 120.0), resident(1.0 / 24.0));
  p = fma(r, p, resident(-1.0 / 6.0));
  p = fma(r, p, 0.5);
  p = fma(r, p, -1.0);
  p = fma(r, p, 1.0);
  return ldexp(e.t[k & 63] * p, -(k >> 6));
}
// weight of an allowed score; +inf among the scores takes all
__device__ __forceinline__ double weight_of(float s, float M, double inv_t, const ExpTable& e) {
  if (M == __builtin_inff()) return s == M ? 1.0 : 0.0;
  return exp_neg(((double)M - (double)s) * inv_t, e);
}

__device__ __forceinline__ double shfl_up_d(double v, int o) { return __shfl_up(v, o); }

// ---------------------------------------------------------------- largest and smallest allowed score of a row's parts
// A row is read in n_parts pieces of part_len entries, a workgroup to a piece; four entries to a lane and step.
template <int DT> struct Four { float s[4]; unsigned live; };      // live: bit q = entry q is inside the row and not masked
template <int DT> __device__ __forceinline__ Four<DT> load_four(const RowView& v, int i, int end) {
  Four<DT> f;
  f.live = 0;
  if (i + 4 <= end) {
    // rows begin anywhere: the loads are as wide as 16 bytes but aligned to an entry only
    if constexpr (DT == PSL_F32) __builtin_memcpy(f.s, (const float*)v.s + i, 16);
    else {
      unsigned short h[4];
      __builtin_memcpy(h, (const unsigned short*)v.s + i, 8);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if constexpr (DT == PSL_BF16) f.s[q] = __uint_as_float((unsigned)h[q] << 16);
        else { _Float16 x; __builtin_memcpy(&x, &h[q], 2); f.s[q] = (float)x; }
      }
    }
    f.live = 15u;
    if (v.m) {
      unsigned m;
      __builtin_memcpy(&m, v.m + i, 4);
#pragma unroll
      for (int q = 0; q < 4; ++q) if (!((m >> (8 * q)) & 255u)) f.live &= ~(1u << q);
    }
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      f.s[q] = 0.f;
      if (i + q < end) { f.s[q] = load_score<DT>(v.s, i + q); if (!v.m || v.m[i + q]) f.live |= 1u << q; }
    }
  }
  return f;
}
template <int DT> __device__ __forceinline__ unsigned four_key(const Four<DT>& f, int q) { return (f.live >> q) & 1u ? key_of(f.s[q]) : 0u; }

template <int DT> __global__ __launch_bounds__(256) void k_draw_range(DrawArgs a) {
  __shared__ unsigned s_mx[4], s_mn[4];
  const int r = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const RowView v = row_view<DT>(a, r);
  const int i0 = blockIdx.x * a.part_len, i1 = min(i0 + a.part_len, a.n_cols);
  unsigned mx = 0u, mn = 0xffffffffu;
  for (int i = i0 + tid * 4; i < i1; i += 1024) {
    const Four<DT> f = load_four<DT>(v, i, i1);
#pragma unroll
    for (int q = 0; q < 4; ++q) { const unsigned k = four_key(f, q); mx = max(mx, k); mn = min(mn, k ? k : 0xffffffffu); }
  }
  for (int o = 1; o < 64; o <<= 1) {
    if (o == a.top_lanes && a.cuts && (tid & (o - 1)) == 0) a.tops[(long long)r * a.n_tops + blockIdx.x * (256 / o) + tid / o] = mx;
    mx = max(mx, (unsigned)__shfl_xor((int)mx, o)); mn = min(mn, (unsigned)__shfl_xor((int)mn, o));
  }
  if (lane == 0) {
    s_mx[tid >> 6] = mx; s_mn[tid >> 6] = mn;
    if (a.top_lanes == 64 && a.cuts) a.tops[(long long)r * a.n_tops + blockIdx.x * 4 + (tid >> 6)] = mx;
  }
  __syncthreads();
  if (tid == 0) {
    a.part_max[(long long)r * a.n_parts + blockIdx.x] = max(max(s_mx[0], s_mx[1]), max(s_mx[2], s_mx[3]));
    a.part_min[(long long)r * a.n_parts + blockIdx.x] = min(min(s_mn[0], s_mn[1]), min(s_mn[2], s_mn[3]));
  }
  // what the next launches add to
  if (a.cuts && blockIdx.x == 0) {
    for (int j = tid; j < kBins; j += 256) { a.bin_cnt[(long long)r * kBins + j] = 0u; a.bin_mass[(long long)r * kBins + j] = 0ull; }
    if (tid == 0) { a.state[r].n_a = 0u; a.state[r].n_b = 0u; a.state[r].drawn = 0; }
  }
}
// the same of the whole row, to every thread of a workgroup (n_parts <= kMaxParts)
struct Range { unsigned mx, mn; };
__device__ __forceinline__ Range row_range(const DrawArgs& a, int r) {
  __shared__ unsigned s_mx, s_mn;
  if (threadIdx.x < 64) {
    unsigned mx = 0u, mn = 0xffffffffu;
    for (int j = threadIdx.x; j < a.n_parts; j += 64) { mx = max(mx, a.part_max[(long long)r * a.n_parts + j]); mn = min(mn, a.part_min[(long long)r * a.n_parts + j]); }
    for (int o = 32; o > 0; o >>= 1) { mx = max(mx, (unsigned)__shfl_xor((int)mx, o)); mn = min(mn, (unsigned)__shfl_xor((int)mn, o)); }
    if (threadIdx.x == 0) { s_mx = mx; s_mn = mn; }
  }
  __syncthreads();
  return Range{s_mx, s_mn};
}
__device__ __forceinline__ bool has_cut(const RowPar& p) { return p.k > 0 || p.p < 1.0; }

// ---------------------------------------------------------------- bins of equal width in M - s
// kBins of them over the row's range, at most kRange temperatures wide; the last one goes on beyond that.  fp32 decides the
// bin: a difference, a product and a truncation never fall as the score falls, so a bin is an interval of scores, and that is
// all it has to be.  A bin's mass is a sum of integers, weights scaled by 2^(q + the bin's own exponent): it has no order, and its
// rounding is 2^-q of the bin's own weights.
struct Binning { float M, scale; double inv_t, width, oct; int q; bool plain; };      // plain: no entry lies behind its bin
__device__ __forceinline__ Binning make_binning(const Range& g, double inv_t, int n_cols) {
  Binning b;
  b.M = score_of(g.mx); b.inv_t = inv_t;
  double range = ((double)b.M - (double)score_of(g.mn)) * inv_t;
  b.plain = range < kRange;
  if (!b.plain) range = kRange;
  // bins per unit of score, a number whatever the row is (equal scores, denormal ones, infinite ones, no temperature), and the
  // width that this number means, in temperatures
  const double sc = (double)kBins * inv_t / range;
  b.plain = b.plain && sc > 1e-36 && sc < 3e38;
  b.scale = sc > 0.0 ? (float)fmin(fmax(sc, 1e-36), 3e38) : 1.f;
  b.width = inv_t / (double)b.scale;
  b.oct = b.width * 1.4426950408889634;             // binary orders per bin
  b.q = min(62 - (32 - __clz(n_cols)), 51);         // the row's sum below 2^63, an entry's below to_integer's limit
  return b;
}
__device__ __forceinline__ int bin_of(const Binning& b, float s) {
  // (NaN, from inf - inf or 0 * inf, converts to 0: the largest score's bin)
  return (int)min(__float2uint_rz((b.M - s) * b.scale), (unsigned)(kBins - 1));
}
__device__ __forceinline__ int bin_shift(const Binning& b, int bin) { return b.q + (int)fmin((double)bin * b.oct, 1000.0); }

// 0 <= x < 2^52 to the nearest integer: 2^52 + x has it in its low bits
__device__ __forceinline__ u64 to_integer(double x) { return (u64)__double_as_longlong(x + 0x1p52) & 0xfffffffffffffull; }

// An entry's scaled weight is its bin's first weight (a table) times e^-f, f < kRange / kBins = 0.047 behind the bin's begin:
// the terms to the seventh leave 1e-15 of it.  What lies beyond kRange, in the last bin, takes the exponential.
__device__ __forceinline__ double first_weight(const Binning& b, int j) { return ldexp(exp(-(double)j * b.width), bin_shift(b, j)); }
// the coefficients stay in registers (the compiler would write them anew for every entry: they are not inline constants)
struct BinPoly { double c7, c6, c5, c4, c3; };
__device__ __forceinline__ BinPoly make_bin_poly() {
  BinPoly p{-1.0 / 5040.0, 1.0 / 720.0, -1.0 / 120.0, 1.0 / 24.0, -1.0 / 6.0};
  asm("" : "+v"(p.c7), "+v"(p.c6), "+v"(p.c5), "+v"(p.c4), "+v"(p.c3));
  return p;
}
template <bool PLAIN, int DT> __device__ __forceinline__ void add_to_bins(const Four<DT>& f, const Binning& b, const BinPoly& c, bool count, bool weigh, int last,
                                                              unsigned* cnt, u64* mass, const double* first) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float s = f.s[q];
    if (((f.live >> q) & 1u) && s > -__builtin_inff()) {
      const int bin = bin_of(b, s);
      if (bin > last) continue;
      if (count) atomicAdd(&cnt[bin], 1u);
      if (weigh) {
        const double y = fma((double)bin, -b.width, ((double)b.M - (double)s) * b.inv_t);
        double p = fma(y, c.c7, c.c6);
        p = fma(y, p, c.c5);
        p = fma(y, p, c.c4);
        p = fma(y, p, c.c3);
        p = fma(y, p, 0.5);
        p = fma(y, p, -1.0);
        p = fma(y, p, 1.0);
        if (!PLAIN && !(fabs(y) <= 0.06)) {        // far scores, odd rows
          p = b.M == __builtin_inff() ? (s == b.M ? 1.0 : 0.0) : exp(-fmin(fmax(y, 0.0), 1100.0));
        }
        atomicAdd(&mass[bin], to_integer(first[bin] * p));
      }
    }
  }
}

// The last bin that matters to a row with top-k: of n_tops maxima of disjoint parts of the row the k-th largest is no larger
// than the row's k-th score, and top-p weighs what top-k leaves.  What lies behind is neither counted nor weighed.  A workgroup of 512, cnt zero before and after.
constexpr int kTops = 1024;
__device__ __forceinline__ int last_bin(const DrawArgs& a, int r, int k, const Binning& b, unsigned* cnt) {
  __shared__ unsigned s_n[8];
  __shared__ int s_last;
  const int tid = threadIdx.x, lane = tid & 63;
  if (tid == 0) s_last = kBins - 1;
  for (int j = tid; j < a.n_tops; j += 512) {
    const unsigned key = a.tops[(long long)r * a.n_tops + j];
    if (key) atomicAdd(&cnt[bin_of(b, score_of(key))], 1u);
  }
  __syncthreads();
  const unsigned c0 = cnt[2 * tid], c1 = cnt[2 * tid + 1];
  cnt[2 * tid] = 0u; cnt[2 * tid + 1] = 0u;
  unsigned incl = c0 + c1;
  for (int o = 1; o < 64; o <<= 1) { const unsigned x = __shfl_up(incl, o); if (lane >= o) incl += x; }
  if (lane == 63) s_n[tid >> 6] = incl;
  __syncthreads();
  for (int w = 0; w < (tid >> 6); ++w) incl += s_n[w];
  if (incl >= (unsigned)k && incl - c0 - c1 < (unsigned)k) s_last = incl - c1 >= (unsigned)k ? 2 * tid : 2 * tid + 1;
  __syncthreads();
  return s_last;
}

// Bound: instructions (65 per entry made this 25 us for twelve rows of 816 000, now 18), then the LDS atomics: entries are counted
// only where that is used and weighed only where top-p does, and neighbouring lanes use different copies.  64 registers, some
// of them spilled before the loop, let a CU hold all four of its workgroups (68: 20.8 us).
constexpr int kCopies = 2;
template <int DT> __global__ __launch_bounds__(512, 8) void k_draw_hist(DrawArgs a) {
  __shared__ unsigned cnt[kCopies][kBins];
  __shared__ u64 mass[kCopies][kBins];
  __shared__ double first[kBins];
  const int r = blockIdx.y, tid = threadIdx.x;
  const RowPar par = row_par(a, r);
  if (!has_cut(par)) return;
  const bool weigh = par.p < 1.0 && par.k != 1, count = par.k > 0 || a.listed_draws;
  const Range g = row_range(a, r);
  if (!g.mx) return;
  const Binning b = make_binning(g, par.inv_t, a.n_cols);
  for (int j = tid; j < kBins; j += 512) {
#pragma unroll
    for (int q = 0; q < kCopies; ++q) { cnt[q][j] = 0u; mass[q][j] = 0ull; }
  }
  __syncthreads();
  const int last = par.k > 0 && par.k <= a.n_tops ? last_bin(a, r, par.k, b, cnt[0]) : kBins - 1;
  if (weigh) for (int j = tid; j <= last; j += 512) first[j] = first_weight(b, j);
  __syncthreads();
  const RowView v = row_view<DT>(a, r);
  const int i0 = blockIdx.x * a.part_len, i1 = min(i0 + a.part_len, a.n_cols);
  unsigned* const my_cnt = cnt[tid & (kCopies - 1)];
  u64* const my_mass = mass[tid & (kCopies - 1)];
  const BinPoly poly = make_bin_poly();
  if (b.plain) {
#pragma unroll 2
    for (int i = i0 + tid * 4; i < i1; i += 2048) add_to_bins<true>(load_four<DT>(v, i, i1), b, poly, count, weigh, last, my_cnt, my_mass, first);
  } else {
    for (int i = i0 + tid * 4; i < i1; i += 2048) add_to_bins<false>(load_four<DT>(v, i, i1), b, poly, count, weigh, last, my_cnt, my_mass, first);
  }
  __syncthreads();
  for (int j = tid; j <= last; j += 512) {
    unsigned c = 0u; u64 m = 0ull;
#pragma unroll
    for (int q = 0; q < kCopies; ++q) { c += cnt[q][j]; m += mass[q][j]; }
    if (c) atomicAdd(&a.bin_cnt[(long long)r * kBins + j], c);
    if (m) atomicAdd(&a.bin_mass[(long long)r * kBins + j], m);
  }
}

// smallest / largest thread of the workgroup for which a condition holds: a ballot per wavefront, then one LDS atomic each
// (an atomic per thread to one address is run lane by lane)
__device__ __forceinline__ void note_first(int* at, bool cond) {
  const u64 m = __ballot(cond);
  if (m && (threadIdx.x & 63) == 0) atomicMin(at, (int)(threadIdx.x & ~63u) + __ffsll((long long)m) - 1);
}
__device__ __forceinline__ void note_last(int* at, bool cond) {
  const u64 m = __ballot(cond);
  if (m && (threadIdx.x & 63) == 0) atomicMax(at, (int)(threadIdx.x & ~63u) + 63 - __clzll((long long)m));
}
// Which bins the two limits fall into, by a workgroup with a thread to a bin, the largest scores first: c entries, mass m.
// cum / excl receive the running sums behind and in front of the bins (behind an empty one: -1).
struct BinsShared { unsigned cnt[kBins / 64]; double mass[kBins / 64], above_k, most; int k, lo, hi, last; unsigned want, na; };
__device__ __forceinline__ void find_bins(const DrawArgs& a, const RowPar& par, const Range& g, const Binning& b, unsigned c, double m,
                                          double* cum, double* excl_out, DrawCut* o, BinsShared& sh) {
  const int j = threadIdx.x, lane = j & 63, wave = j >> 6;
  if (j == 0) {
    sh.k = kBins; sh.lo = kBins; sh.hi = kBins; sh.last = -1; sh.want = 0u; sh.na = 0u;
    o->M = b.M; o->any = g.mx ? 1 : 0; o->inv_t = par.inv_t; o->p = par.k == 1 ? 1.0 : par.p; o->scale = b.scale;
  }
  if (!g.mx || !has_cut(par)) {
    if (j == 0) { o->k_bin = kBins; o->p_hi = -1; o->n_a = 0u; o->n_all = 0u; }
    return;
  }
  unsigned n_incl = c; double incl = m;
  for (int i = 1; i < 64; i <<= 1) {
    const unsigned cu = __shfl_up(n_incl, i); const double mu = shfl_up_d(incl, i);
    if (lane >= i) { n_incl += cu; incl += mu; }
  }
  if (lane == 63) { sh.cnt[wave] = n_incl; sh.mass[wave] = incl; }
  __syncthreads();
  unsigned n_valid = 0u, n_before = 0u; double total = 0.0, before = 0.0;
  for (int w = 0; w < kBins / 64; ++w) {
    if (w == wave) { n_before = n_valid; before = total; }
    n_valid += sh.cnt[w]; total += sh.mass[w];
  }
  // running sums in front of and behind this bin; only bins that hold something are ever chosen
  const double up = __shfl_up(incl, 1), excl = lane ? before + up : before;
  n_incl += n_before; incl += before;
  cum[j] = m > 0.0 ? incl : -1.0;
  excl_out[j] = excl;
  // As many as there are, or more: the limit keeps all of them.  It is looked for all the same where they may be only what was
  // counted, and where they are few enough for one list.
  const unsigned k = (unsigned)par.k > n_valid && n_valid <= (unsigned)kSorted ? n_valid : (unsigned)par.k;
  const bool cut_k = par.k > 0 && k <= n_valid, cut_p = par.p < 1.0 && par.k != 1;
  if (cut_k && n_incl >= k && n_incl - c < k) {
    sh.k = j; sh.want = k - (n_incl - c); sh.na = c; sh.most = incl; sh.above_k = excl;
  }
  __syncthreads();
  const int k_bin = sh.k;
  const double above_k = cut_k ? sh.above_k : total, most = cut_k ? sh.most : total;
  if (cut_p) {
    // top-k leaves a mass between above_k and `most`: the bins before k_bin where its share can fall (none, by rounding: the last)
    const bool held = m > 0.0 && j < k_bin;
    note_last(&sh.last, held);
    note_first(&sh.lo, held && incl >= par.p * above_k);
    note_first(&sh.hi, held && incl >= par.p * most);
  }
  __syncthreads();
  const int p_lo = cut_p ? min(sh.lo, sh.last) : 0, p_hi = cut_p ? min(sh.hi, sh.last) : -1;
  // the last bin that a limit can fall into, and whether all entries up to it are few
  const int end = cut_k ? k_bin : p_hi;
  if (j == max(end, 0)) o->n_all = a.listed_draws && end >= 0 && n_incl <= (unsigned)kSorted ? n_incl : 0u;
  if (j == 64) {
    o->want = sh.want; o->k_bin = k_bin; o->p_lo = p_lo; o->p_hi = p_hi; o->n_a = sh.na; o->above_k = above_k; o->total = total;
  }
}
// One workgroup to a row.  (In every workgroup of k_draw_gather instead, this cost each of them 8 us.)
__global__ __launch_bounds__(kBins) void k_draw_bins(DrawArgs a) {
  __shared__ BinsShared sh;
  const int r = blockIdx.x, j = threadIdx.x;
  const RowPar par = row_par(a, r);
  const Range g = row_range(a, r);
  const Binning b = make_binning(g, par.inv_t, a.n_cols);
  const long long at = (long long)r * kBins + j;
  const unsigned c = a.bin_cnt[at];
  const double m = ldexp((double)a.bin_mass[at], -bin_shift(b, j));
  find_bins(a, par, g, b, c, m, (double*)(a.bin_mass + (long long)r * kBins), a.bin_excl + (long long)r * kBins, a.cut + r, sh);
}

// Entries of those bins, as their 64-bit numbers, in any order: top-k's bin into one list, top-p's into the other, or all that
// a row can keep into the first.  A
// workgroup collects in LDS and asks once for its places in the row's list (a global atomic for every wavefront that found
// something made this 112 us for twelve rows of 816 000); what does not fit there goes to the list by itself.
constexpr int kListBuf = 1024;
struct ListBuf { u64 e[kListBuf]; unsigned n, at; };
__device__ __forceinline__ void list_add(ListBuf& b, u64 x, u64* dst, unsigned* fill, unsigned cap) {
  const unsigned j = atomicAdd(&b.n, 1u);
  if (j < kListBuf) b.e[j] = x;
  else { const unsigned at = atomicAdd(fill, 1u); if (at < cap) dst[at] = x; }
}
template <int DT> __global__ __launch_bounds__(512) void k_draw_gather(DrawArgs a) {
  __shared__ ListBuf buf_a, buf_b;
  const int r = blockIdx.y, tid = threadIdx.x;
  const DrawCut& c = a.cut[r];
  const bool all = c.n_all > 0u, do_a = all || (c.k_bin < kBins && c.n_a <= (unsigned)a.list_cap), do_b = !all && c.p_hi >= 0;
  if (!do_a && !do_b) return;
  Binning b;
  b.M = c.M; b.scale = c.scale;
  // (no such bin: an empty interval)
  const int k_bin = c.k_bin < kBins ? c.k_bin : c.p_hi;
  const int a0 = all ? 0 : k_bin, a1 = do_a ? k_bin : -1, p0 = c.p_lo, p1 = do_b ? c.p_hi : -1;
  if (tid == 0) { buf_a.n = 0u; buf_b.n = 0u; }
  __syncthreads();
  const RowView v = row_view<DT>(a, r);
  const int i0 = blockIdx.x * a.part_len, i1 = min(i0 + a.part_len, a.n_cols);
  u64* la = a.list_a + (long long)r * a.list_cap;
  u64* lb = a.list_b + (long long)r * a.list_cap;
  const unsigned cap = (unsigned)a.list_cap;
#pragma unroll 2
  for (int i = i0 + tid * 4; i < i1; i += 2048) {
    const Four<DT> f = load_four<DT>(v, i, i1);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float x = f.s[q];
      if (((f.live >> q) & 1u) && x > -__builtin_inff()) {
        const int bin = bin_of(b, x);
        if (bin >= a0 && bin <= a1) list_add(buf_a, number_of(key_of(x), i + q), la, &a.state[r].n_a, cap);
        if (bin >= p0 && bin <= p1) list_add(buf_b, number_of(key_of(x), i + q), lb, &a.state[r].n_b, cap);
      }
    }
  }
  __syncthreads();
  const unsigned na = min(buf_a.n, (unsigned)kListBuf), nb = min(buf_b.n, (unsigned)kListBuf);
  if (tid == 0 && na) buf_a.at = atomicAdd(&a.state[r].n_a, na);
  if (tid == 64 && nb) buf_b.at = atomicAdd(&a.state[r].n_b, nb);
  __syncthreads();
  for (unsigned j = tid; j < na; j += 512) if (buf_a.at + j < cap) la[buf_a.at + j] = buf_a.e[j];
  for (unsigned j = tid; j < nb; j += 512) if (buf_b.at + j < cap) lb[buf_b.at + j] = buf_b.e[j];
}

// ---------------------------------------------------------------- the threshold among those entries, by radix selection
// 256 digits of (count, mass): masses are summed as integers, 32 bits before and 32 behind the point at 2^-32, so their sum has no order
struct RadixBins { unsigned cnt[256]; u64 hi[256], lo[256]; };
struct RadixPick { int bin; unsigned above, count; double mass_above, mass; };
struct RadixShared { RadixBins bins; RadixPick pick; u64 mx[16], mn[16]; u64 hi, lo; ExpTable exp; };

__device__ __forceinline__ double fixed_d(u64 hi, u64 lo) { return (double)hi * 0x1p-32 + (double)lo * 0x1p-64; }
struct Fixed { u64 hi, lo; };
__device__ __forceinline__ Fixed to_fixed(double w) {
  const double x = w * 0x1p32;
  const u64 h = (u64)x;
  return Fixed{h, (u64)((x - (double)h) * 0x1p32)};
}

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

// The numbers that src(i) gives for i < n (0: not among them), up to four of them to a thread in registers.
constexpr int kHeld = 4;
template <class Src> struct Numbers {
  const Src& src; int n; u64 x[kHeld];
  __device__ __forceinline__ Numbers(const Src& src_, int n_) : src(src_), n(n_) {
#pragma unroll
    for (int j = 0; j < kHeld; ++j) { const int i = threadIdx.x + 1024 * j; x[j] = n <= kHeld * 1024 && i < n ? src(i) : 0ull; }
  }
  template <class F> __device__ __forceinline__ void each(const F& f) const {
    if (n <= kHeld * 1024) {
#pragma unroll
      for (int j = 0; j < kHeld; ++j) if (x[j]) f(x[j]);
    } else {
      for (int i = threadIdx.x; i < n; i += 1024) { const u64 y = src(i); if (y) f(y); }
    }
  }
};
__device__ __forceinline__ void block_bounds(u64& mx, u64& mn, RadixShared& sh) {
  for (int o = 32; o > 0; o >>= 1) {
    const u64 x = __shfl_xor(mx, o), y = __shfl_xor(mn, o);
    mx = x > mx ? x : mx; mn = y < mn ? y : mn;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) { sh.mx[threadIdx.x >> 6] = mx; sh.mn[threadIdx.x >> 6] = mn; }
  __syncthreads();
  for (int j = 0; j < 16; ++j) { mx = sh.mx[j] > mx ? sh.mx[j] : mx; mn = sh.mn[j] < mn ? sh.mn[j] : mn; }
}

// Digits of up to eight bits, from the highest in which the numbers differ (none across bit 32, where the score ends); a
// level counts the numbers whose higher digits are the ones found so far.  Ends as soon as the digit found is taken whole.
// By count: the smallest of the first `want`.  By mass: the smallest of the shortest prefix that weighs want_mass.
template <class Src> __device__ u64 radix_select(const Numbers<Src>& num, bool by_mass, unsigned want, double want_mass, float M, double inv_t,
                                                 RadixShared& sh) {
  const int tid = threadIdx.x;
  u64 mx = 0ull, mn = ~0ull;
  num.each([&](u64 x) { mx = x > mx ? x : mx; mn = x < mn ? x : mn; });
  block_bounds(mx, mn, sh);
  if (mx <= mn) return mx == mn ? mx : 0ull;
  int hi = 64 - __clzll((long long)(mx ^ mn));          // bits from here on are equal
  u64 prefix = hi == 64 ? 0ull : mx >> hi;
  bool mass_level = by_mass;
  int lo = hi;
  while (hi > 0) {
    lo = hi > 32 ? (hi - 8 > 32 ? hi - 8 : 32) : (hi - 8 > 0 ? hi - 8 : 0);
    if (mass_level && hi <= 32) {
      // one score is left: as many of its entries as the mass still wants, at least one (all of them: the last)
      const double k = ceil(want_mass / weight_of(score_of((unsigned)(mx >> 32)), M, inv_t, sh.exp));
      want = k < 1.0 ? 1u : k < 4294967295.0 ? (unsigned)k : 0xffffffffu;
      mass_level = false;
    }
    __syncthreads();
    for (int j = tid; j < 256; j += 1024) { sh.bins.cnt[j] = 0u; sh.bins.hi[j] = 0ull; sh.bins.lo[j] = 0ull; }
    __syncthreads();
    num.each([&](u64 x) {
      if (hi == 64 || (x >> hi) == prefix) {
        const int d = (int)((x >> lo) & ((1u << (hi - lo)) - 1u));
        atomicAdd(&sh.bins.cnt[d], 1u);
        if (mass_level) {
          const Fixed f = to_fixed(weight_of(score_of((unsigned)(x >> 32)), M, inv_t, sh.exp));
          atomicAdd(&sh.bins.hi[d], f.hi); atomicAdd(&sh.bins.lo[d], f.lo);
        }
      }
    });
    __syncthreads();
    if (tid < 64) { const RadixPick p = radix_pick(sh.bins, mass_level, want, want_mass); if (tid == 0) sh.pick = p; }
    __syncthreads();
    const RadixPick p = sh.pick;
    prefix = (prefix << (hi - lo)) | (unsigned)p.bin;
    hi = lo;
    if (mass_level) {
      want_mass -= p.mass_above;
      if (p.count == 1) break;
      if (lo == 32) mx = prefix << 32;        // the score that is left
    } else {
      want -= p.above;
      if (want >= p.count) break;
    }
  }
  if (lo == 0) return prefix;
  // The digit is taken whole.  Its smallest number, not its lower end: below that end of src's scores others may begin.
  mx = 0ull; mn = ~0ull;
  num.each([&](u64 x) { if ((x >> lo) == prefix) mn = x < mn ? x : mn; });
  block_bounds(mx, mn, sh);
  return mn;
}

// A wavefront's values at the lane whose number differs in bit J: by moves between lanes of a row of 16, by swaps of rows and
// halves beyond (a shuffle goes through the LDS unit and takes several times as long; the sorts below are chains of these).
template <int J> __device__ __forceinline__ unsigned xor_lane(unsigned x) {
  if constexpr (J == 1) return (unsigned)__builtin_amdgcn_mov_dpp((int)x, 0xb1, 0xf, 0xf, true);           // quad_perm 1 0 3 2
  else if constexpr (J == 2) return (unsigned)__builtin_amdgcn_mov_dpp((int)x, 0x4e, 0xf, 0xf, true);      // quad_perm 2 3 0 1
  else if constexpr (J == 4) {
    const int y = __builtin_amdgcn_mov_dpp((int)x, 0x1b, 0xf, 0xf, true);                                   // quad_perm 3 2 1 0: lane ^ 3
    return (unsigned)__builtin_amdgcn_mov_dpp(y, 0x141, 0xf, 0xf, true);                                    // row_half_mirror: lane ^ 7
  } else if constexpr (J == 8) return (unsigned)__builtin_amdgcn_mov_dpp((int)x, 0x128, 0xf, 0xf, true);   // row_ror 8
  else if constexpr (J == 16) {
    const auto p = __builtin_amdgcn_permlane16_swap(x, x, false, false);                                    // rows 0 0 2 2 and 1 1 3 3
    return threadIdx.x & 16 ? p[0] : p[1];
  } else {
    const auto p = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return threadIdx.x & 32 ? p[0] : p[1];
  }
}
template <int J> __device__ __forceinline__ u64 sort_step(u64 x, int k) {
  const u64 y = (u64)xor_lane<J>((unsigned)(x >> 32)) << 32 | xor_lane<J>((unsigned)x);
  const bool larger = ((threadIdx.x & J) == 0) == ((threadIdx.x & k) == 0);
  return (x > y) == larger ? x : y;
}
// Up to 1 024 numbers, one to a thread, in descending order (zeros behind them), by a bitonic network: exchanges between
// wavefronts through LDS.
__device__ __forceinline__ u64 block_sort(u64 x, int n, u64* lds) {
  const int tid = threadIdx.x;
  for (int k = 2; k < 2 * n && k <= kSorted; k <<= 1) {
    for (int j = k >> 1; j >= 64; j >>= 1) {
      __syncthreads();
      lds[tid] = x;
      __syncthreads();
      const u64 y = lds[tid ^ j];
      const bool larger = ((tid & j) == 0) == ((tid & k) == 0);
      x = (x > y) == larger ? x : y;
    }
    if (k >= 64) x = sort_step<32>(x, k);
    if (k >= 32) x = sort_step<16>(x, k);
    if (k >= 16) x = sort_step<8>(x, k);
    if (k >= 8) x = sort_step<4>(x, k);
    if (k >= 4) x = sort_step<2>(x, k);
    x = sort_step<1>(x, k);
  }
  return x;
}
// sums of the sorted weights up to each thread's, in that order
__device__ __forceinline__ double block_running(double w, double* lds16) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int o = 1; o < 64; o <<= 1) { const double t = shfl_up_d(w, o); if (lane >= o) w += t; }
  __syncthreads();
  if (lane == 63) lds16[wave] = w;
  __syncthreads();
  double before = 0.0;
  for (int j = 0; j < wave; ++j) before += lds16[j];
  return before + w;
}

// The threshold of a row with a limit, by a workgroup of 1 024: from the lists (of up to `cap` numbers) and the bins' running sums.
struct CutShared { RadixShared sh; u64 sort[kSorted], thr; double wave[16], kept; int bin, at, end; };
template <int DT> __device__ __forceinline__ u64 find_threshold(const RowView& v, int n_cols, const DrawCut& c, const u64* la, const u64* lb, unsigned n_b,
                                                                unsigned cap, const double* cum, const double* excl, CutShared& S) {
  const int tid = threadIdx.x;
  const float M = c.M;
  const double inv_t = c.inv_t;
  const bool cut_k = c.k_bin < kBins, cut_p = c.p < 1.0;
  u64 thr = 1ull << 32;                             // every allowed entry
  const bool listed_a = c.n_a <= cap, listed_b = n_b <= cap;
  // a list that its entries do not fit into: the row itself, entry by entry
  Binning b;
  b.M = M; b.scale = c.scale;
  auto from_row = [&](int i, int bin) -> u64 {
    const unsigned k = entry_key<DT>(v, i);
    return k && bin_of(b, score_of(k)) == bin ? number_of(k, i) : 0ull;
  };
  auto src_a = [&](int i) -> u64 { return listed_a ? la[i] : from_row(i, c.k_bin); };
  const int len_a = listed_a ? (int)c.n_a : n_cols;
  double kept = 0.0;                              // mass of what top-k keeps of its bin
  bool p_in_a = false;
  if (cut_k && len_a <= kSorted) {
    const u64 x = block_sort(tid < len_a ? src_a(tid) : 0ull, len_a, S.sort);
    if (tid == 0) S.at = (int)c.want - 1;
    if (tid == (int)c.want - 1) S.thr = x;
    double incl = 0.0;
    if (cut_p) {
      incl = block_running(x ? weight_of(score_of((unsigned)(x >> 32)), M, inv_t, S.sh.exp) : 0.0, S.wave);
      if (tid == (int)c.want - 1) S.kept = incl;
    }
    __syncthreads();
    if (cut_p) {
      kept = S.kept;
      const double target = c.p * (c.above_k + kept);
      p_in_a = target > c.above_k;
      if (p_in_a) {
        note_first(&S.at, incl >= target - c.above_k);
        __syncthreads();
        if (tid == S.at) S.thr = x;
        __syncthreads();
      }
    }
    thr = S.thr;
  } else if (cut_k) {
    const Numbers<decltype(src_a)> num(src_a, len_a);
    const u64 thr_k = radix_select(num, false, c.want, 0.0, M, inv_t, S.sh);
    thr = thr_k;
    if (cut_p) {
      __syncthreads();
      if (tid == 0) { S.sh.hi = 0ull; S.sh.lo = 0ull; }
      __syncthreads();
      u64 hi = 0ull, lo = 0ull;
      num.each([&](u64 x) { if (x >= thr_k) { const Fixed f = to_fixed(weight_of(score_of((unsigned)(x >> 32)), M, inv_t, S.sh.exp)); hi += f.hi; lo += f.lo; } });
      for (int o = 32; o > 0; o >>= 1) { hi += __shfl_xor(hi, o); lo += __shfl_xor(lo, o); }
      if ((tid & 63) == 0) { atomicAdd(&S.sh.hi, hi); atomicAdd(&S.sh.lo, lo); }
      __syncthreads();
      kept = fixed_d(S.sh.hi, S.sh.lo);
      const double target = c.p * (c.above_k + kept);
      p_in_a = target > c.above_k;
      if (p_in_a) {
        auto src = [&](int i) -> u64 { const u64 x = src_a(i); return x >= thr_k ? x : 0ull; };
        thr = radix_select(Numbers<decltype(src)>(src, len_a), true, 0u, target - c.above_k, M, inv_t, S.sh);
      }
    }
  }
  if (cut_p && !p_in_a && c.p_hi >= 0) {
    const double target = c.p * (cut_k ? c.above_k + kept : c.total);
    // first bin of [p_lo, p_hi] whose running sum reaches the target (empty ones hold -1; p_hi is not empty)
    if (tid == 0) S.bin = c.p_hi;
    __syncthreads();
    for (int j = c.p_lo + tid; j < c.p_hi; j += 1024) if (cum[j] >= target) atomicMin(&S.bin, j);
    __syncthreads();
    const int bin = S.bin;
    auto src = [&](int i) -> u64 {
      if (!listed_b) return from_row(i, bin);
      const u64 x = lb[i];
      return bin_of(b, score_of((unsigned)(x >> 32))) == bin ? x : 0ull;
    };
    const double before = excl[bin];
    const int len_b = listed_b ? (int)n_b : n_cols;
    u64 t;
    if (len_b <= kSorted) {
      const u64 x = block_sort(tid < len_b ? src(tid) : 0ull, len_b, S.sort);
      const double incl = block_running(x ? weight_of(score_of((unsigned)(x >> 32)), M, inv_t, S.sh.exp) : 0.0, S.wave);
      // (none reaches it, by rounding: the last one)
      if (tid == 0) { S.at = kSorted; S.end = 0; }
      __syncthreads();
      note_first(&S.at, x && incl >= target - before);
      note_last(&S.end, x != 0ull);
      __syncthreads();
      if (tid == min(S.at, S.end)) S.thr = x;
      __syncthreads();
      t = S.thr;
    } else t = radix_select(Numbers<decltype(src)>(src, len_b), true, 0u, target - before, M, inv_t, S.sh);
    if (t > thr) thr = t;                         // (an empty source gives 0)
  }
  return thr;
}
// The draws of a row whose n entries up to the last bin of its limits are all in one list: sorted by score they give the
// threshold, sorted by index the running sums.  (64 x 131 072 bf16, a draw of each row: this makes k_draw_cut 3 us longer and takes
// 14 us out of k_draw_sums and k_draw_pick, which have nothing left to do for the row.)
__device__ __forceinline__ void draw_from_list(const DrawArgs& a, int r, const u64* list, const DrawCut& c, const RowPar& par, CutShared& S, double* run) {
  const int tid = threadIdx.x, n = (int)c.n_all;
  const bool cut_k = c.k_bin < kBins, cut_p = c.p < 1.0;
  u64 x = block_sort(tid < n ? list[tid] : 0ull, n, S.sort);
  const double w = x ? weight_of(score_of((unsigned)(x >> 32)), c.M, c.inv_t, S.sh.exp) : 0.0;
  int end = cut_k ? min(par.k, n) : n;
  if (cut_p) {
    const double incl = block_running(w, S.wave);
    if (tid == end - 1) { S.kept = incl; S.at = end - 1; }
    __syncthreads();
    note_first(&S.at, x && incl >= c.p * (cut_k ? S.kept : c.total));
    __syncthreads();
    end = S.at + 1;
  }
  x = tid < end && w >= fmax(par.m, 0x1p-1074) ? x << 32 | x >> 32 : 0ull;
  x = block_sort(x, end, S.sort);
  const double incl = block_running(x ? weight_of(score_of((unsigned)x), c.M, c.inv_t, S.sh.exp) : 0.0, S.wave);
  if (tid == 0) S.at = kSorted;
  __syncthreads();                                  // (and the sort's last exchange is over)
  run[tid] = incl;
  S.sort[tid] = x;
  note_first(&S.at, !x);
  __syncthreads();
  const int last = S.at - 1;
  const double total = run[kSorted - 1];
  const long long out0 = (long long)r * a.n_draws;
  for (int d = tid; d < a.n_draws; d += 1024) {
    double u = (double)a.u[(long long)r * a.u_stride + d];
    u = u > 0.0 ? (u < 1.0 ? u : 1.0 - 0x1p-24) : 0.0;
    const double target = u * total;
    int lo = 0, hi = last;
    while (lo < hi) { const int mid = (lo + hi) >> 1; if (run[mid] > target) hi = mid; else lo = mid + 1; }
    const u64 e = S.sort[lo];
    a.idx[out0 + d] = (int)~(unsigned)(e >> 32);
    if (a.prob) a.prob[out0 + d] = (float)(weight_of(score_of((unsigned)e), c.M, c.inv_t, S.sh.exp) / total);
  }
}
template <int DT> __global__ __launch_bounds__(1024) void k_draw_cut(DrawArgs a) {
  __shared__ CutShared S;
  __shared__ double run[kSorted];
  exp_table_init(S.sh.exp);
  const int r = blockIdx.x;
  const DrawCut& c = a.cut[r];
  __syncthreads();
  if (c.n_all) {
    if (threadIdx.x == 0) a.state[r].drawn = 1;
    draw_from_list(a, r, a.list_a + (long long)r * a.list_cap, c, row_par(a, r), S, run);
    return;
  }
  u64 thr = 1ull << 32;
  if (c.any && (c.k_bin < kBins || c.p < 1.0))
    thr = find_threshold<DT>(row_view<DT>(a, r), a.n_cols, c, a.list_a + (long long)r * a.list_cap, a.list_b + (long long)r * a.list_cap, a.state[r].n_b,
                             (unsigned)a.list_cap, (const double*)(a.bin_mass + (long long)r * kBins), a.bin_excl + (long long)r * kBins, S);
  if (threadIdx.x == 0) {
    DrawState* o = a.state + r;
    o->thr = thr; o->M = c.M; o->any = c.any; o->inv_t = c.inv_t; o->m = row_par(a, r).m;
  }
}

// what k_draw_sums and k_draw_pick need of a row
__device__ __forceinline__ DrawState row_state(const DrawArgs& a, int r) {
  if (a.cuts) return a.state[r];
  const Range g = row_range(a, r);
  const RowPar par = row_par(a, r);
  return DrawState{1ull << 32, par.inv_t, par.m, score_of(g.mx), g.mx ? 1 : 0, 0u, 0u, 0};
}

// ---------------------------------------------------------------- running sums of the kept weights
// An entry is kept iff its number is at least the threshold, which in scores is: above thr_s, or thr_s itself at an index up to
// thr_i.  (No limit: every score above -inf.)
struct Kept { float thr_s; int thr_i; };
__device__ __forceinline__ Kept kept_from(u64 thr) {
  const unsigned key = (unsigned)(thr >> 32);
  return key <= 1u ? Kept{-__builtin_inff(), -1} : Kept{score_of(key), (int)~(unsigned)thr};
}
__device__ __forceinline__ bool is_kept(float s, int i, const Kept& k) { return s > k.thr_s || (s == k.thr_s && i <= k.thr_i); }
// Which of four entries from index e on are kept, and the sum of their weights.  The four weights are computed side by side,
// needed or not: one behind the other's branch they were a chain (7 x 50 021 entries: 7.4 us, with branches 8.4).
template <int DT> __device__ __forceinline__ unsigned kept_of_four(const Four<DT>& f, int e, const Kept& k, float M, double inv_t, double least, const ExpTable& t, double& w) {
  unsigned bits = 0u;
  w = 0.0;
#pragma unroll
  for (int q = 0; q < 4; ++q) bits |= is_kept(f.s[q], e + q, k) ? 1u << q : 0u;
  bits &= f.live;
  if (bits) {
    double x[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) x[q] = exp_neg(((double)M - (double)f.s[q]) * inv_t, t);
    if (M == __builtin_inff()) {                      // (as weight_of)
#pragma unroll
      for (int q = 0; q < 4; ++q) x[q] = f.s[q] == M ? 1.0 : 0.0;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (!(x[q] >= least)) bits &= ~(1u << q);
      w += (bits >> q) & 1u ? x[q] : 0.0;
    }
  }
  return bits;
}

// One workgroup to a chunk: four entries to a lane, four lanes to a block of 16.  Leaves the running sums at the end of each
// block and which of its entries are kept: a draw then reads neither mask nor threshold.
template <int DT> __global__ __launch_bounds__(256) void k_draw_sums(DrawArgs a) {
  __shared__ double blk[kTile / kBlock];
  __shared__ double wsum[4];
  __shared__ ExpTable s_exp;
  const int r = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  if (a.listed_draws && a.state[r].drawn) return;
  exp_table_init(s_exp);
  const RowView v = row_view<DT>(a, r);
  const DrawState st = row_state(a, r);
  const Kept kp = kept_from(st.thr);
  const double least = fmax(st.m, 0x1p-1074);       // (what weighs nothing is never drawn)
  __syncthreads();
  double carry = 0.0;
  const long long out0 = ((long long)r * a.n_chunks + blockIdx.x) * (a.chunk / kGroup);
  for (int t0 = 0; t0 < a.chunk; t0 += kTile) {
    const long long base = (long long)blockIdx.x * a.chunk + t0;
    if (base >= a.n_cols) break;                    // (uniform; nothing reads the sums behind the row's end)
    Four<DT> f[kTile / 1024];
#pragma unroll
    for (int j = 0; j < kTile / 1024; ++j) {        // all of a thread's loads before any of its weights
      const long long e = base + j * 1024 + tid * 4;
      if (e < a.n_cols) f[j] = load_four<DT>(v, (int)e, a.n_cols);
      else f[j].live = 0u;
    }
#pragma unroll
    for (int j = 0; j < kTile / 1024; ++j) {
      const int e = (int)(base + j * 1024 + tid * 4);
      double w;
      unsigned bits = kept_of_four(f[j], e, kp, st.M, st.inv_t, least, s_exp, w);
      bits <<= 4 * (lane & 3);
      w += __shfl_xor(w, 1);
      w += __shfl_xor(w, 2);
      bits |= (unsigned)__shfl_xor((int)bits, 1);
      bits |= (unsigned)__shfl_xor((int)bits, 2);
      if ((tid & 3) == 0) {
        const int q = j * 64 + (tid >> 2);
        blk[q] = w;
        a.group[out0 + t0 / kGroup + (q >> 3)].kept[q & 7] = (unsigned short)bits;
      }
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
    a.group[out0 + t0 / kGroup + (tid >> 3)].incl[tid & 7] = s;
    if ((tid & 7) == 7) a.group_incl[out0 + t0 / kGroup + (tid >> 3)] = s;
    carry = ((((carry + wsum[0]) + wsum[1]) + wsum[2]) + wsum[3]);
    __syncthreads();
  }
  if (tid == 0) a.chunk_sum[(long long)r * a.n_chunks + blockIdx.x] = carry;
}

// Records of 16 N bytes, one to a lane, at p.  A load reads whole records, the four lanes of a quad to one, so that a wavefront
// asks for 16 of them at a time and not for a piece of each of 64; an exchange inside the quad then hands every lane the
// pieces of its own.  (1.5 M draws from twelve rows of 816 000: 43 us, with every lane loading its own records 51.  Whole quads
// must be there.)
template <int CTRL> __device__ __forceinline__ unsigned quad_move(unsigned x) { return (unsigned)__builtin_amdgcn_mov_dpp((int)x, CTRL, 0xf, 0xf, true); }
template <int CTRL> __device__ __forceinline__ const char* quad_move(const char* p) {
  const u64 b = (u64)(uintptr_t)p;
  return (const char*)(uintptr_t)((u64)quad_move<CTRL>((unsigned)(b >> 32)) << 32 | quad_move<CTRL>((unsigned)b));
}
template <int N> __device__ __forceinline__ void swap_pieces(unsigned (&a)[N], unsigned (&b)[N], bool upper, bool by_two) {
#pragma unroll
  for (int w = 0; w < N; ++w) {
    const unsigned x = a[w], y = b[w];
    const unsigned ys = by_two ? quad_move<0x4e>(y) : quad_move<0xb1>(y), xs = by_two ? quad_move<0x4e>(x) : quad_move<0xb1>(x);
    a[w] = upper ? ys : x;
    b[w] = upper ? y : xs;
  }
}
template <int N> __device__ __forceinline__ void load_records(const char* p, unsigned (&x)[4][N]) {
  const int q = threadIdx.x & 3;
  __builtin_memcpy(x[0], quad_move<0x00>(p) + 4 * N * q, 4 * N);
  __builtin_memcpy(x[1], quad_move<0x55>(p) + 4 * N * q, 4 * N);
  __builtin_memcpy(x[2], quad_move<0xaa>(p) + 4 * N * q, 4 * N);
  __builtin_memcpy(x[3], quad_move<0xff>(p) + 4 * N * q, 4 * N);
  swap_pieces<N>(x[0], x[1], q & 1, false);
  swap_pieces<N>(x[2], x[3], q & 1, false);
  swap_pieces<N>(x[0], x[2], q & 2, true);
  swap_pieces<N>(x[1], x[3], q & 2, true);
}

// ---------------------------------------------------------------- the draws
// A workgroup holds its row's running sums in LDS, at the end of every group if they fit, so that a draw searches there and
// then reads two lines: its group's, and the scores of one block.  Bound: instructions (700 a wavefront of draws, 28 us of
// issue for 1.5 M draws from twelve rows of 816 000, which take 43) and these scattered lines (a search in global memory made
// twelve of them, 82 us).  The workgroups of a row run on one XCD (consecutive ones are dealt out to the eight in turn), whose
// L2 then holds most of the row.
constexpr int kPlaces = 6656, kPickThreads = 1024;      // 52 KB: groups of 850 000 entries
template <int DT> __global__ __launch_bounds__(kPickThreads, 8) void k_draw_pick(DrawArgs a) {
  __shared__ double place[kPlaces];        // running sums inside a chunk, as group_incl
  __shared__ double chunk_incl[kMaxChunks];
  __shared__ double wsum[kPickThreads / 64];
  __shared__ ExpTable s_exp;
  const int tid = threadIdx.x, lane = tid & 63;
  const unsigned total_wg = (unsigned)a.n_rows * (unsigned)a.pick_wgs, per_xcd = (total_wg + 7) / 8;
  const unsigned work = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if (work >= total_wg) return;
  const int r = (int)(work / (unsigned)a.pick_wgs);
  const long long d0 = (long long)(work - (unsigned)r * (unsigned)a.pick_wgs) * a.pick_len;
  const long long d1 = d0 + a.pick_len < a.n_draws ? d0 + a.pick_len : a.n_draws;
  const long long out0 = (long long)r * a.n_draws;
  if (a.listed_draws && a.state[r].drawn) return;
  exp_table_init(s_exp);
  const DrawState st = row_state(a, r);
  const int nc = a.n_chunks;
  if (!st.any) {
    for (long long d = d0 + tid; d < d1; d += kPickThreads) { a.idx[out0 + d] = -1; if (a.prob) a.prob[out0 + d] = 0.f; }
    return;
  }
  // running sums over the row's chunks, one to a thread
  double t = tid < nc ? a.chunk_sum[(long long)r * nc + tid] : 0.0;
  for (int o = 1; o < 64; o <<= 1) { const double x = shfl_up_d(t, o); if (lane >= o) t += x; }
  if (lane == 63) wsum[tid >> 6] = t;
  const int n_groups = (int)(((long long)a.n_cols + kGroup - 1) / kGroup), per_chunk = a.chunk / kGroup, step = a.place_groups, per = per_chunk / step;
  const long long g0 = (long long)r * nc * per_chunk;
  // (what lies behind the row's last group is never looked at)
  for (int j = tid; j < nc * per; j += kPickThreads) { const int g = (j + 1) * step - 1; place[j] = g < n_groups ? a.group_incl[g0 + g] : __builtin_inf(); }
  __syncthreads();
  double before = 0.0;
  for (int j = 0; j < (tid >> 6); ++j) before += wsum[j];
  chunk_incl[tid] = before + t;
  __syncthreads();
  const double total = chunk_incl[kMaxChunks - 1];
  const RowView v = row_view<DT>(a, r);
  const double per_total = 1.0 / total;
  const float per_score = (float)(st.inv_t * 1.4426950408889634);
  const float per_octave = per_score >= 1e-37f ? per_score : __builtin_nanf("");      // (above 0, so that what is not kept is infinitely far; else fp64 decides)
  const DrawGroup* const groups = a.group + g0;
  // (whole wavefronts stay: lanes load for one another.  A lane without a draw of its own finds the one of u = 0.)
  for (long long first = d0 + (tid & ~63); first < d1; first += kPickThreads) {
    const long long d = first + lane;
    double u = d < d1 ? (double)a.u[(long long)r * a.u_stride + d] : 0.0;
    u = u > 0.0 ? (u < 1.0 ? u : 1.0 - 0x1p-24) : 0.0;
    const double target = u * total;                 // below the total: the last chunk passes it
    int ch = 0, hi = nc - 1;
    while (ch < hi) { const int mid = (ch + hi) >> 1; if (chunk_incl[mid] > target) hi = mid; else ch = mid + 1; }
    const double in_chunk = target - (ch ? chunk_incl[ch - 1] : 0.0);
    // the first place, group and block that pass it (the last ones, should rounding leave none)
    const int last_group = min((ch + 1) * per_chunk, n_groups) - 1;
    int lo = ch * per;
    hi = min(lo + per - 1, last_group / step);
    while (lo < hi) { const int mid = (lo + hi) >> 1; if (place[mid] > in_chunk) hi = mid; else lo = mid + 1; }
    int g = lo * step;
    hi = min(g + step - 1, last_group);
    double front = lo > ch * per ? place[lo - 1] : 0.0;
    while (g < hi) {
      const int mid = (g + hi) >> 1;
      const double x = a.group_incl[g0 + mid];
      if (x > in_chunk) hi = mid; else { g = mid + 1; front = x; }
    }
    double incl[8];
    uint4 bits;
    {
      unsigned x[4][4];
      load_records<4>((const char*)(groups + g), x);
      __builtin_memcpy(incl, x, 64);
    }
    __builtin_memcpy(&bits, groups[g].kept, 16);
    int b = 0;
    double back = incl[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) {
      const bool behind = incl[j - 1] <= in_chunk;
      b += behind ? 1 : 0;
      front = behind ? incl[j - 1] : front;
      back = behind ? incl[j] : back;
    }
    const unsigned half = b & 4 ? (b & 2 ? bits.w : bits.z) : (b & 2 ? bits.y : bits.x);
    unsigned kept = b & 1 ? half >> 16 : half & 0xffffu;
    double in_block = in_chunk - front;
    const double mass = back - front;
    int block = g * 8 + b;
    if (!kept) {
      // the target lies within rounding of a border: the first kept entry behind it, or the last before
      const int last_block = (int)(((long long)a.n_cols + kBlock - 1) / kBlock) - 1;
      while (!kept && block < last_block) { ++block; kept = groups[block >> 3].kept[block & 7]; }
      while (!kept && block > 0) { --block; kept = groups[block >> 3].kept[block & 7]; }
      in_block = -1.0;
    }
    const int i0 = block * kBlock;
    Four<DT> f[4];
    constexpr int es = DT == PSL_F32 ? 4 : 2;
    unsigned raw[4][es];                              // (two bytes to an entry: pieces of eight bytes)
    if (__any(i0 + kBlock > a.n_cols)) {
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = load_four<DT>(RowView{v.s, nullptr}, i0 + 4 * j, a.n_cols);
    } else {
      load_records<es>((const char*)v.s + (long long)i0 * es, raw);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if constexpr (DT == PSL_F32) f[j].s[k] = __uint_as_float(raw[j][k]);
          else if constexpr (DT == PSL_BF16) f[j].s[k] = __uint_as_float(k & 1 ? raw[j][k >> 1] & 0xffff0000u : raw[j][k >> 1] << 16);
          else { const unsigned short h = (unsigned short)(raw[j][k >> 1] >> (16 * (k & 1))); _Float16 x; __builtin_memcpy(&x, &h, 2); f[j].s[k] = (float)x; }
        }
    }
    // In fp32 first, weights relative to the block's largest: 16 exponentials of at most one unit of the last place and 15 sums
    // are within 35 * 2^-24 of the block's mass (x 2^-x <= 0.53 bounds what the rounded exponent does), the target's share
    // of it within 6 * 2^-24, so a border that is 2^-18 of it away is on the side it seems to be on.  One draw in ten thousand
    // is not that clear.
    float x[16], top = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < 16; ++j) { x[j] = (kept >> j) & 1u ? f[j >> 2].s[j & 3] : -__builtin_inff(); top = fmaxf(top, x[j]); }
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) { sum += __builtin_amdgcn_exp2f((x[j] - top) * per_octave); x[j] = sum; }
    const float share = (float)in_block * __builtin_amdgcn_rcpf((float)mass) * sum, room = sum * 0x1p-18f;
    // A share that is a number of at least 0 is passed by a kept entry: the sum in front of it is below share - room, the sum with
    // it above share + room.  fp64 decides where the share is no number (the block's mass has no fp32 reciprocal, its entries lie 88
    // temperatures below the largest, and u = 0 makes it 0 / 0) or below 0 (the block was stepped to from one without kept entries).
    // (the sums never fall: as many borders as lie in front of the target's)
    int at = 0, far = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) { at += x[j] < share - room ? 1 : 0; far += x[j] <= share + room ? 1 : 0; }
    if (at != far || at > 15 || !(share >= 0.f) || !(sum < 1e30f)) {
      // in fp64, entry by entry
      double acc = 0.0;
      at = -1;
      for (int j = 0; j < 16; ++j) {
        if ((kept >> j) & 1u) {
          const double w = weight_of(load_score<DT>(v.s, i0 + j), st.M, st.inv_t, s_exp);
          at = j;
          acc += w;
          if (acc > in_block) break;
        }
      }
    }
    if (d < d1) a.idx[out0 + d] = i0 + at;
    if (d < d1 && a.prob) {
      float s4[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) s4[j] = at & 2 ? (at & 1 ? f[j].s[3] : f[j].s[2]) : (at & 1 ? f[j].s[1] : f[j].s[0]);
      const float s = at & 8 ? (at & 4 ? s4[3] : s4[2]) : (at & 4 ? s4[1] : s4[0]);
      const double w = weight_of(s, st.M, st.inv_t, s_exp), p = w * per_total;
      a.prob[out0 + d] = (float)fma(fma(-p, total, w), per_total, p);      // the quotient, by its remainder
    }
  }
}

// ---------------------------------------------------------------- short rows: everything by one workgroup
// The same steps with the row in registers (up to 16 entries to a thread), all else in LDS: one launch instead of seven,
// whose starts and first loads are what a short row costs.
constexpr int kRowCols = 16384, kRowList = 1024;
struct RowShared {
  union { unsigned cnt[kBins]; double running[kBins]; };          // bin counts, later the blocks' running sums (kRowCols / kBlock = kBins)
  union { u64 mass[kBins]; double cum[kBins]; };
  union { double first[kBins]; double excl[kBins]; };
  u64 la[kRowList], lb[kRowList];
  unsigned short kept[kBins];
  CutShared cut;
  BinsShared bins;
  DrawCut c;
  unsigned n_a, n_b;
};
static_assert(kMaxParts * 256 / 64 <= kTops, "tops");
static_assert(sizeof(RowShared) <= 65536, "LDS");
template <int DT> __global__ __launch_bounds__(1024) void k_draw_row(DrawArgs a) {
  __shared__ RowShared S;
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const RowView v = row_view<DT>(a, r);
  const RowPar par = row_par(a, r);
  exp_table_init(S.cut.sh.exp);
  Four<DT> f[4];
  unsigned mx = 0u, mn = 0xffffffffu;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f[j].live = 0u;
    const int i = j * 4096 + tid * 4;
    if (i < a.n_cols) f[j] = load_four<DT>(v, i, a.n_cols);
#pragma unroll
    for (int q = 0; q < 4; ++q) { const unsigned k = four_key(f[j], q); mx = max(mx, k); mn = min(mn, k ? k : 0xffffffffu); }
  }
  for (int o = 32; o > 0; o >>= 1) { mx = max(mx, (unsigned)__shfl_xor((int)mx, o)); mn = min(mn, (unsigned)__shfl_xor((int)mn, o)); }
  if (lane == 0) { S.cut.sh.mx[tid >> 6] = mx; S.cut.sh.mn[tid >> 6] = mn; }
  S.cnt[tid] = 0u; S.mass[tid] = 0ull;
  if (tid == 0) { S.n_a = 0u; S.n_b = 0u; }
  __syncthreads();
  for (int j = 0; j < 16; ++j) { mx = max(mx, (unsigned)S.cut.sh.mx[j]); mn = min(mn, (unsigned)S.cut.sh.mn[j]); }
  const long long out0 = (long long)r * a.n_draws;
  if (!mx) {
    for (int d = tid; d < a.n_draws; d += 1024) { a.idx[out0 + d] = -1; if (a.prob) a.prob[out0 + d] = 0.f; }
    return;
  }
  const float M = score_of(mx);
  u64 thr = 1ull << 32;
  if (has_cut(par)) {
    const Range g{mx, mn};
    const Binning b = make_binning(g, par.inv_t, a.n_cols);
    const bool weigh = par.p < 1.0 && par.k != 1;
    const BinPoly poly = make_bin_poly();
    unsigned c = 0u;
    if (par.k > 0) {
      // Top-k by itself first: where it leaves few entries, a list of them is all that the rest needs, and no mass is.  (1 x 2 048, top-k
      // and top-p: 50 entries 14.8 us, 20.6 by masses, bins and sums; 800 entries 21.3 and 21.9.  Top-k alone, which weighs nothing
      // on the way: 100 entries 14.5 and 15.8, 400 18.4 and 16.1.)
#pragma unroll
      for (int j = 0; j < 4; ++j) add_to_bins<false>(f[j], b, poly, true, false, kBins - 1, S.cnt, S.mass, S.first);
      __syncthreads();
      c = S.cnt[tid];
      find_bins(a, par, g, b, c, 0.0, S.cum, S.excl, &S.c, S.bins);
      __syncthreads();
      if (S.c.k_bin < kBins && S.c.n_all && (weigh || S.c.n_all <= 128u)) {
        const int k_bin = S.c.k_bin;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const unsigned k = four_key(f[j], q);
            if (k && bin_of(b, score_of(k)) <= k_bin) S.la[atomicAdd(&S.n_a, 1u)] = number_of(k, j * 4096 + tid * 4 + q);
          }
        __syncthreads();
        draw_from_list(a, r, S.la, S.c, par, S.cut, S.running);
        return;
      }
      S.mass[tid] = 0ull;
    }
    if (weigh) {
      S.first[tid] = first_weight(b, tid);
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 4; ++j) add_to_bins<false>(f[j], b, poly, false, true, kBins - 1, S.cnt, S.mass, S.first);
      __syncthreads();
    }
    const double m = weigh ? ldexp((double)S.mass[tid], -bin_shift(b, tid)) : 0.0;
    __syncthreads();
    find_bins(a, par, g, b, c, m, S.cum, S.excl, &S.c, S.bins);
    __syncthreads();
    const DrawCut& cut = S.c;
    if (cut.k_bin < kBins || cut.p < 1.0) {
      const bool do_a = cut.k_bin < kBins && cut.n_a <= kRowList, do_b = cut.p_hi >= 0;
      const int ka = do_a ? cut.k_bin : -1, p0 = do_b ? cut.p_lo : 0, p1 = do_b ? cut.p_hi : -1;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const unsigned k = four_key(f[j], q);
          const int i = j * 4096 + tid * 4 + q, bin = k ? bin_of(b, score_of(k)) : -2;
          if (bin == ka) { const unsigned at = atomicAdd(&S.n_a, 1u); if (at < kRowList) S.la[at] = number_of(k, i); }
          if (bin >= p0 && bin <= p1) { const unsigned at = atomicAdd(&S.n_b, 1u); if (at < kRowList) S.lb[at] = number_of(k, i); }
        }
      __syncthreads();
      thr = find_threshold<DT>(v, a.n_cols, cut, S.la, S.lb, S.n_b, kRowList, S.cum, S.excl, S.cut);
    }
    __syncthreads();
  }
  // Running sums at the end of each block of 16 entries, and which of them are kept.  The row is read once more: its
  // registers held through the search above would spill.
  const Kept kp = kept_from(thr);
  const double least = fmax(par.m, 0x1p-1074);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f[j].live = 0u;
    if (j * 4096 + tid * 4 < a.n_cols) f[j] = load_four<DT>(v, j * 4096 + tid * 4, a.n_cols);
    double w;
    unsigned bits = kept_of_four(f[j], j * 4096 + tid * 4, kp, M, par.inv_t, least, S.cut.sh.exp, w);
    bits <<= 4 * (lane & 3);
    w += __shfl_xor(w, 1);
    w += __shfl_xor(w, 2);
    bits |= (unsigned)__shfl_xor((int)bits, 1);
    bits |= (unsigned)__shfl_xor((int)bits, 2);
    if ((tid & 3) == 0) { S.running[j * 256 + (tid >> 2)] = w; S.kept[j * 256 + (tid >> 2)] = (unsigned short)bits; }
  }
  __syncthreads();
  const double incl = block_running(S.running[tid], S.cut.wave);
  S.running[tid] = incl;
  __syncthreads();
  const double total = S.running[kBins - 1];
  const int last_block = (a.n_cols + kBlock - 1) / kBlock - 1;
  for (int d = tid; d < a.n_draws; d += 1024) {
    double u = (double)a.u[(long long)r * a.u_stride + d];
    u = u > 0.0 ? (u < 1.0 ? u : 1.0 - 0x1p-24) : 0.0;
    const double target = u * total;
    int lo = 0, hi = last_block;
    while (lo < hi) { const int mid = (lo + hi) >> 1; if (S.running[mid] > target) hi = mid; else lo = mid + 1; }
    double in_block = target - (lo ? S.running[lo - 1] : 0.0);
    unsigned kept = S.kept[lo];
    if (!kept) {
      // the target lies within rounding of a border: the first kept entry behind it, or the last before
      while (!kept && lo < last_block) kept = S.kept[++lo];
      while (!kept && lo > 0) kept = S.kept[--lo];
      in_block = -1.0;
    }
    double acc = 0.0, w_at = 0.0;
    int at = -1;
    while (kept) {
      const int j = __ffs((int)kept) - 1;
      kept &= kept - 1u;
      w_at = weight_of(load_score<DT>(v.s, lo * kBlock + j), M, par.inv_t, S.cut.sh.exp);
      at = lo * kBlock + j;
      acc += w_at;
      if (acc > in_block) break;
    }
    a.idx[out0 + d] = at;
    if (a.prob) a.prob[out0 + d] = (float)(w_at / total);
  }
}

// ---------------------------------------------------------------- host side
struct DrawLayout { int chunk, n_chunks, n_parts, part_len, list_cap, top_lanes, n_tops; size_t state, cut, chunk_sum, group, group_incl, part_max, part_min, tops, bin_cnt, bin_mass, bin_excl, list_a, list_b, total; };
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
  l.cut = take(sizeof(DrawCut) * n_rows);
  l.chunk_sum = take(sizeof(double) * n_rows * l.n_chunks);
  l.group = take(sizeof(DrawGroup) * n_rows * l.n_chunks * (l.chunk / kGroup));
  l.group_incl = take(sizeof(double) * n_rows * l.n_chunks * (l.chunk / kGroup));
  // Parts: up to 1 024 workgroups over all rows (four of 512 threads on each of 256 CUs: one round; 5 000 draws with
  // top-p from each of twelve rows of 816 000: 94 us, with 512 or 2 048 workgroups 100).  No part below 2 048 entries, and no
  // more than 96 parts below 8 192: a workgroup adds up to 1 024 bins to its row's.  (One row of 131 072, top-k and top-p: 28 us in
  // parts of 2 048, 29 of 4 096, 34 of 8 192; four of 307 200, top-p: 52, 48, 48.)
  const long long cols = n_cols > 0 ? n_cols : 1;
  long long most = (cols + 8191) / 8192 > 96 ? (cols + 8191) / 8192 : 96;
  if (most > (cols + 2047) / 2048) most = (cols + 2047) / 2048;
  if (most > kMaxParts) most = kMaxParts;
  long long parts = 1024 / (n_rows > 0 ? n_rows : 1);
  if (parts < 1) parts = 1;
  if (parts > most) parts = most;
  l.part_len = (int)(((cols + parts - 1) / parts + 2047) / 2048 * 2048);
  l.n_parts = (int)((cols + l.part_len - 1) / l.part_len);
  // Lists hold a quarter of a row (all of it up to 4 096 entries): more entries in one bin mean that many equal scores, and then the
  // row itself is read.
  l.list_cap = (int)(cols / 4 > 4096 ? cols / 4 : cols < 4096 ? cols : 4096);
  l.part_max = take(sizeof(unsigned) * n_rows * l.n_parts);
  l.part_min = take(sizeof(unsigned) * n_rows * l.n_parts);
  // maxima for last_bin: up to kTops of a row (kMaxParts * 256 / 64), of four lanes or more
  l.top_lanes = 4;
  while (l.n_parts * (256 / l.top_lanes) > kTops) l.top_lanes *= 2;
  l.n_tops = l.n_parts * (256 / l.top_lanes);
  l.tops = take(sizeof(unsigned) * n_rows * l.n_tops);
  l.bin_cnt = take(sizeof(unsigned) * n_rows * kBins);
  l.bin_mass = take(sizeof(u64) * n_rows * kBins);
  l.bin_excl = take(sizeof(double) * n_rows * kBins);
  l.list_a = take(sizeof(u64) * n_rows * l.list_cap);
  l.list_b = take(sizeof(u64) * n_rows * l.list_cap);
  l.total = o;
  return l;
}
// whether any row may have a limit, as far as the host knows
static bool may_cut(const psl_draw_args* q) {
  return q->temperature || q->top_k || q->top_p || !(q->temperature_all > 0.0) || q->top_k_all > 0 || q->top_p_all < 1.0;
}
// Short rows in one launch (1 x 2 048, top-k and top-p: 13.3 us, in seven 27; 256 x 16 384: 26 and 39).  A row's draws are then
// one workgroup's: without limits, where three launches would do, up to 1 024 of them (1 x 16 384: 18 and 21 us; for 2 048 24 and
// 21), with limits up to 4 096 (1 x 16 384, both: 30 and 35 us; for 16 384 46 and 42).
static bool in_one_launch(const psl_draw_args* q) { return q->n_cols <= kRowCols && q->n_draws <= (may_cut(q) ? 4096 : 1024); }
constexpr int64_t kNoWorkspace = 256;      // what a call asks for that uses none: `ws` is a pointer all the same
template <int DT> static void launch_draw(const DrawArgs& a, bool one_launch, hipStream_t s) {
  if (one_launch) {
    hipLaunchKernelGGL(k_draw_row<DT>, dim3(a.n_rows), dim3(1024), 0, s, a);
    return;
  }
  hipLaunchKernelGGL(k_draw_range<DT>, dim3(a.n_parts, a.n_rows), dim3(256), 0, s, a);
  if (a.cuts) {
    hipLaunchKernelGGL(k_draw_hist<DT>, dim3(a.n_parts, a.n_rows), dim3(512), 0, s, a);
    hipLaunchKernelGGL(k_draw_bins, dim3(a.n_rows), dim3(kBins), 0, s, a);
    hipLaunchKernelGGL(k_draw_gather<DT>, dim3(a.n_parts, a.n_rows), dim3(512), 0, s, a);
    hipLaunchKernelGGL(k_draw_cut<DT>, dim3(a.n_rows), dim3(1024), 0, s, a);
  }
  hipLaunchKernelGGL(k_draw_sums<DT>, dim3(a.n_chunks, a.n_rows), dim3(256), 0, s, a);
  hipLaunchKernelGGL(k_draw_pick<DT>, dim3((unsigned)(((long long)a.n_rows * a.pick_wgs + 7) / 8 * 8)), dim3(kPickThreads), 0, s, a);
}

}  // namespace psl
using namespace psl;

#define PSL_BAD(...) do { set_error(__VA_ARGS__); return PSL_ERR_ARG; } while (0)
extern "C" int64_t psl_draw_ws_bytes(int32_t n_rows, int32_t n_cols) {
  if (n_rows < 0 || n_cols < 0 || n_rows > 65535 || n_cols > 0x7f000000) PSL_BAD("psl_draw_ws_bytes: %d rows of %d", n_rows, n_cols);
  return (int64_t)draw_layout(n_rows, n_cols).total;
}
extern "C" int64_t psl_draw_call_ws_bytes(const psl_draw_args* q) {
  if (!q) PSL_BAD("psl_draw_call_ws_bytes: null argument");
  const int64_t all = psl_draw_ws_bytes(q->n_rows, q->n_cols);
  return all > kNoWorkspace && in_one_launch(q) ? kNoWorkspace : all;
}

extern "C" int psl_draw_indices(const psl_draw_args* q, void* stream) {
  if (!q) PSL_BAD("psl_draw_indices: null argument");
  if (q->dtype < PSL_F32 || q->dtype > PSL_F16) PSL_BAD("psl_draw_indices: unknown dtype %d", q->dtype);
  if (q->n_rows < 0 || q->n_rows > 65535 || q->n_cols < 0 || q->n_cols > 0x7f000000 || q->n_draws < 0)
    PSL_BAD("psl_draw_indices: %d rows (up to 65535) of %d entries, %d draws", q->n_rows, q->n_cols, q->n_draws);
  if ((long long)q->n_rows * q->n_draws > (1ll << 38)) PSL_BAD("psl_draw_indices: %d x %d draws", q->n_rows, q->n_draws);
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
  const bool one_launch = in_one_launch(q);
  const DrawLayout l = draw_layout(q->n_rows, q->n_cols);
  const int64_t need = one_launch ? kNoWorkspace : (int64_t)l.total;
  if (q->ws_bytes < need) PSL_BAD("psl_draw_indices: workspace of %lld bytes, %lld needed", (long long)q->ws_bytes, (long long)need);
  DrawArgs a{};
  a.n_rows = q->n_rows; a.n_cols = q->n_cols; a.n_draws = q->n_draws;
  a.scores = q->scores; a.stride = q->score_stride; a.mask = q->mask; a.mask_stride = q->mask_stride;
  a.temperature = q->temperature; a.top_k = q->top_k; a.top_p = q->top_p; a.min_p = q->min_p;
  a.t_all = q->temperature_all; a.p_all = q->top_p_all; a.m_all = q->min_p_all; a.k_all = q->top_k_all;
  a.u = q->u; a.u_stride = q->u_stride; a.idx = q->idx; a.prob = q->prob;
  // (the row kernel keeps everything in LDS: its pointers into the workspace stay null)
  if (!one_launch) {
    char* w = (char*)q->ws;
    a.state = (DrawState*)(w + l.state); a.cut = (DrawCut*)(w + l.cut); a.chunk_sum = (double*)(w + l.chunk_sum); a.group = (DrawGroup*)(w + l.group);
    a.group_incl = (double*)(w + l.group_incl);
    a.part_max = (unsigned*)(w + l.part_max); a.part_min = (unsigned*)(w + l.part_min); a.tops = (unsigned*)(w + l.tops);
    a.bin_cnt = (unsigned*)(w + l.bin_cnt); a.bin_mass = (u64*)(w + l.bin_mass); a.bin_excl = (double*)(w + l.bin_excl);
    a.list_a = (u64*)(w + l.list_a); a.list_b = (u64*)(w + l.list_b);
  }
  a.n_chunks = l.n_chunks; a.chunk = l.chunk; a.n_parts = l.n_parts; a.part_len = l.part_len; a.top_lanes = l.top_lanes; a.n_tops = l.n_tops;
  a.list_cap = l.list_cap;
  a.cuts = may_cut(q);
  // A row's workgroup draws from its list: 64 x 131 072 with top-k and top-p, one draw of each: 42 us, by sums and k_draw_pick 59; for
  // 16 384 draws 52 and 84; of a single row 43 and 43, and more draws want more workgroups.
  a.listed_draws = a.cuts && a.n_draws <= 16384;
  // Draws to a workgroup: its start costs a pass over the row's running sums, so several to a thread once the card is full (two
  // workgroups on each of 256 CUs): twelve rows of 816 000, 124 800 draws of each, nothing cut: 83 us, with one to a thread 91.
  a.pick_len = kPickThreads;
  while (a.pick_len < 16 * kPickThreads && (long long)a.n_rows * a.n_draws / a.pick_len >= 512) a.pick_len += kPickThreads;
  a.pick_wgs = (int)((a.n_draws + a.pick_len - 1) / a.pick_len);
  // Places in LDS: every group's end if they fit, else every second, fourth ...  Fewer draws than twice the groups do not repay
  // filling them and start from the chunks (twelve rows of 816 000: 48 and 47 us for 1 024 draws of each, 69 and 76 for 65 536).
  const int per_chunk = a.chunk / kGroup;
  a.place_groups = 1;
  while ((long long)a.n_chunks * (per_chunk / a.place_groups) > (a.n_draws / 2 > a.n_cols / kGroup ? kPlaces : a.n_chunks))
    a.place_groups = per_chunk % (2 * a.place_groups) == 0 ? 2 * a.place_groups : per_chunk;
  hipStream_t s = (hipStream_t)stream;
  if (q->dtype == PSL_F32) launch_draw<PSL_F32>(a, one_launch, s);
  else if (q->dtype == PSL_BF16) launch_draw<PSL_BF16>(a, one_launch, s);
  else launch_draw<PSL_F16>(a, one_launch, s);
  PSL_LAUNCH_CHECK();
  return PSL_OK;
#undef PSL_BAD
}
