// Feature rows held in 8 or 4 bits: quantised as they are written, expanded as they are read.
//
// A row is heads x dim values, cut into groups of G; a group shares one fp32 scale s = max|x| / Q (Q = 127 int8, 7 int4,
// 448 e4m3; rounded to nearest, down where Q s would not be finite) and every code is the NEAREST representable value to x / s,
// ties to even.  fp32's x / s cannot decide that by itself: it rounds quotients beside the middle between two codes onto it (with
// bf16 inputs x = a / 2 that happens in every few rows).  What decides is the residual x - n s, which one fma gives exactly:
//   integers: n = rint(x / s), and x - n s against s / 2 says whether n is the nearest (it nearly always is);
//   e4m3: the quotient rounded to ODD -- truncated, its last bit set when the residual is not zero.  Rounding that 24-bit value
//   once more, to four bits, is the rounding of the exact quotient.
//
// Bound: memory.  A thread owns VEC consecutive values; the lanes of a group find its maximum by moves between lanes, so a value
// is read once and lives in registers until its code is stored.  2.5 M rows of 2 x 32 fp32 to 8 bits and back: 295 us
// for the pair, 5.6 TB/s of the 820 MB that each reads and writes (kernel trace: 165 and 144 in turn; 140 and 142 each by itself),
// where a copy of 1 GiB reaches 5.07 and one of 256 MiB 5.31 (codes and scales fit the 256 MB cache between the two calls).
#include "psl_common.h"

namespace psl {

struct FastDiv {          // x / d for 0 <= x < 2^31: one multiply-high
  unsigned d, m, s;
};
static FastDiv make_fastdiv(unsigned d) {
  FastDiv f{d, 0u, 0u};
  if (d > 1) {
    unsigned s = 0;
    while ((1ull << s) < d) ++s;
    // m = ceil(2^(31+s) / d) < 2^32; the excess m d - 2^(31+s) < d <= 2^s keeps the quotient exact below 2^31
    f.m = (unsigned)(((1ull << (31 + s)) + d - 1) / d);
    f.s = s - 1;
  }
  return f;
}
__device__ __forceinline__ unsigned fast_div(unsigned x, const FastDiv& f) { return f.d == 1 ? x : __umulhi(x, f.m) >> f.s; }

struct RowsArgs {
  const void* rows;        // destination / source row ids, or NULL: first + i
  long long first, capacity, i0;      // i0: first row of this launch (launches cover < 2^31 groups each)
  char* values; unsigned vrow, vhead;           // bytes
  unsigned char* codes; unsigned crow;          // bytes per row; a head holds dim * bits / 8
  float* scales; unsigned srow;                 // floats per row
  const int* owner;        // write: row -> last i that writes it (NULL: the rows are distinct)
  unsigned n;              // rows of this launch
  unsigned group, chunks;                       // values of a group; chunks = group / VEC
  bool heads_apart;                             // the heads of a row of values do not follow one another
  int lanes_log2;          // lanes that share a group
  FastDiv groups_per_row, groups_per_head;
  int rows_bits;           // 32 | 64
};

__device__ __forceinline__ long long row_of(const RowsArgs& a, long long i) {
  if (!a.rows) return a.first + i;
  const long long r = a.rows_bits == 64 ? ((const long long*)a.rows)[i] : (long long)((const int*)a.rows)[i];
  return (r < 0 || r >= a.capacity) ? -1 : r;
}

// ---- VEC values of a type as floats; VEC * sizeof(T) bytes at an address that holds that much alignment (at most 16 B)
template <int BYTES> struct Raw { unsigned w[BYTES / 4]; };
template <> struct Raw<2> { unsigned short w[1]; };
template <> struct Raw<1> { unsigned char w[1]; };
template <int BYTES> __device__ __forceinline__ Raw<BYTES> load_raw(const void* p) {
  Raw<BYTES> r;
  if constexpr (BYTES >= 16) {
#pragma unroll
    for (int k = 0; k < BYTES / 16; ++k) {
      const uint4 t = ((const uint4*)p)[k];
      r.w[4 * k] = t.x; r.w[4 * k + 1] = t.y; r.w[4 * k + 2] = t.z; r.w[4 * k + 3] = t.w;
    }
  } else if constexpr (BYTES == 8) { const uint2 t = *(const uint2*)p; r.w[0] = t.x; r.w[1] = t.y; }
  else if constexpr (BYTES == 4) r.w[0] = *(const unsigned*)p;
  else if constexpr (BYTES == 2) r.w[0] = *(const unsigned short*)p;
  else r.w[0] = *(const unsigned char*)p;
  return r;
}
template <int BYTES> __device__ __forceinline__ void store_raw(void* p, const Raw<BYTES>& r) {
  if constexpr (BYTES >= 16) {
#pragma unroll
    for (int k = 0; k < BYTES / 16; ++k) ((uint4*)p)[k] = make_uint4(r.w[4 * k], r.w[4 * k + 1], r.w[4 * k + 2], r.w[4 * k + 3]);
  } else if constexpr (BYTES == 8) *(uint2*)p = make_uint2(r.w[0], r.w[1]);
  else if constexpr (BYTES == 4) *(unsigned*)p = r.w[0];
  else if constexpr (BYTES == 2) *(unsigned short*)p = (unsigned short)r.w[0];
  else *(unsigned char*)p = (unsigned char)r.w[0];
}

template <int DT> struct Elem { static constexpr int bytes = DT == PSL_F32 ? 4 : 2; };
template <int DT> __device__ __forceinline__ float elem_f(unsigned short h) {
  if constexpr (DT == PSL_BF16) return __uint_as_float((unsigned)h << 16);
  else { _Float16 f; __builtin_memcpy(&f, &h, 2); return (float)f; }
}
template <int DT, int VEC> __device__ __forceinline__ void load_values(const char* p, float (&x)[VEC]) {
  if constexpr (VEC <= 2) {        // what is left where pieces of four are not aligned: element by element
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      if constexpr (DT == PSL_F32) x[k] = ((const float*)p)[k];
      else x[k] = elem_f<DT>(((const unsigned short*)p)[k]);
    }
    return;
  } else {
  const Raw<VEC * Elem<DT>::bytes> r = load_raw<VEC * Elem<DT>::bytes>(p);
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    if constexpr (DT == PSL_F32) x[k] = __uint_as_float(r.w[k]);
    else x[k] = elem_f<DT>((unsigned short)(r.w[k / 2] >> (16 * (k & 1))));
  }
  }
}
template <int DT> __device__ __forceinline__ unsigned short half_bits(float x) {      // one rounding, to nearest even
  unsigned short h;
  if constexpr (DT == PSL_BF16) { const __bf16 b = (__bf16)x; __builtin_memcpy(&h, &b, 2); }
  else { const _Float16 b = (_Float16)x; __builtin_memcpy(&h, &b, 2); }
  return h;
}
template <int DT, int VEC> __device__ __forceinline__ void store_values(char* p, const float (&x)[VEC]) {
  if constexpr (VEC <= 2) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      if constexpr (DT == PSL_F32) ((float*)p)[k] = x[k];
      else ((unsigned short*)p)[k] = half_bits<DT>(x[k]);
    }
  } else {
    Raw<VEC * Elem<DT>::bytes> r;
    if constexpr (DT == PSL_F32) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) r.w[k] = __float_as_uint(x[k]);
    } else {
#pragma unroll
      for (int k = 0; k < VEC / 2; ++k) r.w[k] = (unsigned)half_bits<DT>(x[2 * k]) | ((unsigned)half_bits<DT>(x[2 * k + 1]) << 16);
    }
    store_raw(p, r);
  }
}

template <int FMT> struct Code {
  static constexpr int bits = FMT == PSL_ROWS_INT4 ? 4 : 8;
  static constexpr float top = FMT == PSL_ROWS_INT8 ? 127.f : FMT == PSL_ROWS_INT4 ? 7.f : 448.f;
  // the largest scale whose product with the largest code is finite: below fl32(largest number / top) for 127, that number for 7 and 448
  static constexpr float most = FMT == PSL_ROWS_INT8 ? 0x1.020406p+121f : __builtin_inff();
};

// x / s rounded to odd, sign carried (s > 0, inv = 1 / s to a few units of the last place, the residual not denormal)
__device__ __forceinline__ float quotient_odd(float x, float s, float inv) {
  const float ax = fabsf(x);
  const float q0 = ax * inv;
  const float q = fmaf(fmaf(-q0, s, ax), inv, q0);       // within one unit of the last place of the exact quotient
  const float e = fmaf(-q, s, ax);                       // its exact remainder's sign
  unsigned b = __float_as_uint(q);
  b -= (e < 0.f) ? 1u : 0u;
  b |= (e != 0.f) ? 1u : 0u;
  return copysignf(__uint_as_float(b), x);
}

// codes of VEC values, as the numbers they are (integers; e4m3: rounded to odd, the conversion does the rest)
template <int FMT, int VEC> __device__ __forceinline__ void quotients(const float (&x)[VEC], float s, float inv, float (&q)[VEC]) {
  if constexpr (FMT == PSL_ROWS_E4M3) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) q[k] = quotient_odd(x[k], s, inv);
  } else {
    float far = -1.f;
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      q[k] = rintf(x[k] * inv);
      const float r = fmaf(-q[k], s, x[k]);              // exact: a multiple of the smaller last place, below s
      far = fmaxf(far, fmaf(2.f, fabsf(r), -s));         // above 0: a neighbour is nearer; 0: a tie
    }
    if (far >= 0.f && s > 0.f) {   // (a scale that underflowed to 0: all codes are 0)
      asm volatile("");            // (a branch: rarely taken)
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        // above the middle, or on it with an odd code: at least 0 for an odd one, the smallest number above 0 for an even one
        // (no branch: groups of bf16 reach the middle often enough that half the wavefronts come here)
        const float r = fmaf(-q[k], s, x[k]), h = fmaf(2.f, fabsf(r), -s);
        const float least = __uint_as_float(((unsigned)(int)q[k] & 1u) ^ 1u);
        q[k] += h >= least ? copysignf(1.f, r) : 0.f;
      }
    }
  }
}
// the same where the largest value is below 2^-60: scaled by 2^80, so that residuals are not denormal; a scale in the
// denormals is coarse, and the quotient may pass the largest code
template <int FMT, int VEC> __device__ __forceinline__ void quotients_tiny(const float (&x)[VEC], float s, float (&q)[VEC]) {
  constexpr float f = 0x1p80f;
  const float ss = s * f, inv = 1.f / ss;
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    const float y = fminf(fmaxf(quotient_odd(x[k] * f, ss, inv), -Code<FMT>::top), Code<FMT>::top);
    q[k] = s > 0.f ? (FMT == PSL_ROWS_E4M3 ? y : rintf(y)) : 0.f;
  }
}

template <int FMT, int VEC> __device__ __forceinline__ void encode(const float (&q)[VEC], unsigned char* dst) {
  constexpr int BYTES = VEC * Code<FMT>::bits / 8;
  Raw<BYTES> r;
  if constexpr (FMT == PSL_ROWS_E4M3) {
    if constexpr (VEC == 1) r.w[0] = (unsigned char)(__builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[0], 0, false) & 0xff);
    else if constexpr (VEC == 2) r.w[0] = (unsigned short)(__builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false) & 0xffff);
    else {
#pragma unroll
      for (int k = 0; k < VEC / 4; ++k) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * k], q[4 * k + 1], 0, false);
        r.w[k] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(q[4 * k + 2], q[4 * k + 3], w, true);
      }
    }
  } else {
    // 16 bits of codes at a time as ONE number, q0 + 2^B q1 + ..., made in fp32 with every code raised by half its range: it is below
    // 2^16, so every product and sum is exact; half a range more is the sign bit turned over.
    constexpr int B = Code<FMT>::bits, PER = (BYTES >= 4 ? 32 : BYTES * 8) / B;      // codes per stored word
    constexpr int RUN = PER * B > 16 ? 16 / B : PER;
    constexpr unsigned HALF = B == 4 ? 0x88888888u : 0x80808080u;
#pragma unroll
    for (int k = 0; k < VEC / PER; ++k) {
      unsigned w = 0;
#pragma unroll
      for (int h = 0; h < PER / RUN; ++h) {
        float t = q[k * PER + h * RUN] + (float)(HALF & ((1u << (RUN * B)) - 1u));
#pragma unroll
        for (int j = 1; j < RUN; ++j) t = fmaf(q[k * PER + h * RUN + j], (float)(1u << (B * j)), t);
        w |= (unsigned)t << (16 * h);
      }
      r.w[k] = w ^ (PER * B == 32 ? HALF : HALF & ((1u << (PER * B)) - 1u));
    }
  }
  store_raw(dst, r);
}

template <int FMT, int VEC> __device__ __forceinline__ void decode(const unsigned char* src, float (&q)[VEC]) {
  constexpr int BYTES = VEC * Code<FMT>::bits / 8;
  const Raw<BYTES> r = load_raw<BYTES>(src);
  if constexpr (FMT == PSL_ROWS_E4M3) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const int w = (int)r.w[k / 4];
      const int b = k & 3;
      q[k] = b == 0 ? __builtin_amdgcn_cvt_f32_fp8(w, 0) : b == 1 ? __builtin_amdgcn_cvt_f32_fp8(w, 1)
             : b == 2 ? __builtin_amdgcn_cvt_f32_fp8(w, 2) : __builtin_amdgcn_cvt_f32_fp8(w, 3);
    }
  } else {
    constexpr int B = Code<FMT>::bits, PER = (BYTES >= 4 ? 32 : BYTES * 8) / B;
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const unsigned w = (unsigned)r.w[k / PER];
      q[k] = (float)((int)(w << (32 - B - B * (k % PER))) >> (32 - B));
    }
  }
}

// the place of group `unit`: row i of the call (inside this launch), row of the store (-1: none), group u of the row.  Codes and
// scales of a row's groups lie one behind the other; 32 x 32 -> 64 bit products reach every address.
struct Place { unsigned i, u; int row; };
__device__ __forceinline__ Place place_in_call(const RowsArgs& a, unsigned unit) {
  Place p;
  p.i = fast_div(unit, a.groups_per_row);
  p.u = unit - p.i * a.groups_per_row.d;
  p.row = -1;
  return p;
}
__device__ __forceinline__ Place place_of(const RowsArgs& a, unsigned unit) {
  Place p = place_in_call(a, unit);
  p.row = (int)row_of(a, a.i0 + p.i);
  return p;
}
__device__ __forceinline__ char* values_at(const RowsArgs& a, const Place& p, unsigned es) {
  char* v = a.values + (unsigned long long)p.i * a.vrow;
  if (!a.heads_apart) return v + p.u * a.group * es;
  const unsigned head = fast_div(p.u, a.groups_per_head);
  return v + (unsigned long long)head * a.vhead + (p.u - head * a.groups_per_head.d) * a.group * es;
}
template <int BITS> __device__ __forceinline__ unsigned char* codes_at(const RowsArgs& a, const Place& p) {
  return a.codes + (unsigned long long)(unsigned)p.row * a.crow + (p.u * a.group * BITS >> 3);
}
__device__ __forceinline__ float* scale_at(const RowsArgs& a, const Place& p) { return a.scales + (unsigned long long)(unsigned)p.row * a.srow + p.u; }

// The last of several i with the same row wins: clear the rows' entries, then keep the largest i (two launches: a maximum
// does not depend on the order of the atomics).
__global__ __launch_bounds__(256) void k_rows_owner_clear(RowsArgs a, int* __restrict__ owner) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.n) return;
  const long long r = row_of(a, i);
  if (r >= 0) owner[r] = -1;
}
__global__ __launch_bounds__(256) void k_rows_owner_claim(RowsArgs a, int* __restrict__ owner) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.n) return;
  const long long r = row_of(a, i);
  if (r >= 0) atomicMax(&owner[r], (int)i);
}

// ITERS chunks of a group per lane (lane, lane + L, ...), held in registers between the maximum and the codes
template <int CTRL> __device__ __forceinline__ unsigned max_dpp(unsigned x) {
  return max(x, (unsigned)__builtin_amdgcn_mov_dpp((int)x, CTRL, 0xf, 0xf, true));
}
// maximum over the 2^k lanes of a group (aligned to them)
__device__ __forceinline__ unsigned group_max(unsigned x, int k) {
  if (k > 0) x = max_dpp<0xb1>(x);        // quad_perm 1 0 3 2
  if (k > 1) x = max_dpp<0x4e>(x);        // quad_perm 2 3 0 1
  if (k > 2) x = max_dpp<0x141>(x);       // row_half_mirror: the other four of eight, which agree by now
  if (k > 3) x = max_dpp<0x140>(x);       // row_mirror: the other eight of sixteen
  if (k > 4) x = max(x, (unsigned)__shfl_xor((int)x, 16));
  if (k > 5) x = max(x, (unsigned)__shfl_xor((int)x, 32));
  return x;
}

template <int FMT, int DT, int VEC, int ITERS>
__global__ __launch_bounds__(256) void k_rows_write(RowsArgs a) {
  const unsigned t = blockIdx.x * 256u + threadIdx.x;
  const unsigned unit = t >> a.lanes_log2;
  // Whole wavefronts stay for the maximum; a group's lanes are in range together.  Lanes without a group read the first
  // one's values, lanes without a chunk their group's last: what they add to a maximum is in it already or not used.
  const bool in = unit < a.n * a.groups_per_row.d;
  Place p = place_in_call(a, in ? unit : 0u);
  const unsigned L = 1u << a.lanes_log2, lane = t & (L - 1u);
  float x[ITERS][VEC];
  unsigned top_bits = 0u;         // |x| as bits: ordered like the magnitudes, infinities and NaN above them
  const char* v = values_at(a, p, Elem<DT>::bytes);
#pragma unroll
  for (int it = 0; it < ITERS; ++it) load_values<DT, VEC>(v + min(lane + it * L, a.chunks - 1u) * (unsigned)(VEC * Elem<DT>::bytes), x[it]);
  p.row = (int)row_of(a, a.i0 + p.i);       // (its load behind those of the values: none waits for the other)
#pragma unroll
  for (int it = 0; it < ITERS; ++it) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) top_bits = max(top_bits, __float_as_uint(x[it][k]) & 0x7fffffffu);
  }
  top_bits = group_max(top_bits, a.lanes_log2);
  if (!in || p.row < 0 || (a.owner && a.owner[p.row] != (int)(a.i0 + p.i))) return;
  // an infinite or NaN value makes the whole group NaN: it is not hidden, and nothing finite is made of it
  const float top = __uint_as_float(top_bits);
  const float s = top_bits < 0x7f800000u ? fminf(top / Code<FMT>::top, Code<FMT>::most) : __builtin_nanf("");
  const bool tiny = top < 0x1p-60f && s > 0.f;
  const float inv = s > 0.f ? __builtin_amdgcn_rcpf(s) : 0.f;
  unsigned char* cd = codes_at<Code<FMT>::bits>(a, p);
#pragma unroll
  for (int it = 0; it < ITERS; ++it) {
    const unsigned c = lane + it * L;
    if (c < a.chunks) {
      float q[VEC];
      quotients<FMT, VEC>(x[it], s, inv, q);
      if (tiny) { asm volatile(""); quotients_tiny<FMT, VEC>(x[it], s, q); }      // (the asm keeps this a branch, for groups below 2^-60 alone)
      encode<FMT, VEC>(q, cd + (c * (unsigned)VEC * Code<FMT>::bits >> 3));
    }
  }
  if (lane == 0) *scale_at(a, p) = s;
}

// one chunk of VEC codes per thread
template <int FMT, int DT, int VEC>
__global__ __launch_bounds__(256) void k_rows_read(RowsArgs a, FastDiv chunks, unsigned total) {
  const unsigned t = blockIdx.x * 256u + threadIdx.x;
  if (t >= total) return;
  const unsigned unit = fast_div(t, chunks);
  const unsigned c = t - unit * chunks.d;
  const Place p = place_of(a, unit);
  float y[VEC];
  if (p.row >= 0) {
    const float s = *scale_at(a, p);
    decode<FMT, VEC>(codes_at<Code<FMT>::bits>(a, p) + (c * (unsigned)VEC * Code<FMT>::bits >> 3), y);
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      y[k] *= s;
      // an fp32 number, then converted: one instruction for both (the compiler's choice for fp16, element by element) rounds the
      // exact product instead, and a value would depend on the width of the pieces
      asm("" : "+v"(y[k]));
    }
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k) y[k] = 0.f;
  }
  store_values<DT, VEC>(values_at(a, p, Elem<DT>::bytes) + c * (unsigned)(VEC * Elem<DT>::bytes), y);
}

// chunks of a group that one lane holds at most: 64 lanes x 8 x VEC >= 1024 from pairs on, single elements need 16
// (a lane with one chunk has a kernel of its own: 54 000 rows 3.8 us, in the general one 6.2)
constexpr int max_iters(int vec) { return vec == 1 ? 16 : 8; }
template <int FMT, int DT, int VEC> static void launch_write(const RowsArgs& a, unsigned grid, hipStream_t s) {
  const unsigned iters = (a.chunks + (1u << a.lanes_log2) - 1u) >> a.lanes_log2;
  if (iters == 1) hipLaunchKernelGGL((k_rows_write<FMT, DT, VEC, 1>), dim3(grid), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((k_rows_write<FMT, DT, VEC, max_iters(VEC)>), dim3(grid), dim3(256), 0, s, a);
}
template <int FMT, int DT, int VEC> static void launch_read(const RowsArgs& a, hipStream_t s) {
  const unsigned total = a.n * a.groups_per_row.d * a.chunks;
  hipLaunchKernelGGL((k_rows_read<FMT, DT, VEC>), dim3((total + 255) / 256), dim3(256), 0, s, a, make_fastdiv(a.chunks), total);
}
template <int FMT, int DT> static void dispatch(const RowsArgs& a, int vec, bool write, unsigned grid, hipStream_t s) {
#define PSL_ROWS_CASE(V) if (vec == V) { if (write) launch_write<FMT, DT, V>(a, grid, s); else launch_read<FMT, DT, V>(a, s); return; }
  PSL_ROWS_CASE(8) PSL_ROWS_CASE(4) PSL_ROWS_CASE(2)
  if constexpr (FMT != PSL_ROWS_INT4) { PSL_ROWS_CASE(1) }      // two int4 codes share a byte
#undef PSL_ROWS_CASE
}
template <int FMT> static void dispatch(const RowsArgs& a, int dtype, int vec, bool write, unsigned grid, hipStream_t s) {
  if (dtype == PSL_F32) dispatch<FMT, PSL_F32>(a, vec, write, grid, s);
  else if (dtype == PSL_BF16) dispatch<FMT, PSL_BF16>(a, vec, write, grid, s);
  else dispatch<FMT, PSL_F16>(a, vec, write, grid, s);
}

static int run_rows(const char* who, const psl_rows_args* q, bool write, hipStream_t s) {
#define PSL_BAD(...) do { set_error(__VA_ARGS__); return PSL_ERR_ARG; } while (0)
  if (!q) PSL_BAD("%s: null argument", who);
  if (q->format < PSL_ROWS_INT8 || q->format > PSL_ROWS_INT4) PSL_BAD("%s: unknown format %d", who, q->format);
  if (q->dtype < PSL_F32 || q->dtype > PSL_F16) PSL_BAD("%s: unknown dtype %d", who, q->dtype);
  if (q->heads < 1 || q->heads > 4096 || q->dim < 1 || q->dim > 4096 || q->group < 1 || q->group > 1024 || q->dim % q->group)
    PSL_BAD("%s: heads %d, dim %d, group %d (heads and dim up to 4096, group up to 1024 and a divisor of dim)", who, q->heads, q->dim, q->group);
  const int bits = q->format == PSL_ROWS_INT4 ? 4 : 8, es = q->dtype == PSL_F32 ? 4 : 2;
  if (bits == 4 && (q->group & 1)) PSL_BAD("%s: two int4 codes share a byte: group %d must be even", who, q->group);
  if (q->n < 0 || q->n > 0x7fffffffll || q->capacity < 0 || q->capacity > 0x7fffffffll) PSL_BAD("%s: n %lld, capacity %lld", who, (long long)q->n, (long long)q->capacity);
  if (q->n == 0) return PSL_OK;
  if (!q->values || !q->codes || !q->scales) PSL_BAD("%s: missing pointer", who);
  if (q->rows ? (q->rows_bits != 32 && q->rows_bits != 64) : (q->first < 0 || q->first > q->capacity || q->n > q->capacity - q->first))
    PSL_BAD("%s: rows [%lld, +%lld) of %lld (rows_bits %d)", who, (long long)q->first, (long long)q->n, (long long)q->capacity, q->rows_bits);
  const long long hd = (long long)q->heads * q->dim;
  const long long big = 1ll << 29;          // strides in bytes stay below 2^31
  if (q->value_row_stride < 0 || q->value_head_stride < 0 || q->value_row_stride > big || q->value_head_stride > big || q->codes_row_stride > big || q->scales_row_stride > big ||
      q->codes_row_stride < hd * bits / 8 || q->scales_row_stride < hd / q->group)
    PSL_BAD("%s: bad stride", who);
  // heads inside their row and rows one behind the other, or rows inside their head and heads one behind the other
  const long long vr = q->value_row_stride, vh = q->value_head_stride;
  const bool by_row = (q->heads == 1 || vh >= q->dim) && (q->n == 1 || vr >= (q->heads - 1) * vh + q->dim);
  const bool by_head = (q->n == 1 || vr >= q->dim) && (q->heads == 1 || vh >= (q->n - 1) * vr + q->dim);
  if (!write && !by_row && !by_head) PSL_BAD("%s: rows of the output overlap", who);
  const uintptr_t pv = (uintptr_t)q->values, pc = (uintptr_t)q->codes, ps = (uintptr_t)q->scales;
  if (pv % es || ps % 4 || (q->rows && (uintptr_t)q->rows % (q->rows_bits / 8))) PSL_BAD("%s: misaligned pointer", who);
  // VEC: the widest piece that divides a group and that every address keeps aligned (16-byte loads of values, code words of
  // VEC * bits / 8 bytes).  2.5 M fp32 rows of 2 x 32 to 8 bits, written and read: 140 and 142 us in pieces of 8, 155 and 155 of
  // 4, 249 and 232 of 2, 473 and 395 one by one.
  int vec = 8;
  for (; vec > 1; vec >>= 1) {
    const int va = vec <= 2 ? es : vec * es < 16 ? vec * es : 16, ca = vec * bits / 8;
    if (q->group % vec == 0 && pv % va == 0 && (q->value_row_stride * es) % va == 0 && (q->value_head_stride * es) % va == 0 &&
        pc % ca == 0 && q->codes_row_stride % ca == 0)
      break;
    if (bits == 4 && vec == 2) break;
  }
  RowsArgs a;
  a.rows = q->rows; a.rows_bits = q->rows_bits; a.first = q->first; a.capacity = q->capacity;
  a.vrow = (unsigned)(q->value_row_stride * es); a.vhead = (unsigned)(q->value_head_stride * es);
  a.codes = (unsigned char*)q->codes; a.crow = (unsigned)q->codes_row_stride; a.scales = q->scales; a.srow = (unsigned)q->scales_row_stride;
  a.heads_apart = q->heads > 1 && q->value_head_stride != q->dim;
  a.owner = write && q->rows ? q->owner : nullptr;
  a.group = (unsigned)q->group; a.chunks = (unsigned)(q->group / vec);
  a.groups_per_row = make_fastdiv((unsigned)(hd / q->group)); a.groups_per_head = make_fastdiv((unsigned)(q->dim / q->group));
  // Lanes of a group: a chunk to each, up to 64 lanes.  Groups of 80 = ten chunks leave six of sixteen idle and still win: 200 000
  // rows of three in fp32 take 34 us, 38 with five chunks to each of two lanes (fp16: 37 and 31; 4 099 rows: 3.2 and 5.3).
  int l = 0;
  while (l < 6 && (1u << l) < a.chunks) ++l;
  a.lanes_log2 = l;
  if (a.owner) {
    a.i0 = 0; a.n = (unsigned)q->n; a.values = (char*)q->values;
    const unsigned grid = (unsigned)((q->n + 255) / 256);
    hipLaunchKernelGGL(k_rows_owner_clear, dim3(grid), dim3(256), 0, s, a, q->owner);
    hipLaunchKernelGGL(k_rows_owner_claim, dim3(grid), dim3(256), 0, s, a, q->owner);
  }
  // launches of fewer than 2^30 threads: the 32-bit divisions above stay exact
  const long long per_row = (hd / q->group) * ((long long)a.chunks > (1 << l) ? a.chunks : (1 << l));
  const long long step = (1ll << 30) / per_row;
  for (long long i0 = 0; i0 < q->n; i0 += step) {
    a.i0 = i0; a.n = (unsigned)(q->n - i0 < step ? q->n - i0 : step);
    a.values = (char*)q->values + i0 * q->value_row_stride * es;
    const unsigned grid = (unsigned)((((long long)a.n * a.groups_per_row.d << l) + 255) / 256);
    if (q->format == PSL_ROWS_INT8) dispatch<PSL_ROWS_INT8>(a, q->dtype, vec, write, grid, s);
    else if (q->format == PSL_ROWS_E4M3) dispatch<PSL_ROWS_E4M3>(a, q->dtype, vec, write, grid, s);
    else dispatch<PSL_ROWS_INT4>(a, q->dtype, vec, write, grid, s);
  }
  PSL_LAUNCH_CHECK();
  return PSL_OK;
#undef PSL_BAD
}

}  // namespace psl
using namespace psl;

extern "C" int psl_rows_write(const psl_rows_args* a, void* stream) { return run_rows("psl_rows_write", a, true, (hipStream_t)stream); }
extern "C" int psl_rows_read(const psl_rows_args* a, void* stream) { return run_rows("psl_rows_read", a, false, (hipStream_t)stream); }
