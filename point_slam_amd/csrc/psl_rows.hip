// Feature rows held in 8 or 4 bits: quantised as they are written, expanded as they are read.
//
// A row is heads x dim values, cut into groups of G; a group shares one fp32 scale s = max|x| / Q (Q = 127 int8, 7 int4,
// 448 e4m3) and every code is the NEAREST representable value to x / s, ties to even.  fp32's x / s cannot decide that by
// itself: it rounds quotients beside the middle between two codes onto it (with bf16 inputs x = a / 2 that happens in
// every few rows).  The quotient is therefore rounded to ODD: truncated, its last bit set when the residual
// x - q s is not zero (one fma gives the residual's exact sign).  Rounding that 24-bit value once more to 8 bits or fewer is
// then the rounding of the exact quotient.
//
// Bound: memory.  A thread owns VEC consecutive values; the L lanes of a group find its maximum with L-lane shuffles, so a
// value is read once and lives in registers until its code is stored.
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
  char* values; long long vrow, vhead;          // bytes
  unsigned char* codes; long long crow;         // bytes per row; a head holds dim * bits / 8
  float* scales; long long srow;                // floats per row
  const int* owner;        // write: row -> last i that writes it (NULL: the rows are distinct)
  unsigned n;              // rows of this launch
  int heads, dim, group, chunks;                // chunks = group / VEC
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
};

// x / s rounded to odd, sign carried; s > 0, xs = x * f and ss = s * f with the power of two f that keeps the residual normal
__device__ __forceinline__ float quotient_odd(float xs, float ss, float inv) {
  const float ax = fabsf(xs);
  const float q0 = ax * inv;
  const float q = fmaf(fmaf(-q0, ss, ax), inv, q0);      // within one unit of the last place of the exact quotient
  const float e = fmaf(-q, ss, ax);                      // its exact remainder's sign
  unsigned b = __float_as_uint(q);
  b -= (e < 0.f) ? 1u : 0u;
  b |= (e != 0.f) ? 1u : 0u;
  return copysignf(__uint_as_float(b), xs);
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
    constexpr int B = Code<FMT>::bits, PER = (BYTES >= 4 ? 32 : BYTES * 8) / B;      // codes per stored word
#pragma unroll
    for (int k = 0; k < VEC / PER; ++k) {
      unsigned w = 0;
#pragma unroll
      for (int j = 0; j < PER; ++j) w |= ((unsigned)(int)rintf(q[k * PER + j]) & ((1u << B) - 1u)) << (B * j);
      r.w[k] = w;
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

// the group's place: row i, its row id, head, offset of the group inside the head
struct Place { long long i, row; int head, g; };
__device__ __forceinline__ Place place_of(const RowsArgs& a, unsigned unit) {
  Place p;
  const unsigned i = fast_div(unit, a.groups_per_row);
  const unsigned u = unit - i * a.groups_per_row.d;
  p.head = (int)fast_div(u, a.groups_per_head);
  p.g = (int)(u - (unsigned)p.head * a.groups_per_head.d);
  p.i = a.i0 + i;
  p.row = row_of(a, p.i);
  return p;
}

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
template <int FMT, int DT, int VEC, int ITERS>
__global__ __launch_bounds__(256) void k_rows_write(RowsArgs a) {
  const unsigned long long t = (unsigned long long)blockIdx.x * 256 + threadIdx.x;
  const unsigned long long unit64 = t >> a.lanes_log2;
  // whole wavefronts stay for the shuffles; a group's lanes are in range together
  const bool in = unit64 < (unsigned long long)a.n * a.groups_per_row.d;
  const Place p = in ? place_of(a, (unsigned)unit64) : Place{0, -1, 0, 0};
  const int L = 1 << a.lanes_log2, lane = (int)(t & (unsigned)(L - 1));
  const bool live = p.row >= 0 && !(a.owner && a.owner[p.row] != (int)p.i);
  float x[ITERS][VEC];
  float top = 0.f;
  bool bad = false;
  if (live) {
    const char* v = a.values + p.i * a.vrow + p.head * a.vhead + (long long)p.g * a.group * Elem<DT>::bytes;
#pragma unroll
    for (int it = 0; it < ITERS; ++it) {
      const int c = lane + it * L;
      if (c < a.chunks) {
        load_values<DT, VEC>(v + (long long)c * VEC * Elem<DT>::bytes, x[it]);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const float m = fabsf(x[it][k]);
          bad |= !(m < __builtin_inff());
          top = fmaxf(top, m);
        }
      }
    }
  }
  // an infinite or NaN value makes the whole group NaN: it is not hidden, and nothing finite is made of it
  if (bad) top = __builtin_inff();
  for (int o = L >> 1; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  if (!live) return;
  const bool finite = top < __builtin_inff();
  const float s = finite ? top / Code<FMT>::top : __builtin_nanf("");
  const float f = top < 8.6736174e-19f /* 2^-60 */ ? 1.2089258e24f /* 2^80 */ : 1.f;
  const float ss = s * f, inv = 1.f / ss;
  const long long row = p.row;
  unsigned char* cd = a.codes + row * a.crow + ((long long)p.head * a.dim + (long long)p.g * a.group) * Code<FMT>::bits / 8;
#pragma unroll
  for (int it = 0; it < ITERS; ++it) {
    const int c = lane + it * L;
    if (c < a.chunks) {
      float q[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        // a scale in the denormals is coarse: the quotient may pass the largest code
        const float y = fminf(fmaxf(quotient_odd(x[it][k] * f, ss, inv), -Code<FMT>::top), Code<FMT>::top);
        q[k] = s > 0.f ? y : 0.f;
      }
      encode<FMT, VEC>(q, cd + (long long)c * VEC * Code<FMT>::bits / 8);
    }
  }
  if (lane == 0) a.scales[row * a.srow + (long long)p.head * a.groups_per_head.d + p.g] = s;
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
    const float s = a.scales[p.row * a.srow + (long long)p.head * a.groups_per_head.d + p.g];
    decode<FMT, VEC>(a.codes + p.row * a.crow + ((long long)p.head * a.dim + (long long)p.g * a.group + (long long)c * VEC) * Code<FMT>::bits / 8, y);
#pragma unroll
    for (int k = 0; k < VEC; ++k) y[k] *= s;
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k) y[k] = 0.f;
  }
  store_values<DT, VEC>(a.values + p.i * a.vrow + p.head * a.vhead + ((long long)p.g * a.group + (long long)c * VEC) * Elem<DT>::bytes, y);
}

// chunks of a group that one lane holds at most: 64 lanes x 8 x VEC >= 1024 from pairs on, single elements need 16
constexpr int max_iters(int vec) { return vec == 1 ? 16 : 8; }
template <int FMT, int DT, int VEC> static void launch_write(const RowsArgs& a, unsigned grid, hipStream_t s) {
  const int iters = (a.chunks + (1 << a.lanes_log2) - 1) >> a.lanes_log2;
  if (iters == 1) hipLaunchKernelGGL((k_rows_write<FMT, DT, VEC, 1>), dim3(grid), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((k_rows_write<FMT, DT, VEC, max_iters(VEC)>), dim3(grid), dim3(256), 0, s, a);
}
template <int FMT, int DT, int VEC> static void launch_read(const RowsArgs& a, hipStream_t s) {
  const unsigned total = a.n * a.groups_per_row.d * (unsigned)a.chunks;
  hipLaunchKernelGGL((k_rows_read<FMT, DT, VEC>), dim3((total + 255) / 256), dim3(256), 0, s, a, make_fastdiv((unsigned)a.chunks), total);
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
  if (q->n < 0 || q->n > (1ll << 40) || q->capacity < 0 || q->capacity > (1ll << 40)) PSL_BAD("%s: n %lld, capacity %lld", who, (long long)q->n, (long long)q->capacity);
  if (q->n == 0) return PSL_OK;
  if (!q->values || !q->codes || !q->scales) PSL_BAD("%s: missing pointer", who);
  if (q->rows ? (q->rows_bits != 32 && q->rows_bits != 64) : (q->first < 0 || q->first > q->capacity || q->n > q->capacity - q->first))
    PSL_BAD("%s: rows [%lld, +%lld) of %lld (rows_bits %d)", who, (long long)q->first, (long long)q->n, (long long)q->capacity, q->rows_bits);
  const long long hd = (long long)q->heads * q->dim;
  const long long big = 1ll << 40;
  if (q->value_row_stride < 0 || q->value_head_stride < 0 || q->value_row_stride > big || q->value_head_stride > big || q->codes_row_stride > big || q->scales_row_stride > big ||
      q->codes_row_stride < hd * bits / 8 || q->scales_row_stride < hd / q->group)
    PSL_BAD("%s: bad stride", who);
  if (!write && ((q->heads > 1 && q->value_head_stride < q->dim) || (q->n > 1 && q->value_row_stride < (q->heads - 1) * q->value_head_stride + q->dim)))
    PSL_BAD("%s: rows of the output overlap", who);
  const uintptr_t pv = (uintptr_t)q->values, pc = (uintptr_t)q->codes, ps = (uintptr_t)q->scales;
  if (pv % es || ps % 4 || (q->rows && (uintptr_t)q->rows % (q->rows_bits / 8))) PSL_BAD("%s: misaligned pointer", who);
  if (write && q->rows && q->owner && q->n > 0x7fffffffll) PSL_BAD("%s: %lld rows in one call with an owner table (2^31 - 1 at most)", who, (long long)q->n);
  // VEC: the widest piece that divides a group and that every address keeps aligned (16-byte loads of values, code words of
  // VEC * bits / 8 bytes).  fp32 rows of 32: 8 beats 1 by 6x (54 000 rows).
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
  a.values = (char*)q->values; a.vrow = q->value_row_stride * es; a.vhead = q->value_head_stride * es;
  a.codes = (unsigned char*)q->codes; a.crow = q->codes_row_stride; a.scales = q->scales; a.srow = q->scales_row_stride;
  a.owner = write && q->rows ? q->owner : nullptr;
  a.heads = q->heads; a.dim = q->dim; a.group = q->group; a.chunks = q->group / vec;
  a.groups_per_row = make_fastdiv((unsigned)(hd / q->group)); a.groups_per_head = make_fastdiv((unsigned)(q->dim / q->group));
  // Lanes of a group: the largest power of two that divides its chunks leaves no lane idle (a group of 80 = ten chunks on
  // two lanes); where that would leave more than eight chunks to a lane, the next power of two above, some lanes idle.
  int l = 0;
  while (l < 6 && (a.chunks >> l) % 2 == 0) ++l;
  if ((a.chunks >> l) > 8) { l = 0; while (l < 6 && (1 << l) < a.chunks) ++l; }
  a.lanes_log2 = l;
  if (a.owner) {
    a.i0 = 0; a.n = (unsigned)q->n;
    const unsigned grid = (unsigned)((q->n + 255) / 256);
    hipLaunchKernelGGL(k_rows_owner_clear, dim3(grid), dim3(256), 0, s, a, q->owner);
    hipLaunchKernelGGL(k_rows_owner_claim, dim3(grid), dim3(256), 0, s, a, q->owner);
  }
  // launches of fewer than 2^30 threads: the 32-bit divisions above stay exact
  const long long per_row = (hd / q->group) * ((long long)a.chunks > (1 << l) ? a.chunks : (1 << l));
  const long long step = (1ll << 30) / per_row;
  for (long long i0 = 0; i0 < q->n; i0 += step) {
    a.i0 = i0; a.n = (unsigned)(q->n - i0 < step ? q->n - i0 : step);
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
