// Root-mean-square norm along the channels of NHWC pixels (rows), with the residual's addition in front of it and an optional
// 8-bit output behind it, gfx950.  The per-sample norm of the reference's blocks (norm.hip) has one scalar gain and statistics over
// (C,H,W); here every row (pixel) has its own scale and every channel its own gain:
//   h = rnd_T(x + r),  s = 1 / sqrt(mean_c h^2 + eps),  y = h s gamma
//   backward:  xh = h s,  w = dy gamma:  dx = dr = s (w - xh mean_c(w xh)) + dh,   dgamma = sum_rows dy xh
// where dh is the gradient that reaches h past the norm (the residual stream).  Statistics and a lane's sums are fp32, the joins of
// dgamma's sums fp64; the only roundings to fewer bits are the stores: T (fp32 or bf16) and e4m3.
// Both passes are HBM-bound (6 / 12 flops per element).  A row lives in the registers of a group of LPR lanes (the smallest
// power of two that covers it in one 16-byte chunk per lane, then several chunks per lane of a whole wave): ONE read of every input,
// statistics by lane exchanges, no LDS and no barrier.  16-byte accesses at any element alignment (gfx950 global memory takes
// them); the last chunk of a row whose length is no multiple of 8 (bf16) / 4 (fp32) goes element by element.  Rows longer than the
// registers hold take a workgroup each and read their inputs twice.
#include "common.h"

namespace pg {

typedef unsigned short bf16_t;

__device__ __forceinline__ unsigned rms_pack_bf16(float lo, float hi) {
  unsigned r;
  asm("v_cvt_pk_bf16_f32 %0, %1, %2" : "=v"(r) : "v"(lo), "v"(hi));
  return r;
}
__device__ __forceinline__ float rms_ld1(const float* p) { return *p; }
__device__ __forceinline__ float rms_ld1(const bf16_t* p) { return __uint_as_float((unsigned)*p << 16); }
__device__ __forceinline__ void rms_st1(float* p, float v) { *p = v; }
__device__ __forceinline__ void rms_st1(bf16_t* p, float v) { *p = (bf16_t)(rms_pack_bf16(v, 0.f) & 0xffffu); }
__device__ __forceinline__ float rms_round(float v, const float*) { return v; }
__device__ __forceinline__ float rms_round(float v, const bf16_t*) { return __uint_as_float(rms_pack_bf16(v, 0.f) << 16); }

struct __attribute__((packed, aligned(2))) RmsU4 { unsigned x, y, z, w; };     // 16, 8, 4 bytes at the alignment of one element
struct __attribute__((packed, aligned(2))) RmsU2 { unsigned x, y; };
struct __attribute__((packed, aligned(2))) RmsU1 { unsigned x; };
struct __attribute__((packed, aligned(4))) RmsF4 { float x, y, z, w; };
struct __attribute__((packed, aligned(4))) RmsF2 { float x, y; };
struct __attribute__((packed, aligned(1))) RmsB8 { unsigned x, y; };
struct __attribute__((packed, aligned(1))) RmsB4 { unsigned x; };
struct __attribute__((packed, aligned(1))) RmsB2 { unsigned short x; };

template <typename T> struct RmsV { static constexpr int N = 16 / (int)sizeof(T); };

// A chunk that crosses the row's end is read from the row's last V elements instead and moved down by d = V - C % V places, so that every
// load is one unconditional instruction (loads under a branch of their own were waited for one by one).  d is the same for all lanes.
__device__ __forceinline__ void rms_down(unsigned (&w)[4], int d, const bf16_t*) {
  if (d & 4) { w[0] = w[2]; w[1] = w[3]; w[2] = w[3] = 0u; }
  if (d & 2) { w[0] = w[1]; w[1] = w[2]; w[2] = w[3]; w[3] = 0u; }
  if (d & 1) {
#pragma unroll
    for (int k = 0; k < 3; ++k) w[k] = (w[k] >> 16) | (w[k + 1] << 16);
    w[3] >>= 16;
  }
}
__device__ __forceinline__ void rms_down(unsigned (&w)[4], int d, const float*) {
  if (d & 2) { w[0] = w[2]; w[1] = w[3]; w[2] = w[3] = 0u; }
  if (d & 1) { w[0] = w[1]; w[1] = w[2]; w[2] = w[3]; w[3] = 0u; }
}
__device__ __forceinline__ void rms_put_tail(bf16_t* q, int n, const unsigned (&w)[4]) {
  if (n & 4) { RmsU2 u; u.x = w[0]; u.y = w[1]; *reinterpret_cast<RmsU2*>(q) = u; }
  if (n & 2) reinterpret_cast<RmsU1*>(q + (n & 4))->x = (n & 4) ? w[2] : w[0];
  if (n & 1) {
    unsigned u = w[0];
#pragma unroll
    for (int k = 1; k < 4; ++k)
      if (k == (n >> 1)) u = w[k];
    q[n & 6] = (bf16_t)u;
  }
}
__device__ __forceinline__ void rms_put_tail(float* q, int n, const unsigned (&w)[4]) {
  if (n & 2) { RmsF2 u; u.x = __uint_as_float(w[0]); u.y = __uint_as_float(w[1]); *reinterpret_cast<RmsF2*>(q) = u; }
  if (n & 1) q[n & 2] = __uint_as_float((n & 2) ? w[2] : w[0]);
}
// the chunk of RmsV<T>::N elements that starts at column c (a multiple of it) of a row of C elements; zero behind the row's end
// `ex` (a constant at every call): the chunk is known to be full
template <typename T>
__device__ __forceinline__ void rms_load(bool ex, const T* row, int c, int C, float (&v)[RmsV<T>::N]) {
  constexpr int V = RmsV<T>::N;
  if (!ex && C < V) {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (c + e < C) ? rms_ld1(row + c + e) : 0.f;
    return;
  }
  const RmsU4 u = *reinterpret_cast<const RmsU4*>(row + (ex ? c : min(c, C - V)));
  unsigned w[4] = {u.x, u.y, u.z, u.w};
  if (!ex && (C & (V - 1))) {
    unsigned t[4] = {u.x, u.y, u.z, u.w};
    rms_down(t, V - (C & (V - 1)), row);
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = c + V > C ? t[e] : w[e];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (!ex) w[e] = c < C ? w[e] : 0u;
    if constexpr (V == 4) v[e] = __uint_as_float(w[e]);
    else { v[2 * e] = __uint_as_float(w[e] << 16); v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u); }
  }
}
template <typename T>
__device__ __forceinline__ void rms_store(bool ex, T* row, int c, int C, const float (&v)[RmsV<T>::N]) {
  constexpr int V = RmsV<T>::N;
  if (!ex && c >= C) return;
  unsigned w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (V == 4) w[e] = __float_as_uint(v[e]);
    else w[e] = rms_pack_bf16(v[2 * e], v[2 * e + 1]);
  }
  if (ex || c + V <= C) {
    RmsU4 u;
    u.x = w[0]; u.y = w[1]; u.z = w[2]; u.w = w[3];
    *reinterpret_cast<RmsU4*>(row + c) = u;
  } else {
    rms_put_tail(row + c, C & (V - 1), w);
  }
}
template <int V>
__device__ __forceinline__ void rms_gain(bool ex, const float* g, int c, int C, float (&v)[V]) {
  if (!ex && C < V) {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (c + e < C) ? g[c + e] : 0.f;
    return;
  }
  const float* q = g + (ex ? c : min(c, C - V));
#pragma unroll
  for (int k = 0; k < V / 4; ++k) {
    const RmsF4 f = *reinterpret_cast<const RmsF4*>(q + 4 * k);
    v[4 * k] = f.x; v[4 * k + 1] = f.y; v[4 * k + 2] = f.z; v[4 * k + 3] = f.w;
  }
  if (!ex && (C & (V - 1))) {
    const int d = V - (C & (V - 1));
    float t[V];
#pragma unroll
    for (int e = 0; e < V; ++e) t[e] = v[e];
#pragma unroll
    for (int b = V / 2; b > 0; b >>= 1)
      if (d & b) {
#pragma unroll
        for (int e = 0; e < V; ++e) t[e] = e + b < V ? t[e + b] : 0.f;
      }
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = c + V > C ? t[e] : v[e];
  }
#pragma unroll
  for (int e = 0; e < V; ++e)
    if (!ex) v[e] = c < C ? v[e] : 0.f;
}
template <int LPR>
__device__ __forceinline__ float group_sum(float v, int lpr = LPR) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// 8 bits: q = e4m3(448 z / max|z|), z = h gamma of a group, in fp64 and rounded to fp32 once: the row's s cancels, and a
// value next to a border of e4m3's steps goes to the side that the definition gives (in fp32, with y and the scale rounded first,
// one value in 500 000 changed sides).  scale = s max|z| / 448; where that is zero (a group of zeros, or s is: the row holds an infinity, or its
// squares pass fp32) y is zero: scale 1, q zeros.  s joins in so that a row whose statistic is NaN is NaN.
struct Q8 {
  double r;
  float scale;
  __device__ __forceinline__ Q8(double am, float s) {
    r = 448.0 / am;
    scale = (float)((double)s * am / 448.0);
    if (am == 0.0 || scale == 0.f) { r = 0.0; scale = 1.f; }      // (without eps s is infinite where am is zero)
    if (s != s) { r = (double)s; scale = s; }
  }
};
// round to nearest even; |t| <= 448 up to the rounding of the quotient, which the comparison takes off; NaN stays NaN
__device__ __forceinline__ float q8_clip(float t) { return t > 448.f ? 448.f : (t < -448.f ? -448.f : t); }
template <int V>
__device__ __forceinline__ void q8_store(bool ex, uint8_t* row, int c, int C, const float (&h)[V], const float (&g)[V], const Q8& k) {
  unsigned w[V / 4];
  float t[V];
#pragma unroll
  for (int e = 0; e < V; ++e) t[e] = q8_clip((float)((double)h[e] * (double)g[e] * k.r));
#pragma unroll
  for (int q = 0; q < V / 4; ++q) {
    int p = 0;
    p = __builtin_amdgcn_cvt_pk_fp8_f32(t[4 * q], t[4 * q + 1], p, false);
    p = __builtin_amdgcn_cvt_pk_fp8_f32(t[4 * q + 2], t[4 * q + 3], p, true);
    w[q] = (unsigned)p;
  }
  if (ex || c + V <= C) {
    if constexpr (V == 8) { RmsB8 b; b.x = w[0]; b.y = w[1]; *reinterpret_cast<RmsB8*>(row + c) = b; }
    else { RmsB4 b; b.x = w[0]; *reinterpret_cast<RmsB4*>(row + c) = b; }
  } else if (c < C) {
    const int n = C & (V - 1);
    uint8_t* q = row + c;
    unsigned u = w[0];
    if (V == 8 && (n & 4)) { RmsB4 b; b.x = w[0]; *reinterpret_cast<RmsB4*>(q) = b; q += 4; u = w[V / 4 - 1]; }
    if (n & 2) { RmsB2 b; b.x = (unsigned short)u; *reinterpret_cast<RmsB2*>(q) = b; q += 2; u >>= 16; }
    if (n & 1) *q = (uint8_t)u;
  }
}
template <int V>
__device__ __forceinline__ double abs_max(const float (&h)[V], const float (&g)[V]) {
  double m = 0.0;
#pragma unroll
  for (int e = 0; e < V; ++e) m = fmax(m, fabs((double)h[e] * (double)g[e]));
  return m;
}

struct RmsFwdK {
  const void* x; const void* res; const float* gamma;
  long rows; int C; long ldx, ldr, ldy; float eps;
  void* h; void* y; uint8_t* q; float* scales; int group, ngroups; float* rstd;
};

// HBM-bound: 524288 x 128 bf16 with residual and e4m3 output 92 us (5.1 TB/s), 16384 x 256 fp32 with residual 11.5 us (5.9 TB/s, the last-level cache
// holds part of it), 131072 x 513 bf16 out of rows of 1026 71 us (3.8 TB/s: rows begin inside cache lines); one row 2.5 us.
// Q: an 8-bit output too, with one scale per row (group 0) or per `group` channels (group / V a power of two <= LPR: host)
template <typename T, int LPR, int NCH, bool Q, bool EX>
__global__ __launch_bounds__(256) void rms_fwd_kernel(const RmsFwdK p) {
  constexpr int V = RmsV<T>::N;
  const long row = (long)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  if (row >= p.rows) return;
  const int ln = threadIdx.x % LPR;
  const T* x = reinterpret_cast<const T*>(p.x) + row * p.ldx;
  float h[NCH][V];
#pragma unroll
  for (int i = 0; i < NCH; ++i) rms_load(EX || i < NCH - 1, x, (i * LPR + ln) * V, p.C, h[i]);
  if (p.res) {
    const T* r = reinterpret_cast<const T*>(p.res) + row * p.ldr;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      float t[V];
      rms_load(EX || i < NCH - 1, r, (i * LPR + ln) * V, p.C, t);
#pragma unroll
      for (int e = 0; e < V; ++e) h[i][e] = rms_round(h[i][e] + t[e], x);
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < NCH; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) ss = fmaf(h[i][e], h[i][e], ss);
  ss = group_sum<LPR>(ss);
  const float s = 1.f / sqrtf(ss / (float)p.C + p.eps);
  if (p.h) {
#pragma unroll
    for (int i = 0; i < NCH; ++i) rms_store(EX || i < NCH - 1, reinterpret_cast<T*>(p.h) + row * p.C, (i * LPR + ln) * V, p.C, h[i]);
  }
  if (p.rstd && ln == 0) p.rstd[row] = s;
  float g[NCH][V];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    rms_gain<V>(EX || i < NCH - 1, p.gamma, (i * LPR + ln) * V, p.C, g[i]);
    if (p.y) {
      float y[V];
#pragma unroll
      for (int e = 0; e < V; ++e) y[e] = h[i][e] * s * g[i][e];
      rms_store(EX || i < NCH - 1, reinterpret_cast<T*>(p.y) + row * p.ldy, (i * LPR + ln) * V, p.C, y);
    }
  }
  if constexpr (Q) {
    double am[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) am[i] = abs_max<V>(h[i], g[i]);
    if (p.group == 0) {
#pragma unroll
      for (int i = 1; i < NCH; ++i) am[0] = fmax(am[0], am[i]);
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) am[0] = fmax(am[0], __shfl_xor(am[0], o, 64));
      const Q8 k(am[0], s);
      if (ln == 0) p.scales[row] = k.scale;
#pragma unroll
      for (int i = 0; i < NCH; ++i) q8_store<V>(EX || i < NCH - 1, p.q + row * p.C, (i * LPR + ln) * V, p.C, h[i], g[i], k);
    } else {
      const int gl = p.group / V;                       // lanes of a group
      for (int o = gl >> 1; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < NCH; ++i) am[i] = fmax(am[i], __shfl_xor(am[i], o, 64));
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const int c = (i * LPR + ln) * V;
        const Q8 k(am[i], s);
        if ((ln & (gl - 1)) == 0 && c < p.C) p.scales[row * p.ngroups + c / p.group] = k.scale;
        q8_store<V>(EX || i < NCH - 1, p.q + row * p.C, c, p.C, h[i], g[i], k);
      }
    }
  }
}

// rows that do not fit a wave's registers: a workgroup per row, inputs read twice
__device__ __forceinline__ double block_sum_d(double v, double* red) {
  v = wave_sum_d(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
}
__device__ __forceinline__ double block_max_d(double v, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmax(v, __shfl_xor(v, o, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return fmax(fmax(red[0], red[1]), fmax(red[2], red[3]));
}
template <typename T>
__device__ __forceinline__ void rms_sum_chunk(const T* x, const T* r, int c, int C, float (&h)[RmsV<T>::N]) {
  rms_load(false, x, c, C, h);
  if (r) {
    float t[RmsV<T>::N];
    rms_load(false, r, c, C, t);
#pragma unroll
    for (int e = 0; e < RmsV<T>::N; ++e) h[e] = rms_round(h[e] + t[e], x);
  }
}
template <typename T, bool Q>
__global__ __launch_bounds__(256) void rms_fwd_long_kernel(const RmsFwdK p) {
  constexpr int V = RmsV<T>::N;
  __shared__ double red[4];
  const long row = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(p.x) + row * p.ldx;
  const T* r = p.res ? reinterpret_cast<const T*>(p.res) + row * p.ldr : nullptr;
  double ss = 0.0;
  for (long c = (long)threadIdx.x * V; c < p.C; c += 256 * V) {
    float h[V];
    rms_sum_chunk(x, r, (int)c, p.C, h);
    float a = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) a = fmaf(h[e], h[e], a);
    ss += (double)a;
  }
  const float s = (float)(1.0 / sqrt(block_sum_d(ss, red) / (double)p.C + (double)p.eps));
  if (p.rstd && threadIdx.x == 0) p.rstd[row] = s;
  double am = 0.0;
  for (long c = (long)threadIdx.x * V; c < p.C; c += 256 * V) {
    float h[V], g[V];
    rms_sum_chunk(x, r, (int)c, p.C, h);
    if (p.h) rms_store(false, reinterpret_cast<T*>(p.h) + row * p.C, (int)c, p.C, h);
    rms_gain<V>(false, p.gamma, (int)c, p.C, g);
    if (Q && p.group == 0) am = fmax(am, abs_max<V>(h, g));
#pragma unroll
    for (int e = 0; e < V; ++e) h[e] = h[e] * s * g[e];
    if (p.y) rms_store(false, reinterpret_cast<T*>(p.y) + row * p.ldy, (int)c, p.C, h);
  }
  if constexpr (Q) {
    if (Q && p.group == 0) {
      am = block_max_d(am, red);
      if (threadIdx.x == 0) p.scales[row] = Q8(am, s).scale;
    }
    // groups: the chunks of a group belong to consecutive lanes of one wave; every lane of a wave makes every trip
    const long trips = ((long)p.C + 256 * V - 1) / (256 * V);
    for (long t = 0; t < trips; ++t) {
      const long cl = (t * 256 + threadIdx.x) * V;
      const int c = cl < p.C ? (int)cl : p.C;
      float h[V], g[V];
      rms_sum_chunk(x, r, c, p.C, h);
      rms_gain<V>(false, p.gamma, c, p.C, g);
      if (p.group) {
        am = abs_max<V>(h, g);
        const int gl = p.group / V;
        for (int o = gl >> 1; o > 0; o >>= 1) am = fmax(am, __shfl_xor(am, o, 64));
        if ((threadIdx.x & (gl - 1)) == 0 && c < p.C) p.scales[row * p.ngroups + c / p.group] = Q8(am, s).scale;
      }
      if (c < p.C) q8_store<V>(false, p.q + row * p.C, c, p.C, h, g, Q8(am, s));
    }
  }
}

struct RmsBwdK {
  const void* dy; const void* dh; const void* h; const float* rstd; const float* gamma;
  long rows; int C; long lddy, ldh;
  void* dx; float* part; float* dgamma; int accumulate;
};

// A group of LPR lanes walks rows; every lane keeps the dgamma sums of its own columns in registers, the workgroup's groups are
// joined in LDS, the workgroups by rms_dgamma_kernel (one workgroup: written here).  No atomics: the order is fixed.  HBM-bound: 131072 x
// 512 bf16 with dh 98 us + 4 us for the join (5.3 TB/s); at most 1024 workgroups, so that few partial rows are left.  WG: 256 lanes, or 1024
// for the few rows that one workgroup handles by itself (77 x 189 fp32: 9 us; a second launch costs more than the rows, and several rows of a
// group at a time are slower).
template <typename T, int LPR, int NCH, int WG, bool EX>
__global__ __launch_bounds__(WG) void rms_bwd_kernel(const RmsBwdK p) {
  constexpr int V = RmsV<T>::N, G = WG / LPR;
  __shared__ float red[WG * NCH * V];
  const int ln = threadIdx.x % LPR, grp = threadIdx.x / LPR;
  float acc[NCH][V], gain[NCH][V];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    rms_gain<V>(EX || i < NCH - 1, p.gamma, (i * LPR + ln) * V, p.C, gain[i]);
#pragma unroll
    for (int e = 0; e < V; ++e) acc[i][e] = 0.f;
  }
  for (long row = (long)blockIdx.x * G + grp; row < p.rows; row += (long)gridDim.x * G) {
    const T* dy = reinterpret_cast<const T*>(p.dy) + row * p.lddy;
    const T* h = reinterpret_cast<const T*>(p.h) + row * p.ldh;
    float a[NCH][V], b[NCH][V], d[NCH][V];
#pragma unroll
    for (int i = 0; i < NCH; ++i) { rms_load(EX || i < NCH - 1, dy, (i * LPR + ln) * V, p.C, a[i]); rms_load(EX || i < NCH - 1, h, (i * LPR + ln) * V, p.C, b[i]); }
    if (p.dh) {
#pragma unroll
      for (int i = 0; i < NCH; ++i) rms_load(EX || i < NCH - 1, reinterpret_cast<const T*>(p.dh) + row * p.C, (i * LPR + ln) * V, p.C, d[i]);
    } else {
#pragma unroll
      for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) d[i][e] = 0.f;
    }
    const float s = p.rstd[row];
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        b[i][e] *= s;                                        // xh
        acc[i][e] = fmaf(a[i][e], b[i][e], acc[i][e]);
        a[i][e] *= gain[i][e];                               // w
        dot = fmaf(a[i][e], b[i][e], dot);
      }
    dot = group_sum<LPR>(dot) / (float)p.C;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
#pragma unroll
      for (int e = 0; e < V; ++e) a[i][e] = (a[i][e] - b[i][e] * dot) * s + d[i][e];
      rms_store(EX || i < NCH - 1, reinterpret_cast<T*>(p.dx) + row * p.C, (i * LPR + ln) * V, p.C, a[i]);
    }
  }
  // red[group][column]
#pragma unroll
  for (int i = 0; i < NCH; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) red[(grp * NCH + i) * LPR * V + ln * V + e] = acc[i][e];
  __syncthreads();
  for (int c = threadIdx.x; c < p.C; c += WG) {
    double t = 0.0;
    for (int k = 0; k < G; ++k) t += (double)red[k * NCH * LPR * V + c];
    if (gridDim.x == 1) p.dgamma[c] = (float)(p.accumulate ? (double)p.dgamma[c] + t : t);
    else p.part[(long)blockIdx.x * p.C + c] = (float)t;
  }
}

// dgamma[c] = sum of nblk partial rows, ld apart: 32 columns x 32 slices per workgroup, fp64
__global__ __launch_bounds__(1024) void rms_dgamma_kernel(const float* part, int nblk, int ld, int C, float* dgamma, int accumulate) {
  __shared__ double red[32][33];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), sl = threadIdx.x >> 5;
  double t = 0.0;
  if (c < C) {
#pragma unroll 8
    for (int k = sl; k < nblk; k += 32) t += (double)part[(long)k * ld + c];
  }
  red[sl][threadIdx.x & 31] = t;
  __syncthreads();
  if (threadIdx.x < 32 && c < C) {
    double a = 0.0;
    for (int k = 0; k < 32; ++k) a += red[k][threadIdx.x];
    dgamma[c] = (float)(accumulate ? (double)dgamma[c] + a : a);
  }
}

// long rows: dx by a workgroup per row ...
template <typename T>
__global__ __launch_bounds__(256) void rms_bwd_long_kernel(const RmsBwdK p) {
  constexpr int V = RmsV<T>::N;
  __shared__ double red[4];
  const long row = blockIdx.x;
  const T* dy = reinterpret_cast<const T*>(p.dy) + row * p.lddy;
  const T* h = reinterpret_cast<const T*>(p.h) + row * p.ldh;
  const T* dh = p.dh ? reinterpret_cast<const T*>(p.dh) + row * p.C : nullptr;
  const float s = p.rstd[row];
  double dot = 0.0;
  for (long c = (long)threadIdx.x * V; c < p.C; c += 256 * V) {
    float a[V], b[V], g[V], t = 0.f;
    rms_load(false, dy, (int)c, p.C, a); rms_load(false, h, (int)c, p.C, b);
    rms_gain<V>(false, p.gamma, (int)c, p.C, g);
#pragma unroll
    for (int e = 0; e < V; ++e) t = fmaf(a[e] * g[e], b[e] * s, t);
    dot += (double)t;
  }
  const float m = (float)(block_sum_d(dot, red) / (double)p.C);
  for (long c = (long)threadIdx.x * V; c < p.C; c += 256 * V) {
    float a[V], b[V], g[V], d[V];
    rms_load(false, dy, (int)c, p.C, a); rms_load(false, h, (int)c, p.C, b);
    rms_gain<V>(false, p.gamma, (int)c, p.C, g);
    if (dh) rms_load(false, dh, (int)c, p.C, d);
    else {
#pragma unroll
      for (int e = 0; e < V; ++e) d[e] = 0.f;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) a[e] = (a[e] * g[e] - b[e] * s * m) * s + d[e];
    rms_store(false, reinterpret_cast<T*>(p.dx) + row * p.C, (int)c, p.C, a);
  }
}
// ... and dgamma's partial sums by column strips (256 columns) x row ranges
template <typename T>
__global__ __launch_bounds__(256) void rms_dgamma_long_kernel(const RmsBwdK p) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= p.C) return;
  const T* dy = reinterpret_cast<const T*>(p.dy) + c;
  const T* h = reinterpret_cast<const T*>(p.h) + c;
  double t = 0.0;
  for (long row = blockIdx.y; row < p.rows; row += gridDim.y)
    t += (double)(rms_ld1(dy + row * p.lddy) * (rms_ld1(h + row * p.ldh) * p.rstd[row]));
  p.part[(long)blockIdx.y * p.C + c] = (float)t;
}

// lanes and chunks per lane that hold a row of C elements (V per chunk), nch = 0: it takes the long-row form; all chunks of a lane but the
// last are full.  Rows that fill a power of two of lanes to the last element take one chunk per lane, or several with 64 lanes
// (`ex`: no masks at all).  Others: few rows, and the bf16 backward pass, which keeps most registers, the fewest chunks; otherwise what
// fills the lanes of a wave best, several rows to a wave (300 bf16 channels: 172 -> 116 us per 63 M elements).
// A group of the 8-bit output must lie within one turn of the lanes.
struct RmsShape { int lpr, nch; bool ex; };
static RmsShape rms_shape(long rows, int C, int V, int group, bool bwd) {
  for (int l = 8; l <= 64; l *= 2)
    if (l * V == C) return {l, 1, true};
  for (int n = 2; n * V <= 32; ++n)
    if (64 * V * n == C) return {64, n, true};
  static const int shapes[][2] = {{8, 1}, {8, 2}, {8, 3}, {16, 1}, {16, 2}, {16, 3}, {32, 1}, {32, 2}, {32, 3}, {64, 1}, {64, 2}, {64, 3}, {64, 4}, {64, 5},
                                  {64, 6}, {64, 7}, {64, 8}};
  RmsShape best = {64, 0, false};
  float cost = 1e30f;
  for (const auto& q : shapes) {
    if (q[0] * q[1] * V < C || q[0] * V < group || q[1] * V > 32) continue;
    if (q[0] * (q[1] - 1) * V >= C) continue;
    const float c = rows <= 2048 || (bwd && V == 8) ? (float)(q[1] * 64 + q[0]) : ((float)q[1] + 1.f) * (float)q[0];
    if (c < cost) { cost = c; best = {q[0], q[1], false}; }
  }
  return best;
}
// at most eight rows per group of a workgroup of 1024 lanes: it writes dgamma itself
static bool rms_bwd_single(long rows, int lpr, int nch) { return nch == 1 && rows <= 8 * (1024 / lpr); }
static long rms_bwd_blocks(long rows, int lpr, int nch) {
  if (rms_bwd_single(rows, lpr, nch)) return 1;
  const long g = 256 / lpr;
  long b = (rows + g - 1) / g;
  // otherwise at least two rows per group, at most 4 workgroups per CU
  b = (b + 1) / 2;
  return b > 1024 ? 1024 : b;
}
static int rms_long_slices(long rows) { return rows < 64 ? (int)rows : 64; }
// the kernels count a row's elements in 32 bits, up to a turn of the lanes behind its end
constexpr int MAX_C = 1 << 30;
// a launch has less than 2^32 lanes: more rows go in several
constexpr long MAX_BLOCKS = 1L << 23;
static void rms_dgamma(const float* part, int nblk, int C, float* dgamma, int accumulate, hipStream_t st) {
  constexpr int PIECE = 1 << 26;                       // 2^21 workgroups of 1024
  for (int c0 = 0; c0 < C; c0 += PIECE) {
    const int n = C - c0 < PIECE ? C - c0 : PIECE;
    PG_KLAUNCH(rms_dgamma_kernel, dim3((n + 31) / 32), dim3(1024), 0, st, part ? part + c0 : nullptr, nblk, C, n, dgamma + c0, accumulate);
  }
}
template <typename P>
static P* rms_at(P* p, long elems, size_t size) {
  return p ? reinterpret_cast<P*>(const_cast<char*>(reinterpret_cast<const char*>(p)) + elems * (long)size) : nullptr;
}

}  // namespace pg

using namespace pg;

extern "C" int pg_rms_norm_fwd(const void* x, const void* res, const float* gamma, int64_t rows, int32_t C, int64_t ldx, int64_t ldr,
                               float eps, int32_t io_flags, void* h, void* y, int64_t ldy, void* q, float* scales, int32_t group,
                               float* rstd, void* stream) {
  PG_REQUIRE(x && gamma && rows >= 0 && C > 0 && C <= MAX_C && ldx >= C && eps >= 0.f,
             "pg_rms_norm_fwd: x, gamma, rows >= 0, 0 < C <= 2^30 and ldx >= C required");
  PG_REQUIRE(io_flags == 0 || io_flags == 3, "pg_rms_norm_fwd: io_flags 0 (fp32) or 3 (bf16)");
  PG_REQUIRE(y || q || h, "pg_rms_norm_fwd: nothing to write (y, q and h are all NULL)");
  PG_REQUIRE(!res || ldr >= C, "pg_rms_norm_fwd: ldr >= C required");
  PG_REQUIRE(!y || ldy >= C, "pg_rms_norm_fwd: ldy >= C required");
  PG_REQUIRE(!q || scales, "pg_rms_norm_fwd: an 8-bit output needs `scales`");
  PG_REQUIRE(!q || group == 0 || group == 32 || group == 64 || group == 128 || group == 256,
             "pg_rms_norm_fwd: group 0 (a scale per row), 32, 64, 128 or 256 channels");
  const size_t em = io_flags ? 1 : 3;
  PG_REQUIRE((((size_t)x | (size_t)res | (size_t)h | (size_t)y) & em) == 0 && (((size_t)gamma | (size_t)scales | (size_t)rstd) & 3) == 0,
             "pg_rms_norm_fwd: a pointer is not aligned to its element");
  if (rows == 0) return 0;
  const int V = io_flags ? 8 : 4;
  const int grp = q && group < C ? group : 0;          // a group that is the whole row
  const RmsShape sh = rms_shape((long)rows, C, V, grp, false);
  const int lpr = sh.lpr, nch = sh.nch;
  const long per = nch ? 256 / lpr : 1;                // rows of a workgroup
  const size_t es = io_flags ? 2 : 4;
  PG_REQUIRE(rows <= (1L << 40), "pg_rms_norm_fwd: too many rows");
  PG_REQUIRE(nch || ((h == nullptr || (h != x && h != res)) && (y == nullptr || (y != x && y != res && y != h))),
             "pg_rms_norm_fwd: rows of more than 2048 channels are read twice: outputs must not be inputs");
  PG_REQUIRE((h == nullptr || ((h != x || ldx == C) && (h != res || ldr == C))) &&
             (y == nullptr || ((y != x || ldy == ldx) && (y != res || ldy == ldr) && (y != h || ldy == C))),
             "pg_rms_norm_fwd: an output in place of an input needs the same row stride");
  const int ngroups = grp ? (C + grp - 1) / grp : 1;
  hipStream_t st = (hipStream_t)stream;
  const dim3 wg(256);
#define PG_RF1(T, L, N, EX)                                                                                        \
  do {                                                                                                             \
    if (q) PG_KLAUNCH((rms_fwd_kernel<T, L, N, true, EX>), grid, wg, 0, st, k);                                    \
    else PG_KLAUNCH((rms_fwd_kernel<T, L, N, false, EX>), grid, wg, 0, st, k);                                     \
  } while (0)
  bool none = false;       // a form that the shape's rule gives no row of this type: an error, should the rule change
#define PG_RF14(T, L, M, EX)                                                                                       \
  do {                                                                                                             \
    if (RmsV<T>::N == 4) PG_RF1(T, L, (RmsV<T>::N == 4 ? M : 1), EX);                                              \
    else none = true;                                                                                              \
  } while (0)
#define PG_RF(T)                                                                                                   \
  do {                                                                                                             \
    switch (lpr * 32 + nch * 2 + (sh.ex ? 1 : 0)) {                                                                \
      case 8 * 32 + 3: PG_RF1(T, 8, 1, true); break;                                                               \
      case 16 * 32 + 3: PG_RF1(T, 16, 1, true); break;                                                             \
      case 32 * 32 + 3: PG_RF1(T, 32, 1, true); break;                                                             \
      case 64 * 32 + 3: PG_RF1(T, 64, 1, true); break;                                                             \
      case 64 * 32 + 5: PG_RF1(T, 64, 2, true); break;                                                             \
      case 64 * 32 + 7: PG_RF1(T, 64, 3, true); break;                                                             \
      case 64 * 32 + 9: PG_RF1(T, 64, 4, true); break;                                                             \
      case 64 * 32 + 11: PG_RF14(T, 64, 5, true); break;                                                           \
      case 64 * 32 + 13: PG_RF14(T, 64, 6, true); break;                                                           \
      case 64 * 32 + 15: PG_RF14(T, 64, 7, true); break;                                                           \
      case 64 * 32 + 17: PG_RF14(T, 64, 8, true); break;                                                           \
      case 8 * 32 + 2: PG_RF1(T, 8, 1, false); break;                                                              \
      case 8 * 32 + 4: PG_RF1(T, 8, 2, false); break;                                                              \
      case 8 * 32 + 6: PG_RF1(T, 8, 3, false); break;                                                              \
      case 16 * 32 + 2: PG_RF1(T, 16, 1, false); break;                                                            \
      case 16 * 32 + 4: PG_RF1(T, 16, 2, false); break;                                                            \
      case 16 * 32 + 6: PG_RF1(T, 16, 3, false); break;                                                            \
      case 32 * 32 + 2: PG_RF1(T, 32, 1, false); break;                                                            \
      case 32 * 32 + 4: PG_RF1(T, 32, 2, false); break;                                                            \
      case 32 * 32 + 6: PG_RF1(T, 32, 3, false); break;                                                            \
      case 64 * 32 + 2: PG_RF1(T, 64, 1, false); break;                                                            \
      case 64 * 32 + 4: PG_RF1(T, 64, 2, false); break;                                                            \
      case 64 * 32 + 6: PG_RF1(T, 64, 3, false); break;                                                            \
      case 64 * 32 + 8: PG_RF1(T, 64, 4, false); break;                                                            \
      case 64 * 32 + 10: PG_RF14(T, 64, 5, false); break;                                                          \
      case 64 * 32 + 12: PG_RF14(T, 64, 6, false); break;                                                          \
      case 64 * 32 + 14: PG_RF14(T, 64, 7, false); break;                                                          \
      case 64 * 32 + 16: PG_RF14(T, 64, 8, false); break;                                                          \
      default:                                                                                                     \
        if (nch) { none = true; break; }                                                                           \
        if (q) PG_KLAUNCH((rms_fwd_long_kernel<T, true>), grid, wg, 0, st, k);                                     \
        else PG_KLAUNCH((rms_fwd_long_kernel<T, false>), grid, wg, 0, st, k);                                      \
        break;                                                                                                     \
    }                                                                                                              \
  } while (0)
  for (long r0 = 0; r0 < rows; r0 += MAX_BLOCKS * per) {
    const long n = rows - r0 < MAX_BLOCKS * per ? rows - r0 : MAX_BLOCKS * per;
    const dim3 grid((unsigned)((n + per - 1) / per));
    const RmsFwdK k = {rms_at(x, r0 * ldx, es), rms_at(res, r0 * ldr, es), gamma, n, C, (long)ldx, (long)ldr, (long)ldy, eps,
                       rms_at(h, r0 * C, es), rms_at(y, r0 * ldy, es), rms_at((uint8_t*)q, r0 * C, 1), rms_at(scales, r0 * ngroups, 4), grp, ngroups,
                       rms_at(rstd, r0, 4)};
    if (io_flags == 0) PG_RF(float);
    else PG_RF(bf16_t);
    PG_REQUIRE(!none, "pg_rms_norm_fwd: no kernel for a row of %d lanes x %d chunks", lpr, nch);
  }
#undef PG_RF
#undef PG_RF14
#undef PG_RF1
  PG_LAUNCH_OK("pg_rms_norm_fwd");
  return 0;
}

extern "C" int64_t pg_rms_norm_bwd_workspace(int64_t rows, int32_t C, int32_t io_flags) {
  if (rows <= 0 || C <= 0) return 0;
  const RmsShape sh = rms_shape((long)rows, C, io_flags ? 8 : 4, 0, true);
  const int lpr = sh.lpr, nch = sh.nch;
  const long nb = nch ? rms_bwd_blocks(rows, lpr, nch) : rms_long_slices(rows);
  return nch && nb == 1 ? 0 : (int64_t)nb * C * 4;
}

extern "C" int pg_rms_norm_bwd(const void* dy, int64_t lddy, const void* dh, const void* h, const float* rstd, const float* gamma,
                               int64_t rows, int32_t C, int32_t io_flags, void* dx, float* dgamma, int32_t accumulate,
                               void* workspace, int64_t workspace_bytes, void* stream) {
  return pg_rms_norm_bwd_ex(dy, lddy, dh, h, C, rstd, gamma, rows, C, io_flags, dx, dgamma, accumulate, workspace, workspace_bytes, stream);
}

extern "C" int pg_rms_norm_bwd_ex(const void* dy, int64_t lddy, const void* dh, const void* h, int64_t ldh, const float* rstd,
                                  const float* gamma, int64_t rows, int32_t C, int32_t io_flags, void* dx, float* dgamma,
                                  int32_t accumulate, void* workspace, int64_t workspace_bytes, void* stream) {
  PG_REQUIRE(dy && h && rstd && gamma && dx && dgamma && rows >= 0 && C > 0 && C <= MAX_C && lddy >= C && ldh >= C,
             "pg_rms_norm_bwd: dy, h, rstd, gamma, dx, dgamma, rows >= 0, 0 < C <= 2^30, lddy >= C and ldh >= C required");
  PG_REQUIRE(io_flags == 0 || io_flags == 3, "pg_rms_norm_bwd: io_flags 0 (fp32) or 3 (bf16)");
  const size_t em = io_flags ? 1 : 3;
  PG_REQUIRE((((size_t)dy | (size_t)dh | (size_t)h | (size_t)dx) & em) == 0 &&
             (((size_t)gamma | (size_t)rstd | (size_t)dgamma | (size_t)workspace) & 3) == 0,
             "pg_rms_norm_bwd: a pointer is not aligned to its element");
  const int64_t need = pg_rms_norm_bwd_workspace(rows, C, io_flags);
  PG_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "pg_rms_norm_bwd: workspace of %lld bytes required", (long long)need);
  hipStream_t st = (hipStream_t)stream;
  if (rows == 0) {                 // an empty sum
    if (!accumulate) rms_dgamma(nullptr, 0, C, dgamma, 0, st);
    PG_LAUNCH_OK("pg_rms_norm_bwd");
    return 0;
  }
  const RmsShape sh = rms_shape((long)rows, C, io_flags ? 8 : 4, 0, true);
  const int lpr = sh.lpr, nch = sh.nch;
  const long nb = nch ? rms_bwd_blocks(rows, lpr, nch) : rms_long_slices(rows);
  PG_REQUIRE(rows <= (1L << 40), "pg_rms_norm_bwd: too many rows");
  PG_REQUIRE(nch || (dx != dy && dx != dh && dx != h), "pg_rms_norm_bwd: rows of more than 2048 channels are read twice: dx must not be an input");
  PG_REQUIRE((dx != dy || lddy == C) && (dx != h || ldh == C), "pg_rms_norm_bwd: dx in place of dy or h needs rows of C elements there");
  RmsBwdK k = {dy, dh, h, rstd, gamma, (long)rows, C, (long)lddy, (long)ldh, dx, (float*)workspace, dgamma, accumulate};
  const bool single = rms_bwd_single(rows, lpr, nch);
  bool none = false;
#define PG_RBN(T, L, N, EX) PG_KLAUNCH((rms_bwd_kernel<T, L, N, 256, EX>), dim3((unsigned)nb), dim3(256), 0, st, k)
#define PG_RBN4(T, L, M, EX)                                                                                       \
  do {                                                                                                             \
    if (RmsV<T>::N == 4) PG_RBN(T, L, (RmsV<T>::N == 4 ? M : 1), EX);                                              \
    else none = true;                                                                                              \
  } while (0)
#define PG_RB1(T, L, EX)                                                                                           \
  do {                                                                                                             \
    if (single) PG_KLAUNCH((rms_bwd_kernel<T, L, 1, 1024, EX>), dim3(1), dim3(1024), 0, st, k);                    \
    else PG_RBN(T, L, 1, EX);                                                                                      \
  } while (0)
#define PG_RB(T)                                                                                                   \
  do {                                                                                                             \
    switch (lpr * 32 + nch * 2 + (sh.ex ? 1 : 0)) {                                                                \
      case 8 * 32 + 3: PG_RB1(T, 8, true); break;                                                                  \
      case 16 * 32 + 3: PG_RB1(T, 16, true); break;                                                                \
      case 32 * 32 + 3: PG_RB1(T, 32, true); break;                                                                \
      case 64 * 32 + 3: PG_RB1(T, 64, true); break;                                                                \
      case 64 * 32 + 5: PG_RBN(T, 64, 2, true); break;                                                             \
      case 64 * 32 + 7: PG_RBN(T, 64, 3, true); break;                                                             \
      case 64 * 32 + 9: PG_RBN(T, 64, 4, true); break;                                                             \
      case 64 * 32 + 11: PG_RBN4(T, 64, 5, true); break;                                                           \
      case 64 * 32 + 13: PG_RBN4(T, 64, 6, true); break;                                                           \
      case 64 * 32 + 15: PG_RBN4(T, 64, 7, true); break;                                                           \
      case 64 * 32 + 17: PG_RBN4(T, 64, 8, true); break;                                                           \
      case 8 * 32 + 2: PG_RB1(T, 8, false); break;                                                                 \
      case 8 * 32 + 4: PG_RBN4(T, 8, 2, false); break;                                                             \
      case 8 * 32 + 6: PG_RBN4(T, 8, 3, false); break;                                                             \
      case 16 * 32 + 2: PG_RB1(T, 16, false); break;                                                               \
      case 16 * 32 + 4: PG_RBN4(T, 16, 2, false); break;                                                           \
      case 16 * 32 + 6: PG_RBN4(T, 16, 3, false); break;                                                           \
      case 32 * 32 + 2: PG_RB1(T, 32, false); break;                                                               \
      case 32 * 32 + 4: PG_RBN4(T, 32, 2, false); break;                                                           \
      case 32 * 32 + 6: PG_RBN4(T, 32, 3, false); break;                                                           \
      case 64 * 32 + 2: PG_RB1(T, 64, false); break;                                                               \
      case 64 * 32 + 4: PG_RBN(T, 64, 2, false); break;                                                            \
      case 64 * 32 + 6: PG_RBN(T, 64, 3, false); break;                                                            \
      case 64 * 32 + 8: PG_RBN(T, 64, 4, false); break;                                                            \
      case 64 * 32 + 10: PG_RBN4(T, 64, 5, false); break;                                                          \
      case 64 * 32 + 12: PG_RBN4(T, 64, 6, false); break;                                                          \
      case 64 * 32 + 14: PG_RBN4(T, 64, 7, false); break;                                                          \
      case 64 * 32 + 16: PG_RBN4(T, 64, 8, false); break;                                                          \
      default:                                                                                                     \
        if (nch) { none = true; break; }                                                                           \
        for (long r0 = 0; r0 < rows; r0 += MAX_BLOCKS) {                                                           \
          const long n = rows - r0 < MAX_BLOCKS ? rows - r0 : MAX_BLOCKS;                                          \
          const RmsBwdK kr = {rms_at(dy, r0 * lddy, sizeof(T)), rms_at(dh, r0 * C, sizeof(T)), rms_at(h, r0 * ldh, sizeof(T)), \
                              rms_at(rstd, r0, 4), gamma, n, C, (long)lddy, (long)ldh, rms_at(dx, r0 * C, sizeof(T)), nullptr, nullptr, 0}; \
          PG_KLAUNCH((rms_bwd_long_kernel<T>), dim3((unsigned)n), dim3(256), 0, st, kr);                           \
        }                                                                                                          \
        PG_KLAUNCH((rms_dgamma_long_kernel<T>), dim3((C + 255) / 256, (unsigned)nb), dim3(256), 0, st, k);         \
        break;                                                                                                     \
    }                                                                                                              \
  } while (0)
  if (io_flags == 0) PG_RB(float);
  else PG_RB(bf16_t);
  PG_REQUIRE(!none, "pg_rms_norm_bwd: no kernel for a row of %d lanes x %d chunks", lpr, nch);
#undef PG_RB
#undef PG_RB1
#undef PG_RBN4
#undef PG_RBN
  if (!(nch && nb == 1)) rms_dgamma((const float*)workspace, (int)nb, C, dgamma, accumulate, st);
  PG_LAUNCH_OK("pg_rms_norm_bwd");
  return 0;
}
