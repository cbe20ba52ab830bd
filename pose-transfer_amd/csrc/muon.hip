// Orthogonalisation of matrices by Newton-Schulz products and the optimiser step that uses it (Muon), gfx950.
//
//   X0 = U / (|U|_F + eps),   X_{k+1} = (a I + b A + c A^2) X_k,  A = X_k X_k^T on the short side,  (a, b, c) = (3.4445, -4.7750, 2.0315)
//   step:  m' = mu m + (1 - mu) g;  u = nesterov ? (1 - mu) g + mu m' : m';  p = (1 - lr wd) p - lr scale X_steps(u)
//
// What is computed.  Every X_k is a polynomial of G = X0 X0^T times X0, and polynomials of one symmetric matrix commute and are symmetric.
// So a STAGE of up to three steps takes one product over the long side for G, a chain of m x m products
//   H = G G;  Q = a I + b G + c H;  P <- Q P;  G <- Q (Q G)
// and one product over the long side X <- P X, instead of two long products per step: 4 long products for five steps instead of 10.
// Why stages: G squares the singular values, fp32 sums lose those below 2^-12 of the largest, and each step amplifies what is left by
// up to a = 3.44.  After three steps they are 41 times larger and a new Gram matrix sees them.  Measured against 64 bits on
// gradients with singular values falling as 1/k (256 x 2048): one stage of five steps 1.6e-4 (2-norm, relative), stages of
// 3 + 2 steps 4e-6, the ten-product form in fp32 4e-6.
//
// Arithmetic.  The matrix cores have no fast fp32 form (1 / 16 of the fp16 rate).  Every operand is held as TWO fp16 values, hi + lo =
// 22 bits, scaled by a power of two; a product is three MFMAs, hi hi + hi lo + lo hi, with fp32 accumulation: what an fp32 product
// gives (measured 4.8e-6 against 4.7e-6 through five steps; a bf16 pair with its 16 bits: 4e-5, single bf16 operands: 2e-2).
// fp16 has few exponents: below 2^-3 of a plane's unit the pair loses bits, its error is then 2^-25 absolute.  So every plane's largest value
// lies near fp16's end: X0's largest element at 2^14 .. 2^15; |G|, |Q G| <= 1.5, |Q| <= 3.45 and |P| <= 3.45^3 = 41 bound the others.
// Elements keep 22 bits down to 2^-18 of the largest and 2^-40 of it behind that.  A row that is a fraction r of the others comes out
// with an error of about max(1e-6, 5e-11 / r) of itself (128 x 1152: 7e-7 at r = 1e-4, 6e-6 at 1e-5, 5e-5 at 1e-6; the limit is
// 2^-40 in G), a column of the long side (n of them) with about 1e-12 sqrt(n) / r (the planes between stages); fp32 products keep 1e-6.
// With the mean square at 1 instead of the largest element at 2^14, rows came out at 1.7e-4, 1.8e-3 and 1.7e-2.
// A bf16 input (8 bits) is one fp16 value exactly down to 2^-32 of the largest, behind that to 2^-40 of it: one plane.
//
// Layout.  A matrix is stored by the caller as [taps][rows][cols] with row and tap strides (a packed convolution weight is one matrix
// [rows, taps * cols]).  The planes here are M x N, M <= N the short side, both padded with zeros to multiples of 64: no product checks
// a bound along K, and padding stays zero through every step.  They (and the m x m matrices) are stored in blocks of 16 columns,
// [column / 16][row][16], the rows of a block padded by 8: what a product needs next of any run of rows is contiguous, and neighbouring blocks
// begin on different L2 channels.  (Row-major planes, whose rows lie a large power of two apart, held every product at 6.5 TB/s of operands.)
// All matrices of a call share every launch (a device table of tile ranges).
#include "common.h"
#include <math.h>
#include <new>
#include <vector>

namespace pg {

typedef unsigned short bf16_t;
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;
constexpr int SG = 15, SQ = 14, SP = 10;        // log2 of the scales of G and Q G, of Q, of P
// elements per workgroup of the momentum pass, and runs of up to eight neighbours per workgroup of the square-sum pass: small tensors give
// few workgroups; large ones at most 1024 partial sums, which every workgroup of the split reads
constexpr long MAX_PARTIALS = 1024;
__host__ __device__ constexpr int k0_elems(long n) {
  return n < (1L << 21) ? 4096 : n <= 16384 * MAX_PARTIALS ? 16384 : (int)((n + MAX_PARTIALS * 4096 - 1) / (MAX_PARTIALS * 4096) * 4096);
}
__host__ __device__ constexpr int sq_runs(long runs) {
  return runs <= 512 * MAX_PARTIALS ? 512 : (int)((runs + MAX_PARTIALS * 256 - 1) / (MAX_PARTIALS * 256) * 256);
}
// Q = a I + b G + c G G in the planes' units
constexpr float QUAD_A = NS_A * (float)(1 << SQ), QUAD_B = NS_B / (float)(1 << (SG - SQ)), QUAD_C = NS_C / (float)(1 << (2 * SG - SQ));
constexpr int GT = 128, AI = 128, AJ = 128;      // tiles: Gram; apply (rows, columns)

struct NsMat {
  long src, ld, st;             // the caller's storage: element offset, row stride, tap stride
  int taps, rows, cols, kind;   // kind 1: a vector (Adam), rows = taps = 1
  int M, N, Mp, Np, tall;       // short and long side, padded; tall: the rows are the long side
  int ks, kc;                   // Gram: splits of the long side and their length (a multiple of 32)
  int np;                       // partial sums of squares
  float scale;
  long x, g, part;              // offsets in the workspace: X planes and chain planes (halves), Gram partials (floats)
  int sq0;                      // first partial sum of squares
};
enum { F_MOM, F_SPLIT, F_GRAM, F_JOIN, F_CHAIN, F_APPLY, F_N };       // launches (F_JOIN also: the chain's tiles of 32)
struct NsGroup {                // matrices of one call: a device table, or (tab = nullptr) `n` equal ones
  const NsMat* tab;
  const int* first;             // [F_N][n]: the first workgroup of each record
  int n;
  NsMat u;                      // the single record of equal matrices: offsets of number 0
  long src_step, out_step, x_step, g_step, part_step;
  int per[F_N];                 // workgroups per matrix
};
struct NsRef { NsMat m; int id, tile; long out; };

template <int F>
__device__ __forceinline__ NsRef ns_find(const NsGroup& gr, int b) {
  NsRef r;
  if (gr.tab == nullptr) {
    const int per = gr.per[F];
    r.id = b / per;
    r.tile = b - r.id * per;
    r.m = gr.u;
    r.out = (long)r.id * gr.out_step;
    r.m.src += (long)r.id * gr.src_step;
    r.m.x += (long)r.id * gr.x_step; r.m.g += (long)r.id * gr.g_step; r.m.part += (long)r.id * gr.part_step;
    return r;
  }
  // the last record whose range begins at or before b: 64 at a time, one load and a vote
  int id = -1;
  for (int c = 0; c < gr.n; c += 64) {
    const int i = c + (int)(threadIdx.x & 63);
    const unsigned long long vote = __ballot(i < gr.n && gr.first[F * gr.n + i] <= b);
    id += __popcll(vote);
    if (~vote) break;
  }
  r.id = __builtin_amdgcn_readfirstlane(id);
  r.m = gr.tab[r.id];
  r.tile = b - gr.first[F * gr.n + r.id];
  r.out = r.m.src;
  return r;
}

__device__ __forceinline__ float bf2f(bf16_t v) { return __uint_as_float((unsigned)v << 16); }
__device__ __forceinline__ unsigned ns_pack_bf16(float lo, float hi) {
  unsigned r;
  asm("v_cvt_pk_bf16_f32 %0, %1, %2" : "=v"(r) : "v"(lo), "v"(hi));
  return r;
}
// v = hi + lo in fp16; the remainder is exact in fp32, its rounding is 2^-22 of v (2^-25 where lo is subnormal)
__device__ __forceinline__ void split16(float v, _Float16& hi, _Float16& lo) {
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}
// sum of squares and largest magnitude of some elements of a matrix (a NaN shows in the sum)
struct NsNorm { double sum; float top; int _pad; };
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}
__device__ __forceinline__ NsNorm block_norm256(double sum, float top, NsNorm* red) {
  sum = wave_sum_d(sum);
  top = wave_max(top);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) { red[threadIdx.x >> 6].sum = sum; red[threadIdx.x >> 6].top = top; }
  __syncthreads();
  return {red[0].sum + red[1].sum + red[2].sum + red[3].sum, fmaxf(fmaxf(red[0].top, red[1].top), fmaxf(red[2].top, red[3].top)), 0};
}

// ---------------------------------------------------------------------------------------------- table upload
// the table travels in kernel arguments: nothing of the caller's memory is read after the call, and a captured graph keeps its copy
struct NsChunk { NsMat m[16]; int first[F_N][16]; };
__global__ void ns_table_kernel(NsChunk c, NsMat* tab, int* first, int at, int n, int total) {
  const int words = (int)(sizeof(NsMat) / 4);
  for (int i = threadIdx.x; i < n * words; i += 256)
    reinterpret_cast<unsigned*>(tab + at)[i] = reinterpret_cast<const unsigned*>(&c)[i];
  for (int i = threadIdx.x; i < n * F_N; i += 256) first[(i / n) * total + at + i % n] = c.first[i / n][i % n];
}

// ---------------------------------------------------------------------------------------------- momentum, Adam, sums of squares
struct NsStep {
  float* p; const float* g; const bf16_t* gb; float* m; float* v; bf16_t* pb;
  float mu, gscale, lr, wd;
  int nesterov;
  float b1, b2, eps;
  double b1d, b2d;
  long step0;
  const unsigned long long* ctr;
};
__device__ __forceinline__ float ns_grad(const NsStep& s, long i) { return (s.gb ? bf2f(s.gb[i]) : s.g[i]) * s.gscale; }
__device__ __forceinline__ float ns_update(const NsStep& s, float g, float m1) { return s.nesterov ? (1.f - s.mu) * g + s.mu * m1 : m1; }

// one workgroup = k0_elems consecutive elements of a tensor; 28 bytes / element for Adam's, 12 for a matrix's: HBM-bound (77 M elements of
// 20 matrices: 177 us, 5.2 TB/s; 2.8 M: 13 us)
__global__ __launch_bounds__(256) void muon_momentum_kernel(const NsGroup gr, const NsStep s, NsNorm* sq) {
  __shared__ NsNorm red[4];
  __shared__ double bc[2];
  const NsRef r = ns_find<F_MOM>(gr, blockIdx.x);
  const long n = (long)r.m.taps * r.m.rows * r.m.cols;
  const long e0 = (long)r.tile * k0_elems(n), e1 = min(n, e0 + k0_elems(n));
  const long base = r.m.src;
  if (r.m.kind == 1) {
    if (threadIdx.x < 2) {                             // 1 - beta^t, in fp64, by one lane each
      const double t = (double)(s.step0 + (s.ctr ? (long)s.ctr[0] : 0L));
      bc[threadIdx.x] = 1.0 - pow(threadIdx.x ? s.b2d : s.b1d, t);
    }
    __syncthreads();
    const float step_size = (float)((double)s.lr / bc[0]);
    const float bc2 = (float)sqrt(bc[1]);
#pragma unroll 4
    for (long i = e0 + threadIdx.x; i < e1; i += 256) {
      const float g = ns_grad(s, base + i);
      const float m = s.m[base + i] * s.b1 + (1.f - s.b1) * g;
      const float v = s.v[base + i] * s.b2 + (1.f - s.b2) * g * g;
      const float p = s.p[base + i] - step_size * (m / (sqrtf(v) / bc2 + s.eps));
      s.m[base + i] = m; s.v[base + i] = v; s.p[base + i] = p;
      if (s.pb) s.pb[base + i] = (bf16_t)(ns_pack_bf16(p, 0.f) & 0xffffu);
    }
    return;
  }
  double acc = 0.0;
  float top = 0.f;
  const bool vec = ((base | n) & 3) == 0;
  if (vec) {
#pragma unroll 4
    for (long i = e0 + threadIdx.x * 4; i < e1; i += 1024) {
      float g[4];
      if (s.gb) {
        const uint2 q = *reinterpret_cast<const uint2*>(s.gb + base + i);
        g[0] = __uint_as_float(q.x << 16); g[1] = __uint_as_float(q.x & 0xffff0000u);
        g[2] = __uint_as_float(q.y << 16); g[3] = __uint_as_float(q.y & 0xffff0000u);
      } else {
        const float4 q = *reinterpret_cast<const float4*>(s.g + base + i);
        g[0] = q.x; g[1] = q.y; g[2] = q.z; g[3] = q.w;
      }
      float4 mq = *reinterpret_cast<const float4*>(s.m + base + i);
      float m[4] = {mq.x, mq.y, mq.z, mq.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float gg = g[e] * s.gscale;
        m[e] = s.mu * m[e] + (1.f - s.mu) * gg;
        const float u = ns_update(s, gg, m[e]);
        acc = fma((double)u, (double)u, acc);
        top = fmaxf(top, fabsf(u));
      }
      *reinterpret_cast<float4*>(s.m + base + i) = make_float4(m[0], m[1], m[2], m[3]);
    }
  } else {
    for (long i = e0 + threadIdx.x; i < e1; i += 256) {
      const float gg = ns_grad(s, base + i);
      const float m = s.mu * s.m[base + i] + (1.f - s.mu) * gg;
      s.m[base + i] = m;
      const float u = ns_update(s, gg, m);
      acc = fma((double)u, (double)u, acc);
      top = fmaxf(top, fabsf(u));
    }
  }
  const NsNorm n4 = block_norm256(acc, top, red);
  if (threadIdx.x == 0) sq[blockIdx.x] = n4;
}

// the stored element (row, flat column = tap * cols + col) of a matrix that is orthogonalised
// SRC: 0 = fp32 tensor, 1 = bf16 tensor, 2 = the step's u from (g, m')
template <int SRC>
__device__ __forceinline__ float ns_elem(const void* x, const NsStep& s, long i) {
  if constexpr (SRC == 0) return reinterpret_cast<const float*>(x)[i];
  else if constexpr (SRC == 1) return bf2f(reinterpret_cast<const bf16_t*>(x)[i]);
  else return ns_update(s, ns_grad(s, i), s.m[i]);
}
__device__ __forceinline__ long ns_at(const NsMat& m, int row, int fc) {
  const int tap = m.taps == 1 ? 0 : fc / m.cols;
  return m.src + (long)tap * m.st + (long)row * m.ld + (fc - tap * m.cols);
}
struct __attribute__((packed, aligned(2))) NsU2 { unsigned x, y; };
struct __attribute__((packed, aligned(2))) NsU4 { unsigned x, y, z, w; };      // 16 bytes at the alignment of one element
__device__ __forceinline__ void ns_ld8(const float* q, float (&v)[8]) {
  const NsU4 a = reinterpret_cast<const NsU4*>(q)[0], b = reinterpret_cast<const NsU4*>(q)[1];
  v[0] = __uint_as_float(a.x); v[1] = __uint_as_float(a.y); v[2] = __uint_as_float(a.z); v[3] = __uint_as_float(a.w);
  v[4] = __uint_as_float(b.x); v[5] = __uint_as_float(b.y); v[6] = __uint_as_float(b.z); v[7] = __uint_as_float(b.w);
}
__device__ __forceinline__ void ns_ld8(const bf16_t* q, float (&v)[8]) {
  const NsU4 a = *reinterpret_cast<const NsU4*>(q);
  const unsigned w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) { v[2 * e] = __uint_as_float(w[e] << 16); v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u); }
}
// flat columns fc .. fc + 7 of a stored row, zero behind the last one
template <int SRC>
__device__ __forceinline__ void ns_load8(const NsMat& m, const void* x, const NsStep& s, int row, int fc, float (&v)[8]) {
  const int width = m.taps * m.cols;
  int tap = 0, col = fc;
  if (m.taps > 1) { tap = fc / m.cols; col = fc - tap * m.cols; }
  long at = m.src + (long)tap * m.st + (long)row * m.ld + col;
  if (col + 8 <= m.cols) {
    if constexpr (SRC == 0) ns_ld8(reinterpret_cast<const float*>(x) + at, v);
    else if constexpr (SRC == 1) ns_ld8(reinterpret_cast<const bf16_t*>(x) + at, v);
    else {
      ns_ld8(s.m + at, v);
      if (s.nesterov) {
        float g[8];
        if (s.gb) ns_ld8(s.gb + at, g);
        else ns_ld8(s.g + at, g);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = ns_update(s, g[e] * s.gscale, v[e]);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = fc + e < width ? ns_elem<SRC>(x, s, at) : 0.f;
      ++col; ++at;
      if (col == m.cols) { col = 0; at += m.st - m.cols; }
    }
  }
}

// one workgroup = sq_runs runs of eight stored neighbours
template <int SRC>
__global__ __launch_bounds__(256) void ns_sumsq_kernel(const NsGroup gr, const void* x, NsNorm* sq) {
  __shared__ NsNorm red[4];
  const NsRef r = ns_find<F_MOM>(gr, blockIdx.x);
  const unsigned rpr = (unsigned)(r.m.cols + 7) / 8u;
  const unsigned n = (unsigned)r.m.rows * rpr;
  const unsigned per = (unsigned)sq_runs((long)n), e0 = (unsigned)r.tile * per, e1 = min(n, e0 + per);
  double acc = 0.0;
  float top = 0.f;
  const NsStep s{};
  for (unsigned i = e0 + threadIdx.x; i < e1; i += 256) {
    const unsigned row = i / rpr;
    float v[8];
    ns_load8<SRC>(r.m, x, s, (int)row, (int)(i - row * rpr) * 8, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) { acc = fma((double)v[e], (double)v[e], acc); top = fmaxf(top, fabsf(v[e])); }
  }
  const NsNorm n4 = block_norm256(acc, top, red);
  if (threadIdx.x == 0) sq[blockIdx.x] = n4;
}

// element (i, j) of a plane in blocks of 16 columns; planes of X and of an m x m matrix
__device__ __forceinline__ long cat(int Mp, int i, int j) { return ((long)(j >> 4) * (Mp + 8) + i) * 16 + (j & 15); }
__device__ __forceinline__ long xplane(const NsMat& m) { return (long)m.Np * (m.Mp + 8); }
__device__ __forceinline__ long cplane(const NsMat& m) { return (long)m.Mp * (m.Mp + 8); }

// ---------------------------------------------------------------------------------------------- split into fp16 planes
// planes hold 2^-k U with a largest element of 2^14 .. 2^15 (as far as k goes: an infinity makes the planes infinite)
__device__ __forceinline__ int ns_exponent(float top) {
  return max(-126, min(126, (int)((__float_as_uint(top) >> 23) & 0xff) - 127 - 14));
}
__device__ __forceinline__ float ns_pow2(int k) { return __uint_as_float((unsigned)(k + 127) << 23); }      // |k| <= 126
// A matrix's units: c = 2^k / (|U| + eps), from the first planes' to X0's, and gap with |X0|_F <= 2^-gap: 0 but where eps outweighs |U|.
// Later planes hold 2^(15 + gap(stage)) X: |X| <= 1.21 (the quintic's largest value on [0, 1.21]) fits fp16, and so does an X that began
// at 2^-gap and grew by up to 3.4445^3 < 2^6 a stage; at 2^15 alone it would sink below fp16's smallest values.
struct NsUnit { float c; int gap; };
__device__ __forceinline__ NsUnit ns_unit_of(double sumsq, int k, float eps) {
  const double n = sqrt(sumsq), x0 = n / (n + (double)eps);
  const int e = (int)((__double_as_longlong(x0) >> 52) & 0x7ff) - 1023;              // x0 < 2^(e + 1); NaN: 1024
  return {sumsq == 0.0 ? 0.f : (float)((double)ns_pow2(k) / (n + (double)eps)), max(0, min(96, -(e + 1)))};
}
__device__ __forceinline__ int ns_gap(const NsUnit& u, int stage) { return max(0, u.gap - 6 * stage); }
// from the planes' units at the beginning of a stage to values
__device__ __forceinline__ float ns_value(const NsUnit& u, int stage) { return stage == 0 ? u.c : ns_pow2(-15 - ns_gap(u, stage)); }

// every workgroup joins its matrix's partial sums of squares itself (at most 1024); the first one publishes
// the matrix's units.  12 bytes / element from fp32 pairs (m', g), HBM-bound: 212 - 215 us for 77 M
// elements (4.3 TB/s); 12 us for 512 x 24576 bf16 (6 bytes)
template <int SRC>
__global__ __launch_bounds__(256) void ns_split_kernel(const NsGroup gr, const void* x, const NsStep s, const NsNorm* sq, float eps,
                                                       NsUnit* unit, _Float16* ws) {
  __shared__ NsNorm red[4];
  __shared__ float tile[64][65];
  constexpr bool ONE = SRC == 1;
  const NsRef r = ns_find<F_SPLIT>(gr, blockIdx.x);
  const NsMat& m = r.m;
  const int np = m.np;
  const int first = gr.tab ? m.sq0 : r.id * gr.per[F_MOM];
  // the tile's elements are on their way while the sums are joined
  // wide: 64 rows x 128 columns, 8 plane elements per thread and trip, 1 KB runs per wave
  const int tr = m.Mp / 64, tj = m.Np / 64;
  const int wi = (r.tile % tr) * 64 + ((threadIdx.x >> 1) & 63), wj = (r.tile / tr) * 128 + (threadIdx.x & 1) * 8 + (threadIdx.x >> 7) * 16;
  // tall: 64 x 64 through LDS, plane row i = stored flat column, plane column j = stored row
  const int i0 = (r.tile / tj) * 64, j0 = (r.tile % tj) * 64, tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
  float v[4][8];
  if (!m.tall) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int j = wj + q * 32;
      if (wi < m.M && j < m.N) {
        ns_load8<SRC>(m, x, s, wi, j, v[q]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[q][e] = 0.f;
      }
    }
  } else {
#pragma unroll
    for (int q = 0; q < 16; ++q) {
      const int j = j0 + q * 4 + ty, i = i0 + tx;
      v[q >> 3][q & 7] = (j < m.N && i < m.M) ? ns_elem<SRC>(x, s, ns_at(m, j, i)) : 0.f;
    }
  }
  double a = 0.0;
  float top = 0.f;
  for (int i = threadIdx.x; i < np; i += 256) { a += sq[first + i].sum; top = fmaxf(top, sq[first + i].top); }
  const NsNorm nm = block_norm256(a, top, red);
  const int k = ns_exponent(nm.top);
  const float f = ns_pow2(-k);
  if (r.tile == 0 && threadIdx.x == 0) unit[r.id] = ns_unit_of(nm.sum, k, eps);
  _Float16* hi = ws + m.x;
  _Float16* lo = hi + xplane(m);
  if (!m.tall) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int j = wj + q * 32;
      if (j >= m.Np) break;
      half8 h, l;
#pragma unroll
      for (int e = 0; e < 8; ++e) { _Float16 th, tl; split16(v[q][e] * f, th, tl); h[e] = th; l[e] = tl; }
      *reinterpret_cast<half8*>(hi + cat(m.Mp, wi, j)) = h;
      if constexpr (!ONE) *reinterpret_cast<half8*>(lo + cat(m.Mp, wi, j)) = l;
    }
  } else {
#pragma unroll
    for (int q = 0; q < 16; ++q) tile[q * 4 + ty][tx] = v[q >> 3][q & 7];
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int c = q * 256 + threadIdx.x, i = (c >> 1) & 63, j = (c & 1) * 8 + (c >> 7) * 16;
      half8 h, l;
#pragma unroll
      for (int e = 0; e < 8; ++e) { _Float16 th, tl; split16(tile[j + e][i] * f, th, tl); h[e] = th; l[e] = tl; }
      *reinterpret_cast<half8*>(hi + cat(m.Mp, i0 + i, j0 + j)) = h;
      if constexpr (!ONE) *reinterpret_cast<half8*>(lo + cat(m.Mp, i0 + i, j0 + j)) = l;
    }
  }
}

// ---------------------------------------------------------------------------------------------- product cores
// Workgroups are dealt round-robin to the 8 XCDs, each with an L2 of its own: `grp` consecutive tiles, which share operand rows, go
// to one of them.  grp is the number of tiles of the largest matrix that read the same rows: all tiles of a Gram slice, of a chain matrix,
// of a column strip of the apply product (against a 512-sided matrix's 10, 36 and 4 for every size: 16 x 256 x 4096 283 -> 273 us,
// 1024 x 8192 412 -> 403 us).  The grid is padded to a multiple of 8; < 0: no tile.
__device__ __forceinline__ int xcd_tile(int b, int total, int grp) {
  const int chunk = 8 * grp, full = total / chunk * chunk;
  if (b < full) {
    const int q = b / chunk, r = b - q * chunk;
    return q * chunk + (r & 7) * grp + (r >> 3);
  }
  const int r = b - full, g2 = (total - full + 7) >> 3;
  const int t = full + (r & 7) * g2 + (r >> 3);
  return (r >> 3) < g2 && t < total ? t : -1;
}

// LDS image of an operand: blocks of [rows][16], a row = two 16-byte chunks, chunk c of row r at slot c ^ ((r >> 3) & 1): the 16 lanes
// that a ds_read_b128 serves at a time (16 consecutive rows, one chunk) then cover the 256 bytes of a bank row once.
// Tiles go global -> LDS without registers (one instruction = 64 lanes x 16 bytes = 1 KB in LDS order), ST stages deep; the operand
// reads of a K step and their wait are ONE asm block: the compiler, which would wait for every transfer in flight before any LDS
// read, does not see them, and nothing can come between a read and its wait.  The other waves of the SIMD cover that wait.
__device__ __forceinline__ void dma16(const _Float16* src, char* dst) {
  __builtin_amdgcn_global_load_lds(reinterpret_cast<const float*>(src), reinterpret_cast<float*>(dst), 16, 0, 0);
}
template <int N>
__device__ __forceinline__ void wait_dma() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void wg_barrier() {
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
}
__device__ __forceinline__ int swz(int row) { return (row >> 3) & 1; }

// one K step (16) of T + T fragments, 32 rows (1 KB) apart, planes PS bytes apart
#define NS_RD "ds_read_b128 "
template <int PS>
__device__ __forceinline__ void fetch_nt(unsigned pa, unsigned pb, half8 (&a)[2][1], half8 (&b)[2][1]) {
  asm volatile(NS_RD "%0, %4\n\t" NS_RD "%2, %5\n\t" NS_RD "%1, %4 offset:%6\n\t" NS_RD "%3, %5 offset:%6\n\t" "s_waitcnt lgkmcnt(0)"
               : "=&v"(a[0][0]), "=&v"(a[1][0]), "=&v"(b[0][0]), "=&v"(b[1][0]) : "v"(pa), "v"(pb), "n"(PS) : "memory");
}
template <int PS>
__device__ __forceinline__ void fetch_nt(unsigned pa, unsigned pb, half8 (&a)[2][2], half8 (&b)[2][2]) {
  asm volatile(NS_RD "%0, %8\n\t" NS_RD "%4, %9\n\t" NS_RD "%1, %8 offset:1024\n\t" NS_RD "%5, %9 offset:1024\n\t"
               NS_RD "%2, %8 offset:%10\n\t" NS_RD "%3, %8 offset:%11\n\t" NS_RD "%6, %9 offset:%10\n\t" NS_RD "%7, %9 offset:%11\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(a[0][0]), "=&v"(a[0][1]), "=&v"(a[1][0]), "=&v"(a[1][1]), "=&v"(b[0][0]), "=&v"(b[0][1]), "=&v"(b[1][0]), "=&v"(b[1][1])
               : "v"(pa), "v"(pb), "n"(PS), "n"(PS + 1024) : "memory");
}
template <int PS>
__device__ __forceinline__ void fetch_nt(unsigned pa, unsigned pb, half8 (&a)[1][2], half8 (&b)[1][2]) {
  asm volatile(NS_RD "%0, %4\n\t" NS_RD "%2, %5\n\t" NS_RD "%1, %4 offset:1024\n\t" NS_RD "%3, %5 offset:1024\n\t" "s_waitcnt lgkmcnt(0)"
               : "=&v"(a[0][0]), "=&v"(a[0][1]), "=&v"(b[0][0]), "=&v"(b[0][1]) : "v"(pa), "v"(pb) : "memory");
}

// C[BM][BM] = sum_k A[i][k] B[j][k] over columns k0 .. k1 - 1 (multiples of 32), operands as PL fp16 planes in blocks; 4 waves (2 x 2), two
// blocks per stage, ST stages.  `same`: A and B are the same rows, moved once.  Rows behind a_rows / b_rows read the last one instead:
// their products belong to rows and columns that nobody stores.
template <int BM, int PL, int ST>
struct NtCore {
  static constexpr int T = BM / 64, BLK = BM * 32, OP = PL * 2 * BLK, STAGE = 2 * OP;      // [operand][plane][block][BM][16]
  static constexpr int NI = STAGE / 4096;                           // transfers per wave and stage
  static constexpr int LDS_BYTES = ST * STAGE;
  static_assert((T == 1 || T == 2) && LDS_BYTES <= 64 * 1024, "tile");
  f32x16 acc[T][T];

  __device__ __forceinline__ void run(char* smem, const _Float16* A, int a_rows, const _Float16* B, int b_rows, long plane, int pitch, bool same,
                                      int k0, int k1) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = (wave >> 1) * (BM / 2), wn = (wave & 1) * (BM / 2);
#pragma unroll
    for (int i = 0; i < T; ++i)
#pragma unroll
      for (int j = 0; j < T; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    const _Float16* src[NI];
#pragma unroll
    for (int q = 0; q < NI; ++q) {                   // transfer x of a stage: operand, plane, block, 32 rows
      const int x = q * 4 + wave, op = x / (NI * 2), y = x % (BM / 32), z = x / (BM / 32) % (PL * 2);
      const int row = y * 32 + (lane >> 1);
      src[q] = (op ? B : A) + (z >> 1) * plane + ((long)(k0 / 16 + (z & 1)) * pitch + min(row, (op ? b_rows : a_rows) - 1)) * 16 +
               ((lane & 1) ^ swz(row)) * 8;
    }
    const long step = 32L * pitch;
    auto issue = [&](int st) {
#pragma unroll
      for (int q = 0; q < NI; ++q) {
        if (q == NI / 2 && same) break;
        dma16(src[q], smem + st * STAGE + (q * 4 + wave) * 1024);
        src[q] += step;
      }
    };
    const int n = (k1 - k0) / 32;
    const unsigned lds0 = (unsigned)(size_t)smem;
    const int r = lane & 31;
    const unsigned off = (unsigned)(r * 32 + (((lane >> 5) ^ swz(r)) << 4));
    const unsigned pa = lds0 + wm * 32 + off, pb = lds0 + (same ? 0 : OP) + wn * 32 + off;
#pragma unroll
    for (int q = 0; q < ST - 1; ++q)
      if (q < n) issue(q);
    int cur = 0, nxt = ST - 1;
    for (int it = 0; it < n; ++it) {
      if (it + ST - 2 >= n) wait_dma<0>();
      else if (same) wait_dma<NI / 2 * (ST - 2)>();
      else wait_dma<NI * (ST - 2)>();
      wg_barrier();
      if (it + ST - 1 < n) issue(nxt);
      const unsigned so = (unsigned)(cur * STAGE);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        half8 a[PL][T], b[PL][T];
        fetch_nt<2 * BLK>(pa + so + ks * BLK, pb + so + ks * BLK, a, b);
#pragma unroll
        for (int i = 0; i < T; ++i)
#pragma unroll
          for (int j = 0; j < T; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0][i], b[0][j], acc[i][j], 0, 0, 0);
        if constexpr (PL == 2) {
#pragma unroll
          for (int i = 0; i < T; ++i)
#pragma unroll
            for (int j = 0; j < T; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0][i], b[PL - 1][j], acc[i][j], 0, 0, 0);
#pragma unroll
          for (int i = 0; i < T; ++i)
#pragma unroll
            for (int j = 0; j < T; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[PL - 1][i], b[0][j], acc[i][j], 0, 0, 0);
        }
      }
      cur = cur + 1 == ST ? 0 : cur + 1;
      nxt = nxt + 1 == ST ? 0 : nxt + 1;
    }
  }
};

// tile number of the lower triangle (bi >= bj), row by row
__device__ __forceinline__ void tri(int t, int& bi, int& bj) {
  int i = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
  while ((i + 1) * (i + 2) / 2 <= t) ++i;
  while (i * (i + 1) / 2 > t) --i;
  bi = i;
  bj = t - i * (i + 1) / 2;
}

// G = X X^T over one slice of the long side: fp32 partial tiles, in the order of the accumulators (one float4 = four rows of a column).
// 128 x 128 tiles of the lower triangle, two workgroups per CU; the long side in as many slices as run at once.  The generator's 20 matrices (up to
// 512 x 24576) take 202 - 214 us, 512 x 24576 alone 29 us (two planes) and 16 us (bf16: one).  Bound by power: the counters show the MFMAs busy for 47 % of
// the cycles, and where the chip rests between launches the generator's take 153 us, at 2.0 GHz.  Where few slices
// run (16 x 770 x 189: 144 workgroups, 11 - 13 us) it is launch, first transfer and the partial tiles' way out; more stages or slices gave nothing.
template <int PL>
__global__ __launch_bounds__(256, 2) void ns_gram_kernel(const NsGroup gr, int total, int grp, const _Float16* ws, float* part) {
  typedef NtCore<GT, PL, 2> Core;
  __shared__ __attribute__((aligned(1024))) char smem[Core::LDS_BYTES];
  const int b = xcd_tile(blockIdx.x, total, grp);
  if (b < 0) return;
  const NsRef r = ns_find<F_GRAM>(gr, b);
  const NsMat& m = r.m;
  const int nt = (m.Mp + GT - 1) / GT, ntri = nt * (nt + 1) / 2;
  const int split = r.tile / ntri, t = r.tile - split * ntri;
  int bi, bj;
  tri(t, bi, bj);
  const _Float16* X = ws + m.x;
  Core c;
  c.run(smem, X + (long)bi * GT * 16, m.Mp - bi * GT, X + (long)bj * GT * 16, m.Mp - bj * GT, xplane(m), m.Mp + 8, bi == bj,
        split * m.kc, min(m.Np, (split + 1) * m.kc));
  float4* out = reinterpret_cast<float4*>(part + m.part + (long)r.tile * (GT * GT));
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        out[((wave * 4 + i * 2 + j) * 4 + q) * 64 + lane] =
            make_float4(c.acc[i][j][4 * q], c.acc[i][j][4 * q + 1], c.acc[i][j][4 * q + 2], c.acc[i][j][4 * q + 3]);
}

// join of the slices, in order; both triangles of G from the lower one.  One workgroup = one 32 x 32 block, a float4 per thread: 4 - 7 us, mostly
// launch (11 - 13 us for the generator's 20 matrices)
__global__ __launch_bounds__(256) void ns_gram_join_kernel(const NsGroup gr, const float* part, const NsUnit* unit, int stage, _Float16* ws) {
  const NsRef r = ns_find<F_JOIN>(gr, blockIdx.x);
  const NsMat& m = r.m;
  int bi, bj;
  tri(r.tile, bi, bj);                               // in units of 32
  const int gi = bi / 4, gj = bj / 4, fi = bi & 3, fj = bj & 3;      // its 128-tile, and where in it
  const int nt = (m.Mp + GT - 1) / GT, ntri = nt * (nt + 1) / 2;
  const int wave = (fi >> 1) * 2 + (fj >> 1), frag = wave * 4 + (fi & 1) * 2 + (fj & 1);
  const int lane = threadIdx.x & 63, q = threadIdx.x >> 6;
  const float4* src = reinterpret_cast<const float4*>(part + m.part + (long)(gi * (gi + 1) / 2 + gj) * (GT * GT)) + (frag * 4 + q) * 64 + lane;
  const float c1 = ns_value(unit[r.id], stage);
  const float c2 = c1 * c1 * (float)(1 << SG);
  float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int s = 0; s < m.ks; ++s) {
    const float4 f = src[(long)s * ntri * (GT * GT / 4)];
    v[0] += f.x; v[1] += f.y; v[2] += f.z; v[3] += f.w;
  }
  const int i0 = bi * 32 + 8 * q + 4 * (lane >> 5), j0 = bj * 32 + (lane & 31);
  const long pl = cplane(m);
  _Float16* G = ws + m.g;
  half4 hh, ll;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    _Float16 h, l;
    split16(v[e] * c2, h, l);
    hh[e] = h; ll[e] = l;
    if (i0 + e >= j0) { G[cat(m.Mp, i0 + e, j0)] = h; G[pl + cat(m.Mp, i0 + e, j0)] = l; }
  }
  if (bi != bj) {
    *reinterpret_cast<half4*>(G + cat(m.Mp, j0, i0)) = hh;
    *reinterpret_cast<half4*>(G + pl + cat(m.Mp, j0, i0)) = ll;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (i0 + e > j0) { G[cat(m.Mp, j0, i0 + e)] = hh[e]; G[pl + cat(m.Mp, j0, i0 + e)] = ll[e]; }
  }
}

// chain planes of a matrix: 0 G, 1 Q, 2 Q G, 3 P, 4 the other P  (hi and lo each)
// C = A B of commuting symmetric matrices: the lower triangle of 64 x 64 tiles, mirrored.  `quad`: C = a I + b A + c A A
struct ChainJob { int a, b, c; float mul; int quad; };

// Tiles of 64 x 64 (many matrices): four stages of 16 KB, two workgroups per CU; 17 - 19 us for 472
// tiles of 64 .. 512 columns (32 x 32 tiles: 22 - 23 us; a launch of two jobs 31 and 38 us).  The result leaves through LDS: written four
// neighbours at a time as the mirrored tile, which is copied out as it is and, by transposing reads, turned.
__global__ __launch_bounds__(256, 2) void ns_chain_kernel(const NsGroup gr, ChainJob j0, ChainJob j1, int total, int tiles, int grp, _Float16* ws) {
  typedef NtCore<64, 2, 4> Core;
  __shared__ __attribute__((aligned(1024))) char smem[Core::LDS_BYTES];
  const int t = xcd_tile(blockIdx.x, total, grp);
  if (t < 0) return;
  const ChainJob jb = t >= tiles ? j1 : j0;          // two jobs: the second one's tiles come behind the first one's
  const NsRef r = ns_find<F_CHAIN>(gr, t >= tiles ? t - tiles : t);
  const NsMat& m = r.m;
  int bi, bj;
  tri(r.tile, bi, bj);
  const int Mp = m.Mp;
  const long pl = cplane(m);
  const _Float16* A = ws + m.g + jb.a * 2 * pl;
  const _Float16* B = ws + m.g + jb.b * 2 * pl;
  _Float16* C = ws + m.g + jb.c * 2 * pl;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
  Core core;
  core.run(smem, A + (long)bi * 64 * 16, 64, B + (long)bj * 64 * 16, 64, pl, Mp + 8, bi == bj && jb.a == jb.b, 0, Mp);
  const f32x16& acc = core.acc[0][0];
  const bool diag = bi == bj;
  const int j = wn + (lane & 31);
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int i = wm + 8 * q + 4 * (lane >> 5);
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = acc[4 * q + e] * jb.mul;
    if (jb.quad) {                                   // A[i][j] from A[j][i]: four neighbours
      const long at = cat(Mp, bj * 64 + j, bi * 64 + i);
      const half4 h = *reinterpret_cast<const half4*>(A + at), l = *reinterpret_cast<const half4*>(A + pl + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] += QUAD_B * ((float)h[e] + (float)l[e]);
        if (diag && i + e == j) v[e] += QUAD_A;
      }
    }
    half4 hh, ll;
#pragma unroll
    for (int e = 0; e < 4; ++e) { _Float16 h, l; split16(v[e], h, l); hh[e] = h; ll[e] = l; }
    char* at = smem + (i >> 4) * 2048 + j * 32 + (i & 15) * 2;       // [plane][block of i][64 rows j][16]
    *reinterpret_cast<half4*>(at) = hh;
    *reinterpret_cast<half4*>(at + 8192) = ll;
  }
  __syncthreads();
  const unsigned lds0 = (unsigned)(size_t)smem;
#pragma unroll
  for (int q = 0; q < 4; ++q) {                      // plane q >> 1
    const int x = (q & 1) * 256 + tid, blk = x >> 7, in = x & 127;
    *reinterpret_cast<uint4*>(C + (q >> 1) * pl + cat(Mp, bj * 64, bi * 64 + blk * 16) + in * 8) =
        *reinterpret_cast<const uint4*>(smem + (q >> 1) * 8192 + blk * 2048 + in * 16);
    if (diag) continue;
    // 16 lanes: 16 neighbours i, eight neighbours jc * 8 .. of each
    const int ib = lane >> 4, jc = (q & 1) * 4 + wave, l = lane & 15;
    half4 u, w;
    asm volatile("ds_read_b64_tr_b16 %0, %2\n\tds_read_b64_tr_b16 %1, %2 offset:128\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(u), "=&v"(w) : "v"(lds0 + (unsigned)((q >> 1) * 8192 + ib * 2048 + (jc * 8 + (l >> 2)) * 32 + (l & 3) * 8)) : "memory");
    *reinterpret_cast<half8*>(C + (q >> 1) * pl + cat(Mp, bi * 64 + ib * 16 + l, bj * 64 + jc * 8)) =
        __builtin_shufflevector(u, w, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

// Tiles of 32 x 32 (few matrices: at most two per CU).  Such a product is latency alone: launch, one round of transfers, a few dependent
// MFMAs.  A workgroup brings the whole of its rows (KC columns at a time, 128 KB for 512) in one go; each of its 4 waves moves and
// multiplies every fourth block, with no barrier before the sums are joined.  4.5 - 6 us for one 512 x 512 product
// (136 tiles; 64 x 64 tiles: 8.2 - 10 us).
template <int KC>
__global__ __launch_bounds__(256) void ns_chain32_kernel(const NsGroup gr, ChainJob j0, ChainJob j1, int total, int tiles, _Float16* ws) {
  constexpr int NB = KC / 64;                        // blocks per wave and round
  __shared__ __attribute__((aligned(1024))) char smem[4 * NB * 4096];
  const int t = xcd_tile(blockIdx.x, total, (total + 7) / 8);
  if (t < 0) return;
  const ChainJob jb = t >= tiles ? j1 : j0;
  const NsRef r = ns_find<F_JOIN>(gr, t >= tiles ? t - tiles : t);
  const NsMat& m = r.m;
  int bi, bj;
  tri(r.tile, bi, bj);
  const int Mp = m.Mp;
  const long pl = cplane(m);
  const _Float16* A = ws + m.g + jb.a * 2 * pl;
  const _Float16* B = ws + m.g + jb.b * 2 * pl;
  _Float16* C = ws + m.g + jb.c * 2 * pl;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool diag = bi == bj;
  const int row = lane >> 1;
  const long step = 64L * (Mp + 8);                  // four blocks
  const long own = (long)wave * 16 * (Mp + 8) + row * 16 + ((lane & 1) ^ swz(row)) * 8;
  const _Float16* pa = A + (long)bi * 32 * 16 + own;
  const _Float16* pb = B + (long)bj * 32 * 16 + own;
  // this wave's LDS: [block][A hi, A lo, B hi, B lo][32 rows][16]
  char* const base = smem + wave * (NB * 4096);
  const unsigned lds0 = (unsigned)(size_t)base + (lane & 31) * 32 + (((lane >> 5) ^ swz(lane & 31)) << 4);
  // the four values of A that a quadratic form needs, on their way early
  const int i = 8 * wave + 4 * (lane >> 5), j = lane & 31;
  half4 gh = {0, 0, 0, 0}, gl = {0, 0, 0, 0};
  if (jb.quad) {
    const long at = cat(Mp, bj * 32 + j, bi * 32 + i);
    gh = *reinterpret_cast<const half4*>(A + at);
    gl = *reinterpret_cast<const half4*>(A + pl + at);
  }
  f32x16 acc;
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] = 0.f;
  int left = Mp / 64;                                // blocks of this wave
  while (left > 0) {
    const int nb = min(left, NB);
    left -= nb;
#pragma unroll
    for (int u = 0; u < NB; ++u) {
      if (u >= nb) break;
      dma16(pa, base + u * 4096);
      dma16(pa + pl, base + u * 4096 + 1024);
      dma16(pb, base + u * 4096 + 2048);
      dma16(pb + pl, base + u * 4096 + 3 * 1024);
      pa += step; pb += step;
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int s = 0; s < NB; ++s) {                   // block s - (NB - nb): behind it 4 (NB - 1 - s) transfers are in flight
      const int u = s - (NB - nb);
      if (u < 0) continue;
      switch (NB - 1 - s) {
        case 7: wait_dma<28>(); break;
        case 6: wait_dma<24>(); break;
        case 5: wait_dma<20>(); break;
        case 4: wait_dma<16>(); break;
        case 3: wait_dma<12>(); break;
        case 2: wait_dma<8>(); break;
        case 1: wait_dma<4>(); break;
        default: wait_dma<0>(); break;
      }
      half8 a[2][1], b[2][1];
      const unsigned q = lds0 + u * 4096;
      fetch_nt<1024>(q, q + 2048, a, b);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0][0], b[0][0], acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0][0], b[1][0], acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[1][0], b[0][0], acc, 0, 0, 0);
    }
  }
  // sums of the four waves, in order: wave w finishes rows 8 w .. 8 w + 7
  __syncthreads();
  float4* buf = reinterpret_cast<float4*>(smem);
#pragma unroll
  for (int q = 0; q < 4; ++q) buf[(wave * 4 + q) * 64 + lane] = make_float4(acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]);
  __syncthreads();
  float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float4 f = buf[(w * 4 + wave) * 64 + lane];
    v[0] += f.x; v[1] += f.y; v[2] += f.z; v[3] += f.w;
  }
  const int gi = bi * 32 + i, gj = bj * 32 + j;
  half4 hh, ll;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] *= jb.mul;
    if (jb.quad) v[e] += QUAD_B * ((float)gh[e] + (float)gl[e]) + (gi + e == gj ? QUAD_A : 0.f);
    _Float16 h, l;
    split16(v[e], h, l);
    hh[e] = h; ll[e] = l;
    if (!diag) { C[cat(Mp, gi + e, gj)] = h; C[pl + cat(Mp, gi + e, gj)] = l; }
  }
  *reinterpret_cast<half4*>(C + cat(Mp, gj, gi)) = hh;
  *reinterpret_cast<half4*>(C + pl + cat(Mp, gj, gi)) = ll;
}

// ---------------------------------------------------------------------------------------------- X <- P X
// OUT: 0 = planes of the next stage, 1 = fp32 tensor, 2 = bf16 tensor, 3 = the step's update of p
struct ApplyK {
  const _Float16* wsx; const _Float16* wsg; _Float16* wso;
  int pbuf;
  const NsUnit* unit; int stage;
  float mul;
  void* out; long ldo;
  NsStep s;
};
// one K step of the apply product: 2 fragments of 32 rows of P, one of 32 columns of X; X (K step = 16 of its rows, [column / 16][16 rows][16]) through the
// transposing read: in a group of 16 lanes lane 4 r + c gives the address of four columns of row r and gets one column of four
// rows; two of them make a fragment.  Odd blocks hold their rows in the order 4..7 0..3 12..15 8..11, so that the two blocks a
// 32-lane half reads lie in different banks: the second read's address is the first one's ^ 128.
#define NS_TR "ds_read_b64_tr_b16 "
__device__ __forceinline__ void fetch_apply(unsigned pa, unsigned pb0, unsigned pb1, half8 (&a)[2][2], half4 (&b)[2][2]) {
  asm volatile(NS_RD "%0, %8\n\t" NS_TR "%4, %9\n\t" NS_TR "%5, %10\n\t" NS_RD "%1, %8 offset:1024\n\t"
               NS_RD "%2, %8 offset:4096\n\t" NS_RD "%3, %8 offset:5120\n\t" NS_TR "%6, %9 offset:4096\n\t" NS_TR "%7, %10 offset:4096\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(a[0][0]), "=&v"(a[0][1]), "=&v"(a[1][0]), "=&v"(a[1][1]),
                 "=&v"(b[0][0]), "=&v"(b[0][1]), "=&v"(b[1][0]), "=&v"(b[1][1])
               : "v"(pa), "v"(pb0), "v"(pb1) : "memory");
}
__device__ __forceinline__ void fetch_apply(unsigned pa, unsigned pb0, unsigned pb1, half8 (&a)[2][2], half4 (&b)[1][2]) {
  asm volatile(NS_RD "%0, %6\n\t" NS_TR "%4, %7\n\t" NS_TR "%5, %8\n\t" NS_RD "%1, %6 offset:1024\n\t"
               NS_RD "%2, %6 offset:4096\n\t" NS_RD "%3, %6 offset:5120\n\t" "s_waitcnt lgkmcnt(0)"
               : "=&v"(a[0][0]), "=&v"(a[0][1]), "=&v"(a[1][0]), "=&v"(a[1][1]), "=&v"(b[0][0]), "=&v"(b[0][1])
               : "v"(pa), "v"(pb0), "v"(pb1) : "memory");
}

// A tile is 128 rows x 128 columns, 8 waves (2 x 4) of 64 x 32; K steps of 16 through three stages: 48 KB, three workgroups per CU, so that reads,
// products and epilogues of different waves run under each other.  Bound by power (MFMAs busy for 44 - 47 % of the cycles; after a rest 257 and
// 273 us at 1.9 GHz): 310 - 320 us for each of the generator's two products (128 x 256 tiles, 4 waves of 128 x 64: 302 and 331 us), 512 x 24576 35 us (bf16 X)
// and 44 us (37 and 47 us), the discriminator's 18 and 19 us (29 and 35 us: 88 tiles).
__device__ __forceinline__ void muon_update(const NsStep& s, long at, float keep, float step, float o) {
  const float p = s.p[at] * keep - step * o;
  s.p[at] = p;
  if (s.pb) s.pb[at] = (bf16_t)(ns_pack_bf16(p, 0.f) & 0xffffu);
}
template <int PX, int OUT>
__global__ __launch_bounds__(512, 2) void ns_apply_kernel(const NsGroup gr, int total, int grp, const ApplyK k) {
  constexpr int TM = 2, NW = 8, IPP = AJ / 32;      // IPP: transfers per plane of X
  constexpr int A_BYTES = AI * 2 * 32, B_BYTES = 16 * AJ * 2 * PX, STAGE = A_BYTES + B_BYTES, ST = 3;
  // transfers per wave; 128 columns of one plane keep only the first four waves busy
  constexpr int PA = A_BYTES / 1024 / NW, PB = (B_BYTES / 1024 + NW - 1) / NW, NI = PA + PB;
  constexpr bool HALF = B_BYTES / 1024 < NW;
  __shared__ __attribute__((aligned(1024))) char smem[ST * STAGE];
  const int bt = xcd_tile(blockIdx.x, total, grp);
  if (bt < 0) return;
  const NsRef r = ns_find<F_APPLY>(gr, bt);
  const NsMat& m = r.m;
  const int ti = (m.Mp + AI - 1) / AI;
  const int i0 = (r.tile % ti) * AI, j0 = (r.tile / ti) * AJ;
  const NsUnit un = k.unit[r.id];
  const long pl = cplane(m), xpl = xplane(m);
  const _Float16* P = k.wsg + m.g + k.pbuf * 2 * pl;
  const _Float16* X = k.wsx + m.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = (wave >> 2) * 64, wn = (wave & 3) * 32;
  f32x16 acc[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[i][e] = 0.f;
  // P: 32 rows of a block per transfer; X: 16 rows of two blocks.  Rows and blocks behind the matrix read its last ones: products that
  // nobody stores.
  const _Float16* as[PA];
#pragma unroll
  for (int q = 0; q < PA; ++q) {
    const int row = (q * NW + wave) * 32 + (lane >> 1), plane = row / AI, lr = min(i0 + row - plane * AI, m.Mp - 1);
    as[q] = P + plane * pl + (long)lr * 16 + ((lane & 1) ^ swz(row)) * 8;
  }
  const _Float16* bs[PB];
#pragma unroll
  for (int q = 0; q < PB; ++q) {
    const int x = q * NW + wave, plane = x / IPP, blk = min((j0 >> 4) + x % IPP * 2 + (lane >> 5), m.Np / 16 - 1);
    const int kr = ((lane >> 1) & 15) ^ ((lane >> 5) << 2);
    bs[q] = X + plane * xpl + ((long)blk * (m.Mp + 8) + kr) * 16 + (lane & 1) * 8;
  }
  const long astep = 16L * (m.Mp + 8);
  auto issue = [&](int st) {
#pragma unroll
    for (int q = 0; q < PA; ++q) { dma16(as[q], smem + st * STAGE + (q * NW + wave) * 1024); as[q] += astep; }
#pragma unroll
    for (int q = 0; q < PB; ++q) {
      if (HALF && wave >= 4) break;
      dma16(bs[q], smem + st * STAGE + A_BYTES + (q * NW + wave) * 1024); bs[q] += 256;
    }
  };
  const unsigned lds0 = (unsigned)(size_t)smem;
  const int r4 = (lane >> 2) & 3, cq = lane & 3, mb = (lane >> 4) & 1, kh = lane >> 5;
  const unsigned pa = lds0 + (wm + (lane & 31)) * 32 + ((kh ^ swz(lane & 31)) << 4);
  const unsigned pb0 = lds0 + A_BYTES + ((wn >> 4) + mb) * 512 + (8 * kh + r4 + 4 * mb) * 32 + cq * 8, pb1 = pb0 ^ 128;
  const int n = m.Mp / 16;
  issue(0);
  issue(1);
  int cur = 0, nxt = 2;
  for (int it = 0; it < n; ++it) {
    if (it + 1 >= n) wait_dma<0>();
    else if (HALF && wave >= 4) wait_dma<PA>();
    else wait_dma<NI>();
    wg_barrier();
    if (it + 2 < n) issue(nxt);
    const unsigned so = (unsigned)(cur * STAGE);
    half8 a[2][TM];
    half4 bq[PX][2];
    fetch_apply(pa + so, pb0 + so, pb1 + so, a, bq);
    half8 b[PX];
#pragma unroll
    for (int p = 0; p < PX; ++p) b[p] = __builtin_shufflevector(bq[p][0], bq[p][1], 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      // the transposed product: a lane holds one row of the result and runs of four of its columns
      acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(b[0], a[0][i], acc[i], 0, 0, 0);
      acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(b[0], a[1][i], acc[i], 0, 0, 0);
      if constexpr (PX == 2) acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(b[1], a[0][i], acc[i], 0, 0, 0);
    }
    cur = cur == ST - 1 ? 0 : cur + 1;
    nxt = nxt == ST - 1 ? 0 : nxt + 1;
  }
  const float f = ns_value(un, k.stage) * (OUT == 0 ? ns_pow2(15 + ns_gap(un, k.stage + 1)) : 1.f) * k.mul;
  const float keep = 1.f - k.s.lr * k.s.wd, step = k.s.lr * m.scale;
  if (OUT != 0 && m.tall) {
    // the stored row is the long side: 32 neighbouring lanes hold 32 neighbours of a stored row
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int gi = i0 + wm + i * 32 + (lane & 31);
      if (gi >= m.M) continue;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int gj = j0 + wn + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
        if (gj >= m.N) continue;
        const float v = acc[i][e] * f;
        if constexpr (OUT == 1) reinterpret_cast<float*>(k.out)[r.out + (long)gj * k.ldo + gi] = v;
        else if constexpr (OUT == 2) reinterpret_cast<bf16_t*>(k.out)[r.out + (long)gj * k.ldo + gi] = (bf16_t)(ns_pack_bf16(v, 0.f) & 0xffffu);
        else muon_update(k.s, ns_at(m, gj, gi), keep, step, v);
      }
    }
    return;
  }
  // 32 rows per row of waves at a time through LDS (rows of AJ + 8 floats: both the writes and the reads meet every bank once): a wave then
  // handles whole rows, four neighbours per lane
  constexpr int BS = AJ + 8, RP = 64, LR = AJ / 4, NT = RP * LR / NW / 64;      // LR: lanes of a row; NT: runs of a lane
  float* buf = reinterpret_cast<float*>(smem);
  const int c = lane % LR * 4, gj = j0 + c;
  const long cbase = OUT == 3 && gj < m.N ? ns_at(m, 0, gj) : 0;
  // the row in the pass, and in the matrix, of a lane's t-th run
  auto prow = [&](int t) { return wave * (RP / NW) + t * (64 / LR) + lane / LR; };
  auto mrow = [&](int i, int r) { return i0 + (r >> 5) * 64 + i * 32 + (r & 31); };
  const bool four = gj + 4 <= m.N && (OUT != 3 || (m.cols & 3) == 0);
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    float4 p[NT];
    if constexpr (OUT == 3) {
      if (four) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int gi = mrow(i, prow(t));
          if (gi < m.M) {
            const NsU4 u = *reinterpret_cast<const NsU4*>(k.s.p + cbase + (long)gi * m.ld);
            p[t] = make_float4(__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w));
          }
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<float4*>(buf + ((wave >> 2) * 32 + (lane & 31)) * BS + wn + 8 * q + 4 * (lane >> 5)) =
          make_float4(acc[i][4 * q] * f, acc[i][4 * q + 1] * f, acc[i][4 * q + 2] * f, acc[i][4 * q + 3] * f);
    __syncthreads();
    if constexpr (OUT == 0) {
      // planes: blocks of 32 rows, 1 KB each
#pragma unroll
      for (int t = 0; t < RP / 32 * (AJ / 16) / NW; ++t) {
        const int k16 = t * NW + wave, blk = k16 % (AJ / 16), row = k16 / (AJ / 16) * 32 + (lane >> 1), col = blk * 16 + (lane & 1) * 8;
        const int gi = mrow(i, row);
        if (gi >= m.Mp || j0 + col >= m.Np) continue;
        const float4 u = *reinterpret_cast<const float4*>(buf + row * BS + col), w = *reinterpret_cast<const float4*>(buf + row * BS + col + 4);
        const float x[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
        half8 h, l;
#pragma unroll
        for (int e = 0; e < 8; ++e) { _Float16 th, tl; split16(x[e], th, tl); h[e] = th; l[e] = tl; }
        _Float16* o = k.wso + m.x + cat(m.Mp, gi, j0 + col);
        *reinterpret_cast<half8*>(o) = h;
        *reinterpret_cast<half8*>(o + xpl) = l;
      }
      continue;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int gi = mrow(i, prow(t));
      const float4 v = *reinterpret_cast<const float4*>(buf + prow(t) * BS + c);
      const float x[4] = {v.x, v.y, v.z, v.w};
      if (gi < m.M && four) {
        if constexpr (OUT == 3) {
          const long at = cbase + (long)gi * m.ld;
          const float y[4] = {p[t].x * keep - step * x[0], p[t].y * keep - step * x[1], p[t].z * keep - step * x[2], p[t].w * keep - step * x[3]};
          NsU4 u;
          u.x = __float_as_uint(y[0]); u.y = __float_as_uint(y[1]); u.z = __float_as_uint(y[2]); u.w = __float_as_uint(y[3]);
          *reinterpret_cast<NsU4*>(k.s.p + at) = u;
          if (k.s.pb) {
            NsU2 b;
            b.x = ns_pack_bf16(y[0], y[1]); b.y = ns_pack_bf16(y[2], y[3]);
            *reinterpret_cast<NsU2*>(k.s.pb + at) = b;
          }
        } else {
          const long at = r.out + (long)gi * k.ldo + gj;
          if constexpr (OUT == 1) {
            NsU4 u;
            u.x = __float_as_uint(x[0]); u.y = __float_as_uint(x[1]); u.z = __float_as_uint(x[2]); u.w = __float_as_uint(x[3]);
            *reinterpret_cast<NsU4*>(reinterpret_cast<float*>(k.out) + at) = u;
          } else {
            NsU2 b;
            b.x = ns_pack_bf16(x[0], x[1]); b.y = ns_pack_bf16(x[2], x[3]);
            *reinterpret_cast<NsU2*>(reinterpret_cast<bf16_t*>(k.out) + at) = b;
          }
        }
      } else if (gi < m.M) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (gj + e >= m.N) break;
          const long at = r.out + (long)gi * k.ldo + gj + e;
          if constexpr (OUT == 1) reinterpret_cast<float*>(k.out)[at] = x[e];
          else if constexpr (OUT == 2) reinterpret_cast<bf16_t*>(k.out)[at] = (bf16_t)(ns_pack_bf16(x[e], 0.f) & 0xffffu);
          else muon_update(k.s, ns_at(m, gi, gj + e), keep, step, x[e]);
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------- small matrices
// The chain of a matrix with a short side of at most MP (64, 128) in ONE workgroup: (MP / 32)^2 waves, each with one 32 x 32 block of every
// matrix in its registers; LDS buffers hold the operands of the products under way (fp16 pairs, [plane][block][MP rows][16]).
// A launch of the tiled form costs 5 us whatever its size, a product here 0.6 (64) to 1.2 us (128).
template <int MP>
struct SmallChain {
  static constexpr int W = MP / 32, BUF = MP * MP * 4, PS = MP * MP * 2;
  int lane, wi, wj;
  unsigned fa, fb;
  __device__ __forceinline__ SmallChain(int wave) {
    lane = threadIdx.x & 63; wi = wave / W; wj = wave % W;
    const int r = lane & 31;
    const unsigned off = (unsigned)(r * 32 + (((lane >> 5) ^ swz(r)) << 4));
    fa = (unsigned)(wi * 1024) + off; fb = (unsigned)(wj * 1024) + off;
  }
  // the transposed block of a symmetric matrix: four neighbours of a row at a time
  __device__ __forceinline__ void put(char* buf, const f32x16& v) const {
    const int row = wj * 32 + (lane & 31);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int col = wi * 32 + 8 * q + 4 * (lane >> 5);
      half4 h, l;
#pragma unroll
      for (int e = 0; e < 4; ++e) { _Float16 th, tl; split16(v[4 * q + e], th, tl); h[e] = th; l[e] = tl; }
      char* at = buf + ((col >> 4) * MP + row) * 32 + ((((col >> 3) & 1) ^ swz(row)) << 4) + (col & 7) * 2;
      *reinterpret_cast<half4*>(at) = h;
      *reinterpret_cast<half4*>(at + PS) = l;
    }
  }
  __device__ __forceinline__ f32x16 mul(const char* a, const char* b) const {
    f32x16 acc;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.f;
#pragma unroll
    for (int ks = 0; ks < MP / 16; ++ks) {
      const half8 x0 = *reinterpret_cast<const half8*>(a + fa + ks * (MP * 32)), x1 = *reinterpret_cast<const half8*>(a + fa + ks * (MP * 32) + PS);
      const half8 y0 = *reinterpret_cast<const half8*>(b + fb + ks * (MP * 32)), y1 = *reinterpret_cast<const half8*>(b + fb + ks * (MP * 32) + PS);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(x0, y0, acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(x0, y1, acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(x1, y0, acc, 0, 0, 0);
    }
    return acc;
  }
  // q = a I + b G + c G^2, G's block in g and all of it in `buf`
  __device__ __forceinline__ f32x16 quad(const f32x16& g, const char* buf) const {
    f32x16 q = mul(buf, buf);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      q[e] = q[e] * QUAD_C + QUAD_B * g[e];
      if (wi == wj && 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3) == (lane & 31)) q[e] += QUAD_A;
    }
    return q;
  }
  static __device__ __forceinline__ float pscale(int k) { return 1.f / (float)(1 << (k == 1 ? 2 * SQ - SP : SQ)); }

  // g: this wave's block of G (scale 2^SG).  Returns its block of P, scale 2^(steps > 1 ? SP : SQ).  Every wave of the workgroup calls it;
  // a product begins when both operands are in LDS and its result goes where nobody reads any more.
  // Two buffers: one group of waves.
  __device__ __forceinline__ f32x16 run2(f32x16 g, int steps, char* b1, char* b2) const {
    const float q1 = 1.f / (float)(1 << SQ);
    f32x16 P, y;
    __syncthreads();
    put(b1, g);
    __syncthreads();
    for (int k = 0; k < steps; ++k) {
      const bool more = k + 1 < steps;
      const f32x16 q = quad(g, b1);
      put(b2, q);
      __syncthreads();
      if (more) y = mul(b2, b1) * q1;
      if (k == 0) {
        P = q;
      } else {
        __syncthreads();
        put(b1, P);
        __syncthreads();
        P = mul(b2, b1) * pscale(k);
      }
      if (more) {
        __syncthreads();
        put(b1, y);
        __syncthreads();
        g = mul(b2, b1) * q1;
        __syncthreads();
        put(b1, g);
        __syncthreads();
      }
    }
    return P;
  }
  // Four buffers and two groups of waves (grp): the first one follows G, the second one P; three barriers a step.  P is group
  // (steps > 1)'s; g is group 0's.
  __device__ __forceinline__ f32x16 run4(int grp, f32x16 g, int steps, char* b) const {
    const float q1 = 1.f / (float)(1 << SQ);
    char *const bg = b, *const bq = b + BUF, *const by = b + 2 * BUF, *const bp = b + 3 * BUF;
    f32x16 P;
#pragma unroll
    for (int e = 0; e < 16; ++e) P[e] = 0.f;
    __syncthreads();
    if (grp == 0) put(bg, g);
    __syncthreads();
    for (int k = 0; k < steps; ++k) {
      if (grp == 0) {
        const f32x16 q = quad(g, bg);
        put(bq, q);
        if (k == 0) { P = q; put(bp, q); }
      }
      __syncthreads();
      const bool more = k + 1 < steps;
      if (grp == 0) {
        if (more) put(by, mul(bq, bg) * q1);
      } else if (k > 0) {
        P = mul(bq, bp) * pscale(k);
      }
      if (!more) break;
      __syncthreads();
      if (grp == 0) {
        g = mul(bq, by) * q1;
        put(bg, g);
      } else if (k > 0) {
        put(bp, P);
      }
      __syncthreads();
    }
    return P;
  }
};

// the join of the Gram slices and the whole chain of one stage: one workgroup per matrix, P to buffer 3
template <int MP>
__global__ __launch_bounds__(MP * 8) void ns_chain_small_kernel(const NsGroup gr, const float* part, const NsUnit* unit, int stage,
                                                                                  int steps, _Float16* ws) {
  typedef SmallChain<MP> Sc;
  __shared__ __attribute__((aligned(1024))) char smem[(MP == 64 ? 4 : 2) * Sc::BUF];
  const int id = blockIdx.x, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int grp = wave / (Sc::W * Sc::W);            // 64: two groups of waves; 128: one
  NsMat m = gr.tab ? gr.tab[id] : gr.u;
  if (m.kind == 1) return;
  if (!gr.tab) { m.g += (long)id * gr.g_step; m.part += (long)id * gr.part_step; }
  const Sc sc(wave % (Sc::W * Sc::W));
  const int frag = ((sc.wi >> 1) * 2 + (sc.wj >> 1)) * 4 + (sc.wi & 1) * 2 + (sc.wj & 1);
  const float4* src = reinterpret_cast<const float4*>(part + m.part) + frag * 256 + lane;
  const float c1 = ns_value(unit[id], stage);
  const float c2 = c1 * c1 * (float)(1 << SG);
  f32x16 g;
#pragma unroll
  for (int e = 0; e < 16; ++e) g[e] = 0.f;
  if (grp == 0 && sc.wi * 32 < m.Mp && sc.wj * 32 < m.Mp) {
#pragma unroll 4
    for (int s = 0; s < m.ks; ++s)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 f = src[(long)s * (GT * GT / 4) + q * 64];
        g[4 * q] += f.x; g[4 * q + 1] += f.y; g[4 * q + 2] += f.z; g[4 * q + 3] += f.w;
      }
    g = g * c2;
  }
  f32x16 P;
  if constexpr (MP == 64) P = sc.run4(grp, g, steps, smem);
  else P = sc.run2(g, steps, smem, smem + Sc::BUF);
  const int row = sc.wj * 32 + (lane & 31);
  if (sc.wi * 32 >= m.Mp || sc.wj * 32 >= m.Mp || (MP == 64 && grp != (steps > 1))) return;
  const long pl = cplane(m);
  _Float16* out = ws + m.g + 6 * pl;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    half4 h, l;
#pragma unroll
    for (int e = 0; e < 4; ++e) { _Float16 th, tl; split16(P[4 * q + e], th, tl); h[e] = th; l[e] = tl; }
    _Float16* at = out + cat(m.Mp, row, sc.wi * 32 + 8 * q + 4 * (lane >> 5));
    *reinterpret_cast<half4*>(at) = h;
    *reinterpret_cast<half4*>(at + pl) = l;
  }
}

// the transposing read (fetch_apply) where no transfer is in flight: the compiler places its wait
__device__ __forceinline__ half4 lds_tr(const char* p) {
  typedef __fp16 tr4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) tr4*)p));
}

// Everything in one launch for matrices of at most 64 x NX: X stays in LDS from the first load to the result.  8 waves: the Gram product
// divides the columns among two groups of four, the chain takes four waves, P X goes by strips of 32 columns, in place.
template <int NX, int SRC, int OUT>
__global__ __launch_bounds__(512) void ns_small_kernel(const NsMat m, const void* x, long src_step, void* outp, long out_step, long ldo, int steps, float eps) {
  constexpr int XP = NX * 64 * 2;                     // bytes of a plane: [NX / 16][64 rows][16]
  typedef SmallChain<64> Sc;
  __shared__ __attribute__((aligned(1024))) char smem[2 * XP + 4 * Sc::BUF];         // 64 x 384: all of the CU's 160 KB
  char* const X = smem;
  char* const b1 = smem + 2 * XP;
  NsNorm* const red = reinterpret_cast<NsNorm*>(b1);                // before the first product: of each wave
  NsUnit& unit = *reinterpret_cast<NsUnit*>(b1 + 8 * sizeof(NsNorm));
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  NsMat mm = m;
  mm.src += (long)blockIdx.x * src_step;
  const NsStep none{};
  // runs of eight stored neighbours: at most 64 x NX / 8
  constexpr int RUNS = 64 * NX / 8 / 512;
  const int rpr = (m.cols + 7) / 8, nrun = m.rows * rpr;
  float v[RUNS][8];
  double a = 0.0;
  float top = 0.f;
#pragma unroll
  for (int t = 0; t < RUNS; ++t) {
    const int c = t * 512 + tid;
    if (c < nrun) {
      const int row = c / rpr;
      ns_load8<SRC>(mm, x, none, row, (c - row * rpr) * 8, v[t]);
#pragma unroll
      for (int e = 0; e < 8; ++e) { a = fma((double)v[t][e], (double)v[t][e], a); top = fmaxf(top, fabsf(v[t][e])); }
    }
  }
#pragma unroll
  for (int t = 0; t < 2 * XP / 16 / 512; ++t) *reinterpret_cast<uint4*>(X + (t * 512 + tid) * 16) = make_uint4(0u, 0u, 0u, 0u);
  a = wave_sum_d(a);
  top = wave_max(top);
  if (lane == 0) { red[wave].sum = a; red[wave].top = top; }
  __syncthreads();
  a = 0.0;
#pragma unroll
  for (int w = 0; w < 8; ++w) { a += red[w].sum; top = fmaxf(top, red[w].top); }
  const int k = ns_exponent(top);
  const float f = ns_pow2(-k);
  if (tid == 511) unit = ns_unit_of(a, k, eps);
#pragma unroll
  for (int t = 0; t < RUNS; ++t) {
    const int c = t * 512 + tid;
    if (c >= nrun) continue;
    const int row = c / rpr, col = (c - row * rpr) * 8;
    half8 h, l;
#pragma unroll
    for (int e = 0; e < 8; ++e) { _Float16 th, tl; split16(v[t][e] * f, th, tl); h[e] = th; l[e] = tl; }
    if (!m.tall) {
      char* at = X + ((col >> 4) * 64 + row) * 32 + ((((col >> 3) & 1) ^ swz(row)) << 4);
      *reinterpret_cast<half8*>(at) = h;
      *reinterpret_cast<half8*>(at + XP) = l;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = col + e, j = row;
        if (i >= m.M) break;
        _Float16* at = reinterpret_cast<_Float16*>(X + ((j >> 4) * 64 + i) * 32 + ((((j >> 3) & 1) ^ swz(i)) << 4) + (j & 7) * 2);
        at[0] = h[e];
        at[XP / 2] = l[e];
      }
    }
  }
  const bool on = wave < 4;
  const Sc sc(wave & 3);
  const int r4 = (lane >> 2) & 3, cq = lane & 3, mb = (lane >> 4) & 1, kh = lane >> 5;
  const int nblk = m.Np / 16;
  __syncthreads();
  const NsUnit un = unit;
  for (int stage = 0; steps > 0; ++stage) {
    const float c1 = ns_value(un, stage);
    const int ns = steps < 3 ? steps : 3;
    steps -= ns;
    __syncthreads();
    f32x16 g;
#pragma unroll
    for (int e = 0; e < 16; ++e) g[e] = 0.f;
#pragma unroll 2
    for (int b = wave >> 2; b < nblk; b += 2) {
      const char* at = X + b * 2048;
      const half8 p0 = *reinterpret_cast<const half8*>(at + sc.fa), p1 = *reinterpret_cast<const half8*>(at + sc.fa + XP);
      const half8 q0 = *reinterpret_cast<const half8*>(at + sc.fb), q1 = *reinterpret_cast<const half8*>(at + sc.fb + XP);
      g = __builtin_amdgcn_mfma_f32_32x32x16_f16(p0, q0, g, 0, 0, 0);
      g = __builtin_amdgcn_mfma_f32_32x32x16_f16(p0, q1, g, 0, 0, 0);
      g = __builtin_amdgcn_mfma_f32_32x32x16_f16(p1, q0, g, 0, 0, 0);
    }
    float4* buf = reinterpret_cast<float4*>(b1);
    if (!on) {
#pragma unroll
      for (int q = 0; q < 4; ++q) buf[((wave - 4) * 4 + q) * 64 + lane] = make_float4(g[4 * q], g[4 * q + 1], g[4 * q + 2], g[4 * q + 3]);
    }
    __syncthreads();
    if (on) {
      const float c2 = c1 * c1 * (float)(1 << SG);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 u = buf[(wave * 4 + q) * 64 + lane];
        g[4 * q] = (g[4 * q] + u.x) * c2; g[4 * q + 1] = (g[4 * q + 1] + u.y) * c2;
        g[4 * q + 2] = (g[4 * q + 2] + u.z) * c2; g[4 * q + 3] = (g[4 * q + 3] + u.w) * c2;
      }
    }
    const f32x16 P = sc.run4(wave >> 2, g, ns, b1);
    __syncthreads();
    if ((wave >> 2) == (ns > 1)) sc.put(b1, P);
    __syncthreads();
    const bool last = steps == 0;
    const float mul = c1 * (last ? 1.f : ns_pow2(15 + ns_gap(un, stage + 1))) * (ns > 1 ? 1.f / (float)(1 << SP) : 1.f / (float)(1 << SQ));
    for (int s = wave; s < m.Np / 32; s += 8) {       // a strip of 32 columns: all of its rows are this wave's
      f32x16 acc[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        half8 p[2][2];
        const int r = lane & 31;
        const char* pa = b1 + ks * 2048 + r * 32 + ((kh ^ swz(r)) << 4);
        const char* pb = X + (s * 2 + mb) * 2048 + (ks * 16 + 8 * kh + r4) * 32 + (((cq >> 1) ^ kh) << 4) + (cq & 1) * 8;
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i >> 1][i & 1] = *reinterpret_cast<const half8*>(pa + (i >> 1) * Sc::PS + (i & 1) * 1024);
        const half8 y0 = __builtin_shufflevector(lds_tr(pb), lds_tr(pb + 128), 0, 1, 2, 3, 4, 5, 6, 7);
        const half8 y1 = __builtin_shufflevector(lds_tr(pb + XP), lds_tr(pb + XP + 128), 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(y0, p[0][i], acc[i], 0, 0, 0);
          acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(y0, p[1][i], acc[i], 0, 0, 0);
          acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(y1, p[0][i], acc[i], 0, 0, 0);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = i * 32 + (lane & 31);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int col = s * 32 + 8 * q + 4 * kh;
          float o[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = acc[i][4 * q + e] * mul;
          if (!last) {
            half4 h, l;
#pragma unroll
            for (int e = 0; e < 4; ++e) { _Float16 th, tl; split16(o[e], th, tl); h[e] = th; l[e] = tl; }
            char* at = X + ((col >> 4) * 64 + row) * 32 + ((((col >> 3) & 1) ^ swz(row)) << 4) + (col & 7) * 2;
            *reinterpret_cast<half4*>(at) = h;
            *reinterpret_cast<half4*>(at + XP) = l;
          } else if (row < m.M) {
            if (!m.tall && col + 4 <= m.N) {
              const long at = (long)blockIdx.x * out_step + (long)row * ldo + col;
              if constexpr (OUT == 1) {
                NsU4 u;
                u.x = __float_as_uint(o[0]); u.y = __float_as_uint(o[1]); u.z = __float_as_uint(o[2]); u.w = __float_as_uint(o[3]);
                *reinterpret_cast<NsU4*>(reinterpret_cast<float*>(outp) + at) = u;
              } else {
                NsU2 u;
                u.x = ns_pack_bf16(o[0], o[1]); u.y = ns_pack_bf16(o[2], o[3]);
                *reinterpret_cast<NsU2*>(reinterpret_cast<bf16_t*>(outp) + at) = u;
              }
              continue;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (col + e >= m.N) break;
              const long at = (long)blockIdx.x * out_step + (m.tall ? (long)(col + e) * ldo + row : (long)row * ldo + col + e);
              if constexpr (OUT == 1) reinterpret_cast<float*>(outp)[at] = o[e];
              else reinterpret_cast<bf16_t*>(outp)[at] = (bf16_t)(ns_pack_bf16(o[e], 0.f) & 0xffffu);
            }
          }
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------- host side
static long up(long a, long b) { return (a + b - 1) / b * b; }

struct NsPlan {
  NsGroup gr;
  std::vector<NsMat> mats;      // the table's content (empty: equal matrices)
  std::vector<int> first;       // [F_N][n]
  long n[F_N];                  // workgroups per launch
  int top;                      // largest padded short side
  long off_tab, off_first, off_c, off_sq, off_x, x_halves, off_g, off_part, bytes;
};

// sizes and workgroup counts of one matrix; false: a side or a product of sides out of range
static bool ns_shape(NsMat& m) {
  const long rows = m.rows, cols = (long)m.taps * m.cols;
  if (rows * cols > 0x7fffffffL) return false;
  m.tall = rows > cols;
  const long Mp = up(m.tall ? cols : rows, 64), Np = up(m.tall ? rows : cols, 64);
  if (Mp * Np > 0x7fffffffL) return false;           // also: Np fits an int
  m.M = (int)(m.tall ? cols : rows);
  m.N = (int)(m.tall ? rows : cols);
  m.Mp = (int)Mp;
  m.Np = (int)Np;
  return true;
}
struct NsCounts { long n[F_N], x, g, part; };
// ks: slices of the long side in the Gram product
static NsCounts ns_counts(NsMat& m, long ks, bool flat) {
  NsCounts c{};
  const long n = (long)m.taps * m.rows * m.cols;
  c.n[F_MOM] = flat ? cdiv(n, k0_elems(n)) : cdiv((long)m.rows * cdiv(m.cols, 8), sq_runs((long)m.rows * cdiv(m.cols, 8)));
  m.np = (int)c.n[F_MOM];
  if (m.kind == 1) return c;
  c.n[F_SPLIT] = m.tall ? (long)(m.Mp / 64) * (m.Np / 64) : (long)(m.Mp / 64) * cdiv(m.Np, 128);
  const long nt = cdiv(m.Mp, GT), ntri = nt * (nt + 1) / 2;
  m.ks = ks < 1 ? 1 : ks > m.Np / 256 ? (m.Np < 256 ? 1 : m.Np / 256) : (int)ks;
  m.kc = (int)up(cdiv(m.Np, m.ks), 32);
  m.ks = cdiv(m.Np, m.kc);
  c.n[F_GRAM] = ntri * m.ks;
  const long n64 = m.Mp / 64, n32 = m.Mp / 32;
  c.n[F_CHAIN] = n64 * (n64 + 1) / 2;
  c.n[F_JOIN] = n32 * (n32 + 1) / 2;
  c.n[F_APPLY] = (long)cdiv(m.Mp, AI) * cdiv(m.Np, AJ);
  c.x = 2L * m.Np * (m.Mp + 8);
  c.g = 10L * m.Mp * (m.Mp + 8);
  c.part = c.n[F_GRAM] * GT * GT;
  return c;
}
// Gram tiles of a matrix times its length: the unit in which the long side is divided
static long ns_gram_work(const NsMat& m) {
  const long nt = cdiv(m.Mp, GT);
  return nt * (nt + 1) / 2 * m.Np;
}
static void ns_place(NsPlan& pl, int nmat, long nx, long ng, long npart) {
  auto take = [&](long& off, long bytes) { off = pl.bytes; pl.bytes += up(bytes, 256); };
  pl.bytes = 0;
  take(pl.off_tab, (long)pl.mats.size() * (long)sizeof(NsMat));
  take(pl.off_first, (long)pl.first.size() * 4);
  take(pl.off_c, (long)nmat * (long)sizeof(NsUnit));
  take(pl.off_sq, pl.n[F_MOM] * (long)sizeof(NsNorm));
  pl.x_halves = up(nx, 128);
  take(pl.off_x, pl.x_halves * 2 * 2);               // two sets of planes: X and its successor
  take(pl.off_g, ng * 2);
  take(pl.off_part, npart * 4);
}

// workgroups of a Gram launch that run at once: two per CU
constexpr long GRAM_SLOTS = 512;

// a launch has less than 2^32 lanes: at most this many workgroups of 256 (the chain's launches have two per tile)
constexpr long MAX_GROUPS = 1L << 22;
// A batch goes in pieces whose workspace stays below 2 GB (padded planes of many thin matrices take far more than the matrices): a
// piece of that size runs for milliseconds, its twenty launches cost 0.1 ms.
constexpr long PIECE_BYTES = 2L << 30;

// the plan of `piece` of the batch's matrices
static const char* ns_plan_batch(NsPlan& pl, long batch, long rows, long cols, long sx, long ldx, long so, long& piece) {
  NsMat m{};
  m.taps = 1; m.rows = (int)rows; m.cols = (int)cols; m.ld = ldx; m.st = 0;
  if (!ns_shape(m)) return "a matrix has more than 2^31 - 1 elements (sides rounded up to 64)";
  const long nt = cdiv(m.Mp, GT);
  const NsCounts c = ns_counts(m, GRAM_SLOTS / (nt * (nt + 1) / 2 * batch), false);
  long most = 1;
  for (int f = 0; f < F_N; ++f) most = c.n[f] > most ? c.n[f] : most;
  if (most > MAX_GROUPS) return "a matrix is too large";
  const long fit = PIECE_BYTES / (c.x * 4 + c.g * 2 + c.part * 4);
  piece = MAX_GROUPS / most < fit ? MAX_GROUPS / most : fit < 1 ? 1 : fit;
  if (piece > batch) piece = batch;
  pl.top = m.Mp;
  pl.gr.tab = nullptr;
  pl.gr.u = m;
  pl.gr.src_step = sx; pl.gr.out_step = so; pl.gr.x_step = c.x; pl.gr.g_step = c.g; pl.gr.part_step = c.part;
  for (int f = 0; f < F_N; ++f) {
    pl.gr.per[f] = (int)c.n[f];
    pl.n[f] = c.n[f] * piece;
  }
  ns_place(pl, (int)piece, c.x * piece, c.g * piece, c.part * piece);
  return nullptr;
}

constexpr int MAX_ENTRIES = 1 << 16;
static const char* ns_plan_table(NsPlan& pl, const pg_muon_entry_t* e, int n) {
  if (n > MAX_ENTRIES) return "more than 65536 tensors";
  try {                                              // no exception leaves a C entry
    pl.mats.resize((size_t)n);
    pl.first.resize((size_t)n * F_N);
  } catch (const std::bad_alloc&) {
    return "out of host memory";
  }
  long work = 0;
  for (int i = 0; i < n; ++i) {
    NsMat& m = pl.mats[(size_t)i];
    m = NsMat{};
    if (e[i].taps <= 0 || e[i].rows <= 0 || e[i].cols <= 0 || e[i].off < 0 || (e[i].kind != 0 && e[i].kind != 1)) return "an entry with a size <= 0, a negative offset or an unknown kind";
    m.src = e[i].off; m.taps = e[i].taps; m.rows = e[i].rows; m.cols = e[i].cols; m.kind = e[i].kind; m.scale = e[i].scale;
    m.ld = m.cols; m.st = (long)m.rows * m.cols;
    if ((long)m.taps * m.rows > 0x7fffffffL || (long)m.taps * m.rows * m.cols > 0x7fffffffL) return "a tensor has more than 2^31 - 1 elements";
    if (m.kind == 0) {
      if (!ns_shape(m)) return "a matrix has more than 2^31 - 1 elements (sides rounded up to 64)";
      work += ns_gram_work(m);
      if (m.Mp > pl.top) pl.top = m.Mp;
    }
  }
  long x = 0, g = 0, part = 0;
  for (int i = 0; i < n; ++i) {
    NsMat& m = pl.mats[(size_t)i];
    // a matrix gets workgroups in proportion to its work, rounded down: all slices run at once, and no second round begins for a few
    const long nt = cdiv(m.Mp, GT), share = m.kind == 0 ? GRAM_SLOTS * ns_gram_work(m) / work / (nt * (nt + 1) / 2) : 0;
    const NsCounts c = ns_counts(m, share, true);
    m.sq0 = (int)pl.n[F_MOM];
    m.x = x; m.g = g; m.part = part;
    x += c.x; g += c.g; part += c.part;
    for (int f = 0; f < F_N; ++f) {
      pl.first[(size_t)(f * n + i)] = (int)pl.n[f];
      pl.n[f] += c.n[f];
      if (pl.n[f] > MAX_GROUPS) return "too many tensors for one call";
    }
  }
  ns_place(pl, n, x, g, part);
  pl.gr.n = n;
  return nullptr;
}

struct NsSource { int kind; const void* x; };      // kind: ns_elem's SRC

// everything behind the sums of squares.  out_kind: ns_apply_kernel's OUT of the last product
static void ns_run(const NsPlan& pl, char* w, const NsSource& in, const NsStep& step, int steps, float eps, int out_kind, void* out,
                   long ldo, hipStream_t st) {
  const NsGroup& gr = pl.gr;
  NsUnit* unit = reinterpret_cast<NsUnit*>(w + pl.off_c);
  const NsNorm* sq = reinterpret_cast<const NsNorm*>(w + pl.off_sq);
  _Float16* xin = reinterpret_cast<_Float16*>(w + pl.off_x);
  _Float16* xout = xin + pl.x_halves;
  _Float16* g = reinterpret_cast<_Float16*>(w + pl.off_g);
  float* part = reinterpret_cast<float*>(w + pl.off_part);
  const dim3 blk(256);
  auto tri_tiles = [&](int t) { const int n = cdiv(pl.top, t); return n * (n + 1) / 2; };      // of the largest matrix
  if (in.kind == 0) PG_KLAUNCH((ns_split_kernel<0>), dim3((unsigned)pl.n[F_SPLIT]), blk, 0, st, gr, in.x, step, sq, eps, unit, xin);
  else if (in.kind == 1) PG_KLAUNCH((ns_split_kernel<1>), dim3((unsigned)pl.n[F_SPLIT]), blk, 0, st, gr, in.x, step, sq, eps, unit, xin);
  else PG_KLAUNCH((ns_split_kernel<2>), dim3((unsigned)pl.n[F_SPLIT]), blk, 0, st, gr, in.x, step, sq, eps, unit, xin);
  for (int stage = 0; steps > 0; ++stage) {
    const int ns = steps < 3 ? steps : 3;
    steps -= ns;
    const bool last = steps == 0;
    const bool one = stage == 0 && in.kind == 1;
    if (one) PG_KLAUNCH((ns_gram_kernel<1>), dim3((unsigned)up(pl.n[F_GRAM], 8)), blk, 0, st, gr, (int)pl.n[F_GRAM], tri_tiles(GT), (const _Float16*)xin, part);
    else PG_KLAUNCH((ns_gram_kernel<2>), dim3((unsigned)up(pl.n[F_GRAM], 8)), blk, 0, st, gr, (int)pl.n[F_GRAM], tri_tiles(GT), (const _Float16*)xin, part);
    // buffers: 0 G, 1 Q, 2 Q G, 3 and 4 P in turn; the first step's Q is the first P (and keeps Q's scale)
    const float q1 = 1.f / (float)(1 << SQ);
    int p = 3, psc = SQ;
    const bool many = pl.n[F_JOIN] > 512;
    const int nc = (int)pl.n[many ? F_CHAIN : F_JOIN];
    if (pl.top <= 128) {
      const dim3 gm((unsigned)gr.n);
      if (pl.top == 64) PG_KLAUNCH((ns_chain_small_kernel<64>), gm, dim3(512), 0, st, gr, (const float*)part, (const NsUnit*)unit, stage, ns, g);
      else PG_KLAUNCH((ns_chain_small_kernel<128>), gm, dim3(1024), 0, st, gr, (const float*)part, (const NsUnit*)unit, stage, ns, g);
      psc = ns > 1 ? SP : SQ;
    } else {
      PG_KLAUNCH(ns_gram_join_kernel, dim3((unsigned)pl.n[F_JOIN]), blk, 0, st, gr, (const float*)part, (const NsUnit*)unit, stage, g);
      auto chain = [&](const ChainJob& a, const ChainJob* b) {
        const int total = b ? 2 * nc : nc;
        const dim3 gd((unsigned)up(total, 8));
        const ChainJob b1 = b ? *b : a;
        if (many) PG_KLAUNCH(ns_chain_kernel, gd, blk, 0, st, gr, a, b1, total, nc, tri_tiles(64), g);
        // all tiles run at once: 1, 2 or 5 workgroups to a CU by their LDS, fewer columns at a time (two jobs of 184 tiles: 9.4 us in
        // two turns of 512 columns, 7.4 us in one with 256; of 336 tiles: 9.3 us with 256, 5.8 us with 128)
        else if (total > 512) PG_KLAUNCH((ns_chain32_kernel<128>), gd, blk, 0, st, gr, a, b1, total, nc, g);
        else if (pl.top <= 256 || total > 256) PG_KLAUNCH((ns_chain32_kernel<256>), gd, blk, 0, st, gr, a, b1, total, nc, g);
        else PG_KLAUNCH((ns_chain32_kernel<512>), gd, blk, 0, st, gr, a, b1, total, nc, g);
      };
      for (int k = 0; k < ns; ++k) {
        const int q = k == 0 ? 3 : 1;
        const ChainJob quad = {0, 0, q, QUAD_C, 1};
        const ChainJob qg = {q, 0, 2, q1, 0}, qp = {q, p, 7 - p, (float)ldexp(1.0, SP - SQ - psc), 0}, qqg = {q, 2, 0, q1, 0};
        const bool more = k + 1 < ns;
        chain(quad, nullptr);
        if (more) chain(qg, k > 0 ? &qp : nullptr);
        else if (k > 0) chain(qp, nullptr);
        if (more) chain(qqg, nullptr);
        if (k > 0) { p = 7 - p; psc = SP; }
      }
    }
    ApplyK a;
    memset(&a, 0, sizeof(a));
    a.wsx = xin; a.wsg = g; a.wso = xout; a.pbuf = p;
    a.unit = unit; a.stage = stage;
    a.mul = (float)ldexp(1.0, -psc);
    a.out = out; a.ldo = ldo; a.s = step;
    const int o = last ? out_kind : 0;
    const int na = (int)pl.n[F_APPLY];
    const dim3 gd((unsigned)up(na, 8));
#define NS_APPLY(PX, O) PG_KLAUNCH((ns_apply_kernel<PX, O>), gd, dim3(512), 0, st, gr, na, cdiv(pl.top, AI), a)
    if (one) {
      if (o == 0) NS_APPLY(1, 0);
      else if (o == 1) NS_APPLY(1, 1);
      else NS_APPLY(1, 2);
    } else {
      if (o == 0) NS_APPLY(2, 0);
      else if (o == 1) NS_APPLY(2, 1);
      else if (o == 2) NS_APPLY(2, 2);
      else NS_APPLY(2, 3);
    }
#undef NS_APPLY
    _Float16* t = xin; xin = xout; xout = t;
  }
}

}  // namespace pg

using namespace pg;

namespace pg {
// the one-launch form: short side <= 64, long side <= 384
static bool ns_is_small(int64_t rows, int64_t cols) { return (rows < cols ? rows : cols) <= 64 && (rows < cols ? cols : rows) <= 384; }
template <int SRC, int OUT>
static void ns_small(const NsMat& m, const void* x, long xs, void* out, long os, long ldo, int steps, float eps, unsigned batch, hipStream_t st) {
  if (m.Np <= 64) PG_KLAUNCH((ns_small_kernel<64, SRC, OUT>), dim3(batch), dim3(512), 0, st, m, x, xs, out, os, ldo, steps, eps);
  else if (m.Np <= 192) PG_KLAUNCH((ns_small_kernel<192, SRC, OUT>), dim3(batch), dim3(512), 0, st, m, x, xs, out, os, ldo, steps, eps);
  else PG_KLAUNCH((ns_small_kernel<384, SRC, OUT>), dim3(batch), dim3(512), 0, st, m, x, xs, out, os, ldo, steps, eps);
}
}  // namespace pg

extern "C" int64_t pg_orthogonalise_workspace(int64_t batch, int64_t rows, int64_t cols) {
  if (batch <= 0 || rows <= 0 || cols <= 0) return 0;
  if (batch > 0x3fffffff || rows > 0x7fffffff || cols > 0x7fffffff) return -1;
  if (ns_is_small(rows, cols)) return 0;
  NsPlan pl{};
  long piece;
  return ns_plan_batch(pl, batch, rows, cols, 0, cols, 0, piece) ? -1 : pl.bytes;
}

extern "C" int pg_orthogonalise(const void* x, int32_t x_is_bf16, int64_t batch, int64_t rows, int64_t cols, int64_t x_batch, int64_t ldx,
                                void* out, int32_t out_is_bf16, int64_t out_batch, int64_t ldo, int32_t steps, float eps,
                                void* workspace, int64_t workspace_bytes, void* stream) {
  PG_REQUIRE(batch >= 0 && rows >= 0 && cols >= 0, "pg_orthogonalise: batch, rows and cols must not be negative");
  if (batch == 0 || rows == 0 || cols == 0) return 0;
  PG_REQUIRE(x && out && ldx >= cols && ldo >= cols, "pg_orthogonalise: x, out, ldx >= cols and ldo >= cols required");
  PG_REQUIRE(batch == 1 || (x_batch >= 0 && out_batch >= (rows - 1) * ldo + cols), "pg_orthogonalise: output matrices of the batch overlap");
  PG_REQUIRE(steps >= 1 && steps <= 32, "pg_orthogonalise: steps 1..32");
  PG_REQUIRE(eps > 0.f, "pg_orthogonalise: eps > 0 required");
  PG_REQUIRE(((size_t)x & (x_is_bf16 ? 1 : 3)) == 0 && ((size_t)out & (out_is_bf16 ? 1 : 3)) == 0 && ((size_t)workspace & 255) == 0,
             "pg_orthogonalise: x / out aligned to their element, workspace to 256 bytes");
  PG_REQUIRE(batch <= 0x3fffffff && rows <= 0x7fffffff && cols <= 0x7fffffff, "pg_orthogonalise: sizes out of range");
  if (ns_is_small(rows, cols)) {
    NsMat m{};
    m.taps = 1; m.rows = (int)rows; m.cols = (int)cols; m.ld = (long)ldx;
    ns_shape(m);
    hipStream_t st = (hipStream_t)stream;
    for (int64_t b = 0; b < batch; b += MAX_GROUPS) {        // a workgroup of 512 per matrix
      const unsigned nb = (unsigned)(batch - b < MAX_GROUPS ? batch - b : MAX_GROUPS);
      const char* xb = reinterpret_cast<const char*>(x) + b * x_batch * (x_is_bf16 ? 2 : 4);
      char* ob = reinterpret_cast<char*>(out) + b * out_batch * (out_is_bf16 ? 2 : 4);
      if (x_is_bf16 && out_is_bf16) ns_small<1, 2>(m, xb, (long)x_batch, ob, (long)out_batch, (long)ldo, steps, eps, nb, st);
      else if (x_is_bf16) ns_small<1, 1>(m, xb, (long)x_batch, ob, (long)out_batch, (long)ldo, steps, eps, nb, st);
      else if (out_is_bf16) ns_small<0, 2>(m, xb, (long)x_batch, ob, (long)out_batch, (long)ldo, steps, eps, nb, st);
      else ns_small<0, 1>(m, xb, (long)x_batch, ob, (long)out_batch, (long)ldo, steps, eps, nb, st);
    }
    PG_LAUNCH_OK("pg_orthogonalise");
    return 0;
  }
  NsPlan pl{};
  long piece = 0;
  const char* bad = ns_plan_batch(pl, batch, rows, cols, x_batch, ldx, out_batch, piece);
  PG_REQUIRE(bad == nullptr, "pg_orthogonalise: %s", bad);
  PG_REQUIRE(workspace && workspace_bytes >= pl.bytes, "pg_orthogonalise: workspace of %lld bytes required", (long long)pl.bytes);
  char* w = reinterpret_cast<char*>(workspace);
  hipStream_t st = (hipStream_t)stream;
  NsNorm* sq = reinterpret_cast<NsNorm*>(w + pl.off_sq);
  const NsStep none{};
  for (int64_t b = 0; b < batch; b += piece) {
    pl.gr.n = (int)(batch - b < piece ? batch - b : piece);
    for (int f = 0; f < F_N; ++f) pl.n[f] = (long)pl.gr.per[f] * pl.gr.n;
    const NsSource in = {x_is_bf16 ? 1 : 0, reinterpret_cast<const char*>(x) + b * x_batch * (x_is_bf16 ? 2 : 4)};
    if (x_is_bf16) PG_KLAUNCH((ns_sumsq_kernel<1>), dim3((unsigned)pl.n[F_MOM]), dim3(256), 0, st, pl.gr, in.x, sq);
    else PG_KLAUNCH((ns_sumsq_kernel<0>), dim3((unsigned)pl.n[F_MOM]), dim3(256), 0, st, pl.gr, in.x, sq);
    ns_run(pl, w, in, none, steps, eps, out_is_bf16 ? 2 : 1, reinterpret_cast<char*>(out) + b * out_batch * (out_is_bf16 ? 2 : 4), (long)ldo, st);
  }
  PG_LAUNCH_OK("pg_orthogonalise");
  return 0;
}

extern "C" int64_t pg_muon_workspace(const pg_muon_entry_t* entries, int32_t n) {
  if (!entries || n <= 0) return 0;
  NsPlan pl{};
  return ns_plan_table(pl, entries, n) ? -1 : pl.bytes;
}

extern "C" int pg_muon_step(const pg_muon_t* d, void* stream) {
  PG_REQUIRE(d && d->entries && d->n >= 0, "pg_muon_step: descriptor and entries required");
  if (d->n == 0) return 0;
  PG_REQUIRE(d->p && (d->g || d->g_bf16) && d->m, "pg_muon_step: p, g (or g_bf16) and m required");
  PG_REQUIRE((((size_t)d->p | (size_t)d->g | (size_t)d->m | (size_t)d->v) & 15) == 0 && (((size_t)d->g_bf16 | (size_t)d->p_bf16) & 7) == 0 &&
             ((size_t)d->workspace & 255) == 0, "pg_muon_step: arenas 16-byte (bf16: 8-byte) aligned, workspace 256-byte aligned");
  PG_REQUIRE(d->steps >= 1 && d->steps <= 32 && d->eps > 0.f, "pg_muon_step: steps 1..32 and eps > 0 required");
  NsPlan pl{};
  const char* bad = ns_plan_table(pl, d->entries, d->n);
  PG_REQUIRE(bad == nullptr, "pg_muon_step: %s", bad);
  for (int i = 0; i < d->n; ++i) {
    const pg_muon_entry_t& e = d->entries[i];
    PG_REQUIRE(e.off <= d->total - (int64_t)e.taps * e.rows * e.cols, "pg_muon_step: entry %d ends behind the arena", i);
    PG_REQUIRE(e.kind == 0 || d->v, "pg_muon_step: an Adam entry needs v");
    // 1 - beta^t divides: t >= 1 whatever a counter, which begins at 0, adds
    PG_REQUIRE(e.kind == 0 || (d->step >= 1 && d->beta1 >= 0.0 && d->beta1 < 1.0 && d->beta2 >= 0.0 && d->beta2 < 1.0),
               "pg_muon_step: an Adam entry needs step >= 1 and betas in [0, 1)");
    if (i > 0) {
      const pg_muon_entry_t& q = d->entries[i - 1];
      PG_REQUIRE(e.off >= q.off + (int64_t)q.taps * q.rows * q.cols, "pg_muon_step: entries %d and %d overlap or are out of order", i - 1, i);
    }
  }
  PG_REQUIRE(d->workspace && d->workspace_bytes >= pl.bytes, "pg_muon_step: workspace of %lld bytes required", (long long)pl.bytes);
  hipStream_t st = (hipStream_t)stream;
  char* w = reinterpret_cast<char*>(d->workspace);
  NsMat* tab = reinterpret_cast<NsMat*>(w + pl.off_tab);
  int* first = reinterpret_cast<int*>(w + pl.off_first);
  for (int i = 0; i < d->n; i += 16) {
    NsChunk c;
    const int cnt = d->n - i < 16 ? d->n - i : 16;
    memset(&c, 0, sizeof(c));
    for (int k = 0; k < cnt; ++k) {
      c.m[k] = pl.mats[(size_t)(i + k)];
      for (int f = 0; f < F_N; ++f) c.first[f][k] = pl.first[(size_t)(f * d->n + i + k)];
    }
    PG_KLAUNCH(ns_table_kernel, dim3(1), dim3(256), 0, st, c, tab, first, i, cnt, d->n);
  }
  pl.gr.tab = tab;
  pl.gr.first = first;
  NsStep s{};
  s.p = d->p; s.g = d->g; s.gb = reinterpret_cast<const bf16_t*>(d->g_bf16); s.m = d->m; s.v = d->v;
  s.pb = reinterpret_cast<bf16_t*>(d->p_bf16);
  s.mu = d->momentum; s.gscale = d->grad_scale; s.lr = d->lr; s.wd = d->weight_decay; s.nesterov = d->nesterov;
  s.b1 = (float)d->beta1; s.b2 = (float)d->beta2; s.eps = d->adam_eps; s.b1d = d->beta1; s.b2d = d->beta2;
  s.step0 = (long)d->step; s.ctr = reinterpret_cast<const unsigned long long*>(d->ctr);
  PG_KLAUNCH(muon_momentum_kernel, dim3((unsigned)pl.n[F_MOM]), dim3(256), 0, st, pl.gr, s, reinterpret_cast<NsNorm*>(w + pl.off_sq));
  if (pl.n[F_GRAM] > 0) {
    const NsSource in = {2, nullptr};
    ns_run(pl, w, in, s, d->steps, d->eps, 3, nullptr, 0, st);
  }
  PG_LAUNCH_OK("pg_muon_step");
  return 0;
}
