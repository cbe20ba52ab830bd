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
// gives (measured 4.8e-6 against 4.7e-6 through five steps; a bf16 pair with its 16 bits: 4e-5, single bf16 operands: 2e-2).  X0's
// scale makes its rms 1 within a factor 2^0.5: its largest element is then at most sqrt(rows cols) <= 2^15.5, the loss of a tiny one's last bits
// is 2^-25 of the rms.  |G|, |Q G| <= 1.5, |Q| <= 3.45, |P| <= 3.45^3 = 41 bound the others' scales.  A bf16 input is one fp16 value exactly (8 bits): one plane.
//
// Layout.  A matrix is stored by the caller as [taps][rows][cols] with row and tap strides (a packed convolution weight is one matrix
// [rows, taps * cols]); the planes here are [M][N], M <= N the short side, both padded with zeros to multiples of 64: no product checks
// a bound along K, and padding stays zero through every step.  All matrices of a call share every launch (a device table of tile ranges).
#include "common.h"
#include <math.h>
#include <vector>

namespace pg {

typedef unsigned short bf16_t;
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;
constexpr int SG = 12, SP = 10;                 // log2 of the scales of G, Q, Q G and of P
constexpr int K0_ELEMS = 16384;                 // elements per workgroup of the momentum / square-sum pass
constexpr int GT = 128, CT = 64, AI = 128, AJ = 128;      // tiles: Gram, chain, apply (rows, columns)

struct NsMat {
  long src, ld, st;             // the caller's storage: element offset, row stride, tap stride
  int taps, rows, cols, kind;   // kind 1: a vector (Adam), rows = taps = 1
  int M, N, Mp, Np, tall;       // short and long side, padded; tall: the rows are the long side
  int ks, kc;                   // Gram: splits of the long side and their length (a multiple of 32)
  int np;                       // partial sums of squares
  float scale;
  long x, g, part;              // offsets in the workspace: X planes and chain planes (halves), Gram partials (floats)
  int b0, b1, bg, br, bc, ba;   // first workgroup in: momentum, split, Gram, its join, chain, apply
};
struct NsGroup {                // matrices of one call: a device table, or (tab = nullptr) `n` equal ones
  const NsMat* tab;
  int n;
  NsMat u;                      // the single record of equal matrices: offsets of number 0
  long src_step, out_step, x_step, g_step, part_step;
  int n0, n1, ng, nr, nc, na;   // workgroups per matrix
};
struct NsRef { NsMat m; int id, tile; long out; };

template <int NsMat::*FIRST, int NsGroup::*PER>
__device__ __forceinline__ NsRef ns_find(const NsGroup& gr, int b) {
  NsRef r;
  if (gr.tab == nullptr) {
    const int per = gr.*PER;
    r.id = b / per;
    r.tile = b - r.id * per;
    r.m = gr.u;
    r.out = (long)r.id * gr.out_step;
    r.m.src += (long)r.id * gr.src_step;
    r.m.x += (long)r.id * gr.x_step; r.m.g += (long)r.id * gr.g_step; r.m.part += (long)r.id * gr.part_step;
    return r;
  }
  int lo = 0, hi = gr.n - 1;    // the last record whose range begins at or before b
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (gr.tab[mid].*FIRST <= b) lo = mid;
    else hi = mid - 1;
  }
  r.id = lo;
  r.m = gr.tab[lo];
  r.tile = b - r.m.*FIRST;
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
__device__ __forceinline__ double block_sum_d256(double v, double* red) {
  v = wave_sum_d(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
}

// ---------------------------------------------------------------------------------------------- table upload
struct NsChunk { NsMat m[16]; };
__global__ void ns_table_kernel(NsChunk c, NsMat* tab, int n) {
  const int words = (int)(sizeof(NsMat) / 4);
  for (int i = threadIdx.x; i < n * words; i += 64)
    reinterpret_cast<unsigned*>(tab)[i] = reinterpret_cast<const unsigned*>(&c)[i];
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

// one workgroup = K0_ELEMS consecutive elements of a tensor; 28 bytes / element for Adam's, 12 for a matrix's
__global__ __launch_bounds__(256) void muon_momentum_kernel(const NsGroup gr, const NsStep s, double* sq) {
  __shared__ double red[4];
  const NsRef r = ns_find<&NsMat::b0, &NsGroup::n0>(gr, blockIdx.x);
  const long n = (long)r.m.taps * r.m.rows * r.m.cols;
  const long e0 = (long)r.tile * K0_ELEMS, e1 = min(n, e0 + K0_ELEMS);
  const long base = r.m.src;
  if (r.m.kind == 1) {
    const double t = (double)(s.step0 + (s.ctr ? (long)s.ctr[0] : 0L));
    const float step_size = (float)((double)s.lr / (1.0 - pow(s.b1d, t)));
    const float bc2 = (float)sqrt(1.0 - pow(s.b2d, t));
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
        const double u = (double)ns_update(s, gg, m[e]);
        acc = fma(u, u, acc);
      }
      *reinterpret_cast<float4*>(s.m + base + i) = make_float4(m[0], m[1], m[2], m[3]);
    }
  } else {
    for (long i = e0 + threadIdx.x; i < e1; i += 256) {
      const float gg = ns_grad(s, base + i);
      const float m = s.mu * s.m[base + i] + (1.f - s.mu) * gg;
      s.m[base + i] = m;
      const double u = (double)ns_update(s, gg, m);
      acc = fma(u, u, acc);
    }
  }
  acc = block_sum_d256(acc, red);
  if (threadIdx.x == 0) sq[blockIdx.x] = acc;
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

// one workgroup = K0_ELEMS / 8 runs of eight stored neighbours
template <int SRC>
__global__ __launch_bounds__(256) void ns_sumsq_kernel(const NsGroup gr, const void* x, double* sq) {
  __shared__ double red[4];
  const NsRef r = ns_find<&NsMat::b0, &NsGroup::n0>(gr, blockIdx.x);
  const unsigned rpr = (unsigned)(r.m.cols + 7) / 8u;
  const unsigned n = (unsigned)r.m.rows * rpr;
  const unsigned e0 = (unsigned)r.tile * (K0_ELEMS / 8), e1 = min(n, e0 + K0_ELEMS / 8);
  double acc = 0.0;
  const NsStep s{};
  for (unsigned i = e0 + threadIdx.x; i < e1; i += 256) {
    const unsigned row = i / rpr;
    float v[8];
    ns_load8<SRC>(r.m, x, s, (int)row, (int)(i - row * rpr) * 8, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc = fma((double)v[e], (double)v[e], acc);
  }
  acc = block_sum_d256(acc, red);
  if (threadIdx.x == 0) sq[blockIdx.x] = acc;
}

// ---------------------------------------------------------------------------------------------- split into fp16 planes
// every workgroup joins its matrix's partial sums of squares itself (a few hundred doubles); the first one publishes
// c = 2^k / (|U| + eps), the factor from the planes' units to X0's
template <int SRC>
__global__ __launch_bounds__(256) void ns_split_kernel(const NsGroup gr, const void* x, const NsStep s, const double* sq, float eps,
                                                       float* cfac, _Float16* ws) {
  __shared__ double red[4];
  __shared__ float tile[64][65];
  constexpr bool ONE = SRC == 1;
  const NsRef r = ns_find<&NsMat::b1, &NsGroup::n1>(gr, blockIdx.x);
  const NsMat& m = r.m;
  const long n = (long)m.taps * m.rows * m.cols;
  const int np = m.np;
  const int first = gr.tab ? m.b0 : r.id * gr.n0;
  double a = 0.0;
  for (int i = threadIdx.x; i < np; i += 256) a += sq[first + i];
  a = block_sum_d256(a, red);
  const double norm = sqrt(a);
  // 2^k >= rms / 2^0.75, so that the largest element, at most sqrt(n) rms, stays below 2^(15.5 + 0.75 - 0.5) ... 55200 in the planes
  const double rms = sqrt(a / (double)n);
  int k = 0;
  if (rms > 0.0 && rms < 1e300) k = max(-126, min(126, (int)rint(log2(rms) + 0.25)));
  const float f = (float)ldexp(1.0, -k);
  if (r.tile == 0 && threadIdx.x == 0) cfac[r.id] = norm == 0.0 ? 0.f : (float)(ldexp(1.0, k) / (norm + (double)eps));
  _Float16* hi = ws + m.x;
  _Float16* lo = hi + (long)m.Mp * m.Np;
  if (!m.tall) {
    // 1024 chunks of 8 plane elements per workgroup
    const int cpr = m.Np / 8;
    const long nch = (long)m.Mp * cpr;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const long ch = (long)r.tile * 1024 + q * 256 + threadIdx.x;
      if (ch >= nch) break;
      const int i = (int)(ch / cpr), j = (int)(ch - (long)i * cpr) * 8;
      float v[8];
      if (i < m.M && j < m.N) {
        ns_load8<SRC>(m, x, s, i, j, v);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.f;
      }
      half8 h, l;
#pragma unroll
      for (int e = 0; e < 8; ++e) { _Float16 th, tl; split16(v[e] * f, th, tl); h[e] = th; l[e] = tl; }
      *reinterpret_cast<half8*>(hi + (long)i * m.Np + j) = h;
      if constexpr (!ONE) *reinterpret_cast<half8*>(lo + (long)i * m.Np + j) = l;
    }
  } else {
    // 64 x 64 tile through LDS: plane row i = stored flat column, plane column j = stored row
    const int tj = m.Np / 64;
    const int i0 = (r.tile / tj) * 64, j0 = (r.tile % tj) * 64;
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    for (int q = ty; q < 64; q += 4) {
      const int j = j0 + q, i = i0 + tx;
      tile[q][tx] = (j < m.N && i < m.M) ? ns_elem<SRC>(x, s, ns_at(m, j, i)) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int c = q * 256 + threadIdx.x, i = c >> 3, j = (c & 7) * 8;
      half8 h, l;
#pragma unroll
      for (int e = 0; e < 8; ++e) { _Float16 th, tl; split16(tile[j + e][i] * f, th, tl); h[e] = th; l[e] = tl; }
      *reinterpret_cast<half8*>(hi + (long)(i0 + i) * m.Np + j0 + j) = h;
      if constexpr (!ONE) *reinterpret_cast<half8*>(lo + (long)(i0 + i) * m.Np + j0 + j) = l;
    }
  }
}

// ---------------------------------------------------------------------------------------------- product core, both operands K-contiguous
// C[BM][BN] = sum_k A[i][k] B[j][k], operands as PL fp16 planes; 4 waves (2 x 2), K in steps of 32 through two LDS stages.
// An LDS row is 32 halves = four 16-byte slots, chunk c of row r at slot c ^ ((r >> 2) & 3): the 16 lanes that a
// ds_read_b128 serves at a time (16 consecutive rows, one chunk) then cover the 256 bytes of a bank row once.
template <int BM, int BN, int PL>
struct NtCore {
  static constexpr int TM = BM / 64, TN = BN / 64;
  static constexpr int ROWS = (BM + BN) * PL;                       // LDS rows of a stage
  static constexpr int PASS = ROWS * 4 / 256;                       // 16-byte chunks per thread
  static constexpr int LDS_BYTES = 2 * ROWS * 64;
  f32x16 acc[TM][TN];

  __device__ __forceinline__ void run(char* smem, const _Float16* A, long a_plane, long lda, int a_rows, const _Float16* B, long b_plane,
                                      long ldb, int b_rows, int k0, int k1) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = (wave >> 1) * (BM / 2), wn = (wave & 1) * (BN / 2);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    const _Float16* src[PASS];
    int dst[PASS];
#pragma unroll
    for (int q = 0; q < PASS; ++q) {
      const int c = q * 256 + tid, row = c >> 2, slot = c & 3;
      const bool isA = row < BM * PL;
      const int rr = isA ? row : row - BM * PL;
      const int pl = rr / (isA ? BM : BN), lr = rr - pl * (isA ? BM : BN);
      const bool ok = lr < (isA ? a_rows : b_rows);
      src[q] = !ok ? nullptr : (isA ? A + pl * a_plane + (long)lr * lda : B + pl * b_plane + (long)lr * ldb) + slot * 8;
      dst[q] = row * 64 + ((slot ^ ((row >> 2) & 3)) << 4);
    }
    uint4 v[PASS];
    auto load = [&](int k) {
#pragma unroll
      for (int q = 0; q < PASS; ++q) v[q] = src[q] ? *reinterpret_cast<const uint4*>(src[q] + k) : make_uint4(0u, 0u, 0u, 0u);
    };
    auto put = [&](int st) {
#pragma unroll
      for (int q = 0; q < PASS; ++q) *reinterpret_cast<uint4*>(smem + st * (ROWS * 64) + dst[q]) = v[q];
    };
    auto frag = [&](int st, int row, int ks) {
      const int c = ks * 2 + (lane >> 5);
      return *reinterpret_cast<const half8*>(smem + st * (ROWS * 64) + row * 64 + ((c ^ ((row >> 2) & 3)) << 4));
    };
    load(k0);
    put(0);
    __syncthreads();
    int st = 0;
    for (int k = k0; k < k1; k += 32) {
      const bool more = k + 32 < k1;
      if (more) load(k + 32);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        half8 a[PL][TM], b[PL][TN];
#pragma unroll
        for (int pl = 0; pl < PL; ++pl) {
#pragma unroll
          for (int i = 0; i < TM; ++i) a[pl][i] = frag(st, pl * BM + wm + i * 32 + (lane & 31), ks);
#pragma unroll
          for (int j = 0; j < TN; ++j) b[pl][j] = frag(st, BM * PL + pl * BN + wn + j * 32 + (lane & 31), ks);
        }
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) {
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0][i], b[0][j], acc[i][j], 0, 0, 0);
            if constexpr (PL == 2) {
              acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0][i], b[1][j], acc[i][j], 0, 0, 0);
              acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[1][i], b[0][j], acc[i][j], 0, 0, 0);
            }
          }
      }
      if (more) put(st ^ 1);
      __syncthreads();
      st ^= 1;
    }
  }
  // f(row, column, value) of the tile, for every accumulator element: rows 8 (e >> 2) + 4 (lane >> 5) + (e & 3), column lane & 31
  template <typename F>
  __device__ __forceinline__ void each4(F&& f) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = (wave >> 1) * (BM / 2), wn = (wave & 1) * (BN / 2);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float v[4] = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
          f(wm + i * 32 + 8 * q + 4 * (lane >> 5), wn + j * 32 + (lane & 31), v);
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

// G = X X^T over one slice of the long side: fp32 partial tiles
template <int PL>
__global__ __launch_bounds__(256, 2) void ns_gram_kernel(const NsGroup gr, const _Float16* ws, float* part) {
  typedef NtCore<GT, GT, PL> Core;
  __shared__ __attribute__((aligned(16))) char smem[Core::LDS_BYTES];
  const NsRef r = ns_find<&NsMat::bg, &NsGroup::ng>(gr, blockIdx.x);
  const NsMat& m = r.m;
  const int nt = (m.Mp + GT - 1) / GT, ntri = nt * (nt + 1) / 2;
  const int split = r.tile / ntri, t = r.tile - split * ntri;
  int bi, bj;
  tri(t, bi, bj);
  const _Float16* X = ws + m.x;
  const long plane = (long)m.Mp * m.Np;
  Core c;
  c.run(smem, X + (long)bi * GT * m.Np, plane, m.Np, m.Mp - bi * GT, X + (long)bj * GT * m.Np, plane, m.Np, m.Mp - bj * GT,
        split * m.kc, min(m.Np, (split + 1) * m.kc));
  float* out = part + m.part + (long)r.tile * (GT * GT);
  c.each4([&](int i, int j, const float (&v)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) out[(i + e) * GT + j] = v[e];
  });
}

// join of the slices, in order; both triangles of G from the lower one; one workgroup = 64 x 64 elements
__global__ __launch_bounds__(256) void ns_gram_join_kernel(const NsGroup gr, const float* part, const float* cfac, float cconst, _Float16* ws) {
  __shared__ float tile[64][65];
  const NsRef r = ns_find<&NsMat::br, &NsGroup::nr>(gr, blockIdx.x);
  const NsMat& m = r.m;
  int bi, bj;
  tri(r.tile, bi, bj);                               // in units of 64
  const int gi = bi / 2, gj = bj / 2;                // the 128-tile that holds it
  const int nt = (m.Mp + GT - 1) / GT, ntri = nt * (nt + 1) / 2;
  const long t0 = gi * (gi + 1) / 2 + gj;
  const float c1 = cfac ? cfac[r.id] : cconst;
  const float c2 = c1 * c1 * (float)(1 << SG);
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
  for (int q = ty; q < 64; q += 4) {
    const float* src = part + m.part + t0 * (GT * GT) + (long)((bi & 1) * 64 + q) * GT + (bj & 1) * 64 + tx;
    float a = 0.f;
    for (int s = 0; s < m.ks; ++s) a += src[(long)s * ntri * (GT * GT)];
    tile[q][tx] = a * c2;
  }
  __syncthreads();
  _Float16* G = ws + m.g;
  const long pl = (long)m.Mp * m.Mp;
  for (int q = ty; q < 64; q += 4) {
    _Float16 h, l;
    const float v = (bi == bj && tx > q) ? tile[tx][q] : tile[q][tx];
    split16(v, h, l);
    const long at = (long)(bi * 64 + q) * m.Mp + bj * 64 + tx;
    G[at] = h; G[pl + at] = l;
    if (bi != bj) {
      split16(tile[tx][q], h, l);
      const long bt = (long)(bj * 64 + q) * m.Mp + bi * 64 + tx;
      G[bt] = h; G[pl + bt] = l;
    }
  }
}

// chain planes of a matrix: 0 G, 1 Q, 2 Q G, 3 P, 4 the other P  (hi and lo each)
// C = A B of commuting symmetric matrices: the lower triangle of 64 x 64 tiles, mirrored.  `quad`: C = a I + b A + c A A
struct ChainJob { int a, b, c; float mul; int quad; };
__global__ __launch_bounds__(256, 2) void ns_chain_kernel(const NsGroup gr, ChainJob j0, ChainJob j1, int njobs, _Float16* ws) {
  typedef NtCore<CT, CT, 2> Core;
  __shared__ __attribute__((aligned(16))) char smem[Core::LDS_BYTES];
  const int job = njobs == 2 ? (int)(blockIdx.x & 1) : 0;
  const NsRef r = ns_find<&NsMat::bc, &NsGroup::nc>(gr, njobs == 2 ? (int)(blockIdx.x >> 1) : (int)blockIdx.x);
  const ChainJob jb = job ? j1 : j0;
  const NsMat& m = r.m;
  int bi, bj;
  tri(r.tile, bi, bj);
  const long pl = (long)m.Mp * m.Mp;
  const _Float16* A = ws + m.g + jb.a * 2 * pl;
  const _Float16* B = ws + m.g + jb.b * 2 * pl;
  _Float16* C = ws + m.g + jb.c * 2 * pl;
  Core c;
  c.run(smem, A + (long)bi * CT * m.Mp, pl, m.Mp, CT, B + (long)bj * CT * m.Mp, pl, m.Mp, CT, 0, m.Mp);
  c.each4([&](int i, int j, const float (&v)[4]) {
    const int gi = bi * CT + i, gj = bj * CT + j;
    half4 hh, ll;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float t = v[e] * jb.mul;
      const long at = (long)(gi + e) * m.Mp + gj;
      if (jb.quad) {
        t += NS_B * ((float)A[at] + (float)A[pl + at]);
        if (gi + e == gj) t += NS_A * (float)(1 << SG);
      }
      _Float16 h, l;
      split16(t, h, l);
      hh[e] = h; ll[e] = l;
      if (bi != bj || gi + e >= gj) { C[at] = h; C[pl + at] = l; }
    }
    if (bi != bj) {
      const long bt = (long)gj * m.Mp + gi;
      *reinterpret_cast<half4*>(C + bt) = hh;
      *reinterpret_cast<half4*>(C + pl + bt) = ll;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (gi + e > gj) { C[(long)gj * m.Mp + gi + e] = hh[e]; C[pl + (long)gj * m.Mp + gi + e] = ll[e]; }
    }
  });
}

// ---------------------------------------------------------------------------------------------- X <- P X
// OUT: 0 = planes of the next stage, 1 = fp32 tensor, 2 = bf16 tensor, 3 = the step's update of p
struct ApplyK {
  const _Float16* wsx; const _Float16* wsg; _Float16* wso;
  int pbuf;
  const float* cfac; float cconst;        // planes' units -> values
  float mul;
  void* out; long ldo;
  NsStep s;
};
template <int PX, int OUT>
__global__ __launch_bounds__(256, 2) void ns_apply_kernel(const NsGroup gr, const ApplyK k) {
  constexpr int A_BYTES = AI * 2 * 64, B_BYTES = 32 * AJ * 2 * PX, STAGE = A_BYTES + B_BYTES;
  constexpr int PA = AI * 2 * 4 / 256, PB = 32 * (AJ / 8) * PX / 256;
  __shared__ __attribute__((aligned(16))) char smem[2 * STAGE];
  const NsRef r = ns_find<&NsMat::ba, &NsGroup::na>(gr, blockIdx.x);
  const NsMat& m = r.m;
  const int ti = (m.Mp + AI - 1) / AI;
  const int i0 = (r.tile % ti) * AI, j0 = (r.tile / ti) * AJ;
  const long pl = (long)m.Mp * m.Mp, xpl = (long)m.Mp * m.Np;
  const _Float16* P = k.wsg + m.g + k.pbuf * 2 * pl;
  const _Float16* X = k.wsx + m.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
  f32x16 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  const _Float16* as[PA]; int ad[PA];
#pragma unroll
  for (int q = 0; q < PA; ++q) {
    const int c = q * 256 + tid, row = c >> 2, slot = c & 3, plane = row / AI, lr = row - plane * AI;
    as[q] = i0 + lr < m.Mp ? P + plane * pl + (long)(i0 + lr) * m.Mp + slot * 8 : nullptr;
    ad[q] = row * 64 + ((slot ^ ((row >> 2) & 3)) << 4);
  }
  // X rows = K: [32][128] halves per plane, chunk c of row k at slot c ^ ((k & 3) << 2) for the transposing reads
  const _Float16* bs[PB]; int bd[PB];
#pragma unroll
  for (int q = 0; q < PB; ++q) {
    const int c = q * 256 + tid, row = c >> 4, slot = c & 15, plane = row >> 5, kr = row & 31;
    bs[q] = j0 + slot * 8 < m.Np ? X + plane * xpl + (long)kr * m.Np + j0 + slot * 8 : nullptr;
    bd[q] = A_BYTES + row * (AJ * 2) + ((slot ^ ((kr & 3) << 2)) << 4);
  }
  uint4 va[PA], vb[PB];
  auto load = [&](int kk) {
#pragma unroll
    for (int q = 0; q < PA; ++q) va[q] = as[q] ? *reinterpret_cast<const uint4*>(as[q] + kk) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int q = 0; q < PB; ++q) vb[q] = bs[q] ? *reinterpret_cast<const uint4*>(bs[q] + (long)kk * m.Np) : make_uint4(0u, 0u, 0u, 0u);
  };
  auto put = [&](int st) {
#pragma unroll
    for (int q = 0; q < PA; ++q) *reinterpret_cast<uint4*>(smem + st * STAGE + ad[q]) = va[q];
#pragma unroll
    for (int q = 0; q < PB; ++q) *reinterpret_cast<uint4*>(smem + st * STAGE + bd[q]) = vb[q];
  };
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  const int r4 = (lane >> 2) & 3, cq = lane & 3, mb = (lane >> 4) & 1, kh = lane >> 5;
  load(0);
  put(0);
  __syncthreads();
  int st = 0;
  for (int kk = 0; kk < m.Mp; kk += 32) {
    const bool more = kk + 32 < m.Mp;
    if (more) load(kk + 32);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      half8 a[2][2], b[PX][2];
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = p * AI + wm + i * 32 + (lane & 31), c = ks * 2 + kh;
          a[p][i] = *reinterpret_cast<const half8*>(smem + st * STAGE + row * 64 + ((c ^ ((row >> 2) & 3)) << 4));
        }
#pragma unroll
      for (int p = 0; p < PX; ++p)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int chunk = ((wn + j * 32) >> 3) + 2 * mb + (cq >> 1);
          char* q = smem + st * STAGE + A_BYTES + (p * 32 + ks * 16 + 8 * kh + r4) * (AJ * 2) + ((chunk ^ (r4 << 2)) << 4) + ((cq & 1) << 3);
          const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)q);
          const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(q + 4 * AJ * 2));
          typedef short s16x8 __attribute__((ext_vector_type(8)));
          const s16x8 w = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
          b[p][j] = __builtin_bit_cast(half8, w);
        }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0][i], b[0][j], acc[i][j], 0, 0, 0);
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[1][i], b[0][j], acc[i][j], 0, 0, 0);
          if constexpr (PX == 2) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0][i], b[1][j], acc[i][j], 0, 0, 0);
        }
    }
    if (more) put(st ^ 1);
    __syncthreads();
    st ^= 1;
  }
  const float f = (k.cfac ? k.cfac[r.id] : k.cconst) * k.mul;
  const float keep = 1.f - k.s.lr * k.s.wd, step = k.s.lr * m.scale;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int gj = j0 + wn + j * 32 + (lane & 31);
    if constexpr (OUT == 0) {
      if (gj >= m.Np) continue;
    } else {
      if (gj >= m.N) continue;
    }
    // wide: the column is the lane's for all rows; tall: it is the stored row
    const long cbase = OUT == 0 ? (long)gj : m.tall ? 0L : ns_at(m, 0, gj);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int ii = i0 + wm + i * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
        const float v = acc[i][j][e] * f;
        if constexpr (OUT == 0) {
          if (ii < m.Mp) {
            _Float16 h, l;
            split16(v, h, l);
            _Float16* o = k.wso + m.x + (long)ii * m.Np + gj;
            o[0] = h; o[xpl] = l;
          }
        } else {
          if (ii < m.M) {
            if constexpr (OUT == 3) {
              const long at = m.tall ? ns_at(m, gj, ii) : cbase + (long)ii * m.ld;
              const float p = k.s.p[at] * keep - step * v;
              k.s.p[at] = p;
              if (k.s.pb) k.s.pb[at] = (bf16_t)(ns_pack_bf16(p, 0.f) & 0xffffu);
            } else {
              const long at = r.out + (m.tall ? (long)gj * k.ldo + ii : (long)ii * k.ldo + gj);
              if constexpr (OUT == 1) reinterpret_cast<float*>(k.out)[at] = v;
              else reinterpret_cast<bf16_t*>(k.out)[at] = (bf16_t)(ns_pack_bf16(v, 0.f) & 0xffffu);
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
  long n0, n1, ng, nr, nc, na;  // workgroups per launch
  int nscal;
  long off_tab, off_c, off_sq, off_x, x_halves, off_g, off_part, bytes;
};

// sizes and workgroup counts of one matrix; false: a side or a product of sides out of range
static bool ns_shape(NsMat& m) {
  const long rows = m.rows, cols = (long)m.taps * m.cols;
  if (rows * cols > 0x7fffffffL) return false;
  m.tall = rows > cols;
  m.M = (int)(m.tall ? cols : rows);
  m.N = (int)(m.tall ? rows : cols);
  m.Mp = (int)up(m.M, 64);
  m.Np = (int)up(m.N, 64);
  if ((long)m.Mp * m.Np > 0x7fffffffL) return false;
  return true;
}
struct NsCounts { long n0, n1, ng, nr, nc, na, x, g, part; };
static NsCounts ns_counts(NsMat& m, long others, bool flat) {
  NsCounts c;
  const long n = (long)m.taps * m.rows * m.cols;
  c.n0 = flat ? cdiv(n, K0_ELEMS) : cdiv((long)m.rows * cdiv(m.cols, 8), K0_ELEMS / 8);
  m.np = (int)c.n0;
  if (m.kind == 1) { c.n1 = c.ng = c.nr = c.nc = c.na = c.x = c.g = c.part = 0; return c; }
  c.n1 = m.tall ? (long)(m.Mp / 64) * (m.Np / 64) : cdiv((long)m.Mp * m.Np / 8, 1024);
  const long nt = cdiv(m.Mp, GT), ntri = nt * (nt + 1) / 2;
  // slices of the long side: enough workgroups for two per CU, at least 512 columns each
  long ks = cdiv(512, ntri * (others > 0 ? others : 1));
  if (ks > m.Np / 512) ks = m.Np / 512;
  if (ks < 1) ks = 1;
  m.kc = (int)up(cdiv(m.Np, ks), 32);
  m.ks = (int)cdiv(m.Np, m.kc);
  c.ng = ntri * m.ks;
  const long n64 = m.Mp / 64;
  c.nr = c.nc = n64 * (n64 + 1) / 2;
  c.na = (long)cdiv(m.Mp, AI) * cdiv(m.Np, AJ);
  c.x = 2L * m.Mp * m.Np;
  c.g = 10L * m.Mp * m.Mp;
  c.part = (long)c.ng * GT * GT;
  return c;
}
static void ns_place(NsPlan& pl, int nmat, long nx, long ng, long npart) {
  auto take = [&](long& off, long bytes) { off = pl.bytes; pl.bytes += up(bytes, 256); };
  pl.bytes = 0;
  take(pl.off_tab, (long)pl.mats.size() * (long)sizeof(NsMat));
  take(pl.off_c, (long)nmat * 4);
  take(pl.off_sq, pl.n0 * 8);
  pl.x_halves = up(nx, 128);
  take(pl.off_x, pl.x_halves * 2 * 2);               // two sets of planes: X and its successor
  take(pl.off_g, ng * 2);
  take(pl.off_part, npart * 4);
}

static const char* ns_plan_batch(NsPlan& pl, long batch, long rows, long cols, long sx, long ldx, long so) {
  NsMat m{};
  m.taps = 1; m.rows = (int)rows; m.cols = (int)cols; m.ld = ldx; m.st = 0;
  if (!ns_shape(m)) return "a matrix has more than 2^31 - 1 elements";
  const NsCounts c = ns_counts(m, batch, false);
  pl.gr.tab = nullptr;
  pl.gr.n = (int)batch;
  pl.gr.u = m;
  pl.gr.src_step = sx; pl.gr.out_step = so; pl.gr.x_step = c.x; pl.gr.g_step = c.g; pl.gr.part_step = c.part;
  pl.gr.n0 = (int)c.n0; pl.gr.n1 = (int)c.n1; pl.gr.ng = (int)c.ng; pl.gr.nr = (int)c.nr; pl.gr.nc = (int)c.nc; pl.gr.na = (int)c.na;
  pl.n0 = c.n0 * batch; pl.n1 = c.n1 * batch; pl.ng = c.ng * batch; pl.nr = c.nr * batch; pl.nc = c.nc * batch; pl.na = c.na * batch;
  const long top = 0x3fffffffL;
  if (pl.n0 > top || pl.n1 > top || pl.ng > top || pl.nc > top || pl.na > top) return "too many matrices for one call";
  ns_place(pl, (int)batch, c.x * batch, c.g * batch, c.part * batch);
  return nullptr;
}

static const char* ns_plan_table(NsPlan& pl, const pg_muon_entry_t* e, int n) {
  pl.mats.resize((size_t)n);
  long work = 0;
  for (int i = 0; i < n; ++i) {
    NsMat& m = pl.mats[(size_t)i];
    m = NsMat{};
    if (e[i].taps <= 0 || e[i].rows <= 0 || e[i].cols <= 0 || e[i].off < 0 || (e[i].kind != 0 && e[i].kind != 1)) return "an entry with a size <= 0, a negative offset or an unknown kind";
    m.src = e[i].off; m.taps = e[i].taps; m.rows = e[i].rows; m.cols = e[i].cols; m.kind = e[i].kind; m.scale = e[i].scale;
    m.ld = m.cols; m.st = (long)m.rows * m.cols;
    if ((long)m.taps * m.rows > 0x7fffffffL || (long)m.taps * m.rows * m.cols > 0x7fffffffL) return "a tensor has more than 2^31 - 1 elements";
    if (m.kind == 0) {
      if (!ns_shape(m)) return "a matrix has more than 2^31 - 1 elements";
      work += (long)m.Mp * m.Np;
    }
  }
  long b0 = 0, b1 = 0, bg = 0, br = 0, bc = 0, ba = 0, x = 0, g = 0, part = 0;
  for (int i = 0; i < n; ++i) {
    NsMat& m = pl.mats[(size_t)i];
    // a matrix shares the machine with the others in proportion to its size
    const long others = m.kind == 0 ? work / ((long)m.Mp * m.Np) : 1;
    const NsCounts c = ns_counts(m, others, true);
    m.b0 = (int)b0; m.b1 = (int)b1; m.bg = (int)bg; m.br = (int)br; m.bc = (int)bc; m.ba = (int)ba;
    m.x = x; m.g = g; m.part = part;
    b0 += c.n0; b1 += c.n1; bg += c.ng; br += c.nr; bc += c.nc; ba += c.na; x += c.x; g += c.g; part += c.part;
    if (b0 > 0x3fffffffL || b1 > 0x3fffffffL || bg > 0x3fffffffL || ba > 0x3fffffffL || bc > 0x3fffffffL) return "too many tensors for one call";
  }
  pl.n0 = b0; pl.n1 = b1; pl.ng = bg; pl.nr = br; pl.nc = bc; pl.na = ba;
  ns_place(pl, n, x, g, part);
  pl.gr.n = n;
  return nullptr;
}

struct NsSource { int kind; const void* x; };      // kind: ns_elem's SRC

// everything behind the sums of squares.  out_kind: ns_apply_kernel's OUT of the last product
static void ns_run(const NsPlan& pl, char* w, const NsSource& in, const NsStep& step, int steps, float eps, int out_kind, void* out,
                   long ldo, hipStream_t st) {
  const NsGroup& gr = pl.gr;
  float* cfac = reinterpret_cast<float*>(w + pl.off_c);
  const double* sq = reinterpret_cast<const double*>(w + pl.off_sq);
  _Float16* xin = reinterpret_cast<_Float16*>(w + pl.off_x);
  _Float16* xout = xin + pl.x_halves;
  _Float16* g = reinterpret_cast<_Float16*>(w + pl.off_g);
  float* part = reinterpret_cast<float*>(w + pl.off_part);
  const dim3 blk(256);
  if (in.kind == 0) PG_KLAUNCH((ns_split_kernel<0>), dim3((unsigned)pl.n1), blk, 0, st, gr, in.x, step, sq, eps, cfac, xin);
  else if (in.kind == 1) PG_KLAUNCH((ns_split_kernel<1>), dim3((unsigned)pl.n1), blk, 0, st, gr, in.x, step, sq, eps, cfac, xin);
  else PG_KLAUNCH((ns_split_kernel<2>), dim3((unsigned)pl.n1), blk, 0, st, gr, in.x, step, sq, eps, cfac, xin);
  // planes between stages: |X| <= 1.21 (the quintic's largest value on [0, 1.21]), so 2^15 X fits fp16; its rms there is >= 0.5
  const float sx = 32768.f;
  bool first = true;
  while (steps > 0) {
    const int ns = steps < 3 ? steps : 3;
    steps -= ns;
    const bool last = steps == 0;
    const float* cf = first ? cfac : nullptr;
    const bool one = first && in.kind == 1;
    if (one) PG_KLAUNCH((ns_gram_kernel<1>), dim3((unsigned)pl.ng), blk, 0, st, gr, (const _Float16*)xin, part);
    else PG_KLAUNCH((ns_gram_kernel<2>), dim3((unsigned)pl.ng), blk, 0, st, gr, (const _Float16*)xin, part);
    PG_KLAUNCH(ns_gram_join_kernel, dim3((unsigned)pl.nr), blk, 0, st, gr, (const float*)part, cf, 1.f / sx, g);
    // buffers: 0 G, 1 Q, 2 Q G, 3 and 4 P in turn; the first step's Q is the first P (and keeps Q's scale)
    const float q1 = 1.f / (float)(1 << SG);
    int p = 3, psc = SG;
    for (int k = 0; k < ns; ++k) {
      const int q = k == 0 ? 3 : 1;
      const ChainJob quad = {0, 0, q, NS_C * q1, 1};
      PG_KLAUNCH(ns_chain_kernel, dim3((unsigned)pl.nc), blk, 0, st, gr, quad, quad, 1, g);
      const ChainJob qg = {q, 0, 2, q1, 0}, qp = {q, p, 7 - p, (float)ldexp(1.0, SP - SG - psc), 0}, qqg = {q, 2, 0, q1, 0};
      const bool more = k + 1 < ns;
      if (more && k > 0) PG_KLAUNCH(ns_chain_kernel, dim3((unsigned)pl.nc * 2), blk, 0, st, gr, qg, qp, 2, g);
      else if (more) PG_KLAUNCH(ns_chain_kernel, dim3((unsigned)pl.nc), blk, 0, st, gr, qg, qg, 1, g);
      else if (k > 0) PG_KLAUNCH(ns_chain_kernel, dim3((unsigned)pl.nc), blk, 0, st, gr, qp, qp, 1, g);
      if (more) PG_KLAUNCH(ns_chain_kernel, dim3((unsigned)pl.nc), blk, 0, st, gr, qqg, qqg, 1, g);
      if (k > 0) { p = 7 - p; psc = SP; }
    }
    ApplyK a;
    memset(&a, 0, sizeof(a));
    a.wsx = xin; a.wsg = g; a.wso = xout; a.pbuf = p;
    a.cfac = cf; a.cconst = 1.f / sx;
    a.mul = (float)ldexp(1.0, -psc) * (last ? 1.f : sx);
    a.out = out; a.ldo = ldo; a.s = step;
    const int o = last ? out_kind : 0;
    const dim3 gd((unsigned)pl.na);
    if (one) {
      if (o == 0) PG_KLAUNCH((ns_apply_kernel<1, 0>), gd, blk, 0, st, gr, a);
      else if (o == 1) PG_KLAUNCH((ns_apply_kernel<1, 1>), gd, blk, 0, st, gr, a);
      else PG_KLAUNCH((ns_apply_kernel<1, 2>), gd, blk, 0, st, gr, a);
    } else {
      if (o == 0) PG_KLAUNCH((ns_apply_kernel<2, 0>), gd, blk, 0, st, gr, a);
      else if (o == 1) PG_KLAUNCH((ns_apply_kernel<2, 1>), gd, blk, 0, st, gr, a);
      else if (o == 2) PG_KLAUNCH((ns_apply_kernel<2, 2>), gd, blk, 0, st, gr, a);
      else PG_KLAUNCH((ns_apply_kernel<2, 3>), gd, blk, 0, st, gr, a);
    }
    _Float16* t = xin; xin = xout; xout = t;
    first = false;
  }
}

}  // namespace pg

using namespace pg;

extern "C" int64_t pg_orthogonalise_workspace(int64_t batch, int64_t rows, int64_t cols) {
  if (batch <= 0 || rows <= 0 || cols <= 0) return 0;
  if (batch > 0x3fffffff || rows > 0x7fffffff || cols > 0x7fffffff) return -1;
  NsPlan pl{};
  return ns_plan_batch(pl, batch, rows, cols, 0, cols, 0) ? -1 : pl.bytes;
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
  NsPlan pl{};
  const char* bad = ns_plan_batch(pl, batch, rows, cols, x_batch, ldx, out_batch);
  PG_REQUIRE(bad == nullptr, "pg_orthogonalise: %s", bad);
  PG_REQUIRE(workspace && workspace_bytes >= pl.bytes, "pg_orthogonalise: workspace of %lld bytes required", (long long)pl.bytes);
  char* w = reinterpret_cast<char*>(workspace);
  hipStream_t st = (hipStream_t)stream;
  double* sq = reinterpret_cast<double*>(w + pl.off_sq);
  if (x_is_bf16) PG_KLAUNCH((ns_sumsq_kernel<1>), dim3((unsigned)pl.n0), dim3(256), 0, st, pl.gr, x, sq);
  else PG_KLAUNCH((ns_sumsq_kernel<0>), dim3((unsigned)pl.n0), dim3(256), 0, st, pl.gr, x, sq);
  const NsSource in = {x_is_bf16 ? 1 : 0, x};
  const NsStep none{};
  ns_run(pl, w, in, none, steps, eps, out_is_bf16 ? 2 : 1, out, (long)ldo, st);
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
    PG_REQUIRE(e.off + (int64_t)e.taps * e.rows * e.cols <= d->total, "pg_muon_step: entry %d ends behind the arena", i);
    PG_REQUIRE(e.kind == 0 || d->v, "pg_muon_step: an Adam entry needs v");
    if (i > 0) {
      const pg_muon_entry_t& q = d->entries[i - 1];
      PG_REQUIRE(e.off >= q.off + (int64_t)q.taps * q.rows * q.cols, "pg_muon_step: entries %d and %d overlap or are out of order", i - 1, i);
    }
  }
  PG_REQUIRE(d->workspace && d->workspace_bytes >= pl.bytes, "pg_muon_step: workspace of %lld bytes required", (long long)pl.bytes);
  hipStream_t st = (hipStream_t)stream;
  char* w = reinterpret_cast<char*>(d->workspace);
  NsMat* tab = reinterpret_cast<NsMat*>(w + pl.off_tab);
  for (size_t i = 0; i < pl.mats.size(); i += 16) {
    NsChunk c;
    const int cnt = (int)(pl.mats.size() - i < 16 ? pl.mats.size() - i : 16);
    memset(&c, 0, sizeof(c));
    memcpy(&c, &pl.mats[i], (size_t)cnt * sizeof(NsMat));
    PG_KLAUNCH(ns_table_kernel, dim3(1), dim3(64), 0, st, c, tab + i, cnt);
  }
  pl.gr.tab = tab;
  NsStep s{};
  s.p = d->p; s.g = d->g; s.gb = reinterpret_cast<const bf16_t*>(d->g_bf16); s.m = d->m; s.v = d->v;
  s.pb = reinterpret_cast<bf16_t*>(d->p_bf16);
  s.mu = d->momentum; s.gscale = d->grad_scale; s.lr = d->lr; s.wd = d->weight_decay; s.nesterov = d->nesterov;
  s.b1 = (float)d->beta1; s.b2 = (float)d->beta2; s.eps = d->adam_eps; s.b1d = d->beta1; s.b2d = d->beta2;
  s.step0 = (long)d->step; s.ctr = reinterpret_cast<const unsigned long long*>(d->ctr);
  PG_KLAUNCH(muon_momentum_kernel, dim3((unsigned)pl.n0), dim3(256), 0, st, pl.gr, s, reinterpret_cast<double*>(w + pl.off_sq));
  if (pl.ng > 0) {
    const NsSource in = {2, nullptr};
    ns_run(pl, w, in, s, d->steps, d->eps, 3, nullptr, 0, st);
  }
  PG_LAUNCH_OK("pg_muon_step");
  return 0;
}
