// Bucketed relative-bias attention on the CUDA cores (see
// bucket_attention.cuh for the formulas): fp32 tensors, and bf16 ones that
// the tensor-core kernels do not serve (head size 16, rows that are not 16-byte
// aligned, gradients of 128 with many buckets). All products, the softmax and its sums are fp32.
//
// Tiles of 64 queries x 64 keys, 256 threads, a 4 x 4 block of scores a thread
// (queries 4 ty + i, keys tx + 16 j). Operands are staged as they are ([row][dim],
// rows padded by four words): a score product reads 16-byte pieces along the
// dims, eight of them per 64 fused multiply-adds, without bank conflicts, and
// the second products read the same rows across the dims. P and dS pass through
// shared memory with the reduced index outermost (rows of 68 words). The bias row
// of a head is spread over the map once per CTA, so a pair's bias is one shared
// load. Bound: latency and the instructions beside the FMAs (about half of all):
// 2 x 8 heads x 1,024 tokens, fp32, head size 64: 187 us forward (23 TFLOP/s),
// 672 us for the gradients (22 TFLOP/s); bf16, head size 128: 347 and 1,268 us.
//
// Backward, with P recomputed from lse:
//   dP = dO v^T,  delta_i = dO_i . out_i,  dS = P (dP - delta)
//   dv_j = sum_i P_ij dO_i,  dk_j = scale sum_i dS_ij q_i  (over the group)
//   dq_i = scale sum_j dS_ij k_j,  dbias[b, h] = sum of dS over b's pairs
// One CTA per key tile forms dk and dv, one per query tile dq and the bias
// sums, so every sum has a fixed order and no atomics are needed: a
// bias sum is kept per (bucket, query row) in shared memory by the thread
// that owns the row.
#include <algorithm>

#include "bucket_attention.cuh"

namespace mb {
namespace bucket {

constexpr int TQ = 64, TK = 64, PITCH = 68, kThreads = 256;

template <int D>
constexpr int kRow = D + 4;  // words of a staged row
template <int D>
constexpr int kCtas = D == 128 ? 1 : 2;  // per SM, as shared memory allows

// Rows [r0, r0 + 64) of a (rows, D) operand on their way through registers, so
// that a tile's loads run under the one before it; rows at or past `n` are zero.
template <typename T, int D>
struct Rows {
  T v[D / 4];
  __device__ __forceinline__ void load(const T* src, int64_t ld, int r0, int n) {
#pragma unroll
    for (int u = 0; u < D / 4; ++u) {
      const int i = threadIdx.x + u * kThreads, r = r0 + i / D;
      v[u] = r < n ? src[(int64_t)r * ld + i % D] : from_f<T>(0.f);
    }
  }
  __device__ __forceinline__ void store(float* dst) const {
#pragma unroll
    for (int u = 0; u < D / 4; ++u) {
      const int i = threadIdx.x + u * kThreads;
      dst[i / D * kRow<D> + i % D] = to_f(v[u]);
    }
  }
};
template <typename T, int D>
__device__ __forceinline__ void stage(float* dst, const T* src, int64_t ld, int r0, int n) {
  Rows<T, D> rows;
  rows.load(src, ld, r0, n);
  rows.store(dst);
}

// acc[i][j] += sum_d a[4 ty + i][d] b[tx + 16 j][d]
template <int D>
__device__ __forceinline__ void product(const float* a, const float* b, int ty, int tx, float acc[4][4]) {
#pragma unroll 4
  for (int d = 0; d < D; d += 4) {
    float4 x[4], y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const float4*>(a + (4 * ty + i) * kRow<D> + d);
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const float4*>(b + (tx + 16 * j) * kRow<D> + d);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        acc[i][j] = fmaf(x[i].x, y[j].x, acc[i][j]);
        acc[i][j] = fmaf(x[i].y, y[j].y, acc[i][j]);
        acc[i][j] = fmaf(x[i].z, y[j].z, acc[i][j]);
        acc[i][j] = fmaf(x[i].w, y[j].w, acc[i][j]);
      }
  }
}

// Column of a thread's c-th of C result columns: pieces of up to four.
template <int C>
__device__ __forceinline__ int column(int tx, int c) {
  constexpr int W = C < 4 ? C : 4;
  return c / W * 16 * W + W * tx + c % W;
}

// acc[i][c] += sum_r p[r][4 ty + i] m[r][column(c)] over 64 rows r
template <int C>
__device__ __forceinline__ void product_rows(const float* p, const float* m, int ty, int tx, float acc[4][C]) {
  constexpr int ROW = kRow<16 * C>;
#pragma unroll 4
  for (int r = 0; r < 64; ++r) {
    const float4 x = *reinterpret_cast<const float4*>(p + r * PITCH + 4 * ty);
    const float xs[4] = {x.x, x.y, x.z, x.w};
    float y[C];
    if constexpr (C >= 4) {
#pragma unroll
      for (int c = 0; c < C; c += 4) {
        const float4 v = *reinterpret_cast<const float4*>(m + r * ROW + column<C>(tx, c));
        y[c] = v.x, y[c + 1] = v.y, y[c + 2] = v.z, y[c + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int c = 0; c < C; ++c) y[c] = m[r * ROW + column<C>(tx, c)];
    }
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i][c] = fmaf(xs[i], y[c], acc[i][c]);
  }
}

__device__ __forceinline__ int2 coords_of(const Args& a, int64_t p, int r, int n) {
  const int32_t* c = a.coords + p * a.c_pos + 2 * (int64_t)r;
  return r < n ? make_int2(__ldg(c), __ldg(c + 1)) : make_int2(0, 0);
}

// The head's bias per map entry (`tab` holds the bias column behind them).
__device__ __forceinline__ void stage_bias(const Args& a, int h, float* tab) {
  spread_bias<kThreads>(a, h, tab + (2 * a.rq + 1) * (2 * a.rr + 1), [&](int i, int, float b) { tab[i] = b; });
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, kCtas<D>) forward_kernel(const Args a) {
  extern __shared__ float sm[];
  float* qt = sm;                     // [row][D + 4]
  float* kt = qt + 64 * kRow<D>;
  float* vt = kt + 64 * kRow<D>;
  float* pt = vt + 64 * kRow<D>;         // [key][68]
  int2* ck = reinterpret_cast<int2*>(pt + 64 * PITCH);
  float* tab = reinterpret_cast<float*>(ck + TK);
  const int n_tiles = (int)((a.length + TQ - 1) / TQ);
  const int tile = blockIdx.x % n_tiles, h = (blockIdx.x / n_tiles) % a.heads;
  const int64_t p = blockIdx.x / n_tiles / a.heads;
  const int kvh = h / (a.heads / a.kv_heads);
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const int nv = valid_of(a, p), q0 = tile * TQ;
  const T* qb = (const T*)a.q + p * a.sq.pos + h * a.sq.head;
  const T* kb = (const T*)a.k + p * a.sk.pos + kvh * a.sk.head;
  const T* vb = (const T*)a.v + p * a.sv.pos + kvh * a.sv.head;
  constexpr int C = D / 16;
  float o[4][C] = {}, m[4], l[4] = {};
  int2 cq[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    cq[i] = coords_of(a, p, q0 + 4 * ty + i, nv);
  }
  if (q0 < nv) {
    stage<T, D>(qt, qb, a.sq.row, q0, nv);
    stage_bias(a, h, tab);
    const float scale = a.scale * kLog2e;
    Rows<T, D> k_next, v_next;
    k_next.load(kb, a.sk.row, 0, nv);
    v_next.load(vb, a.sv.row, 0, nv);
    for (int k0 = 0; k0 < nv; k0 += TK) {
      __syncthreads();  // the last tile's operands are read
      k_next.store(kt);
      v_next.store(vt);
      if (threadIdx.x < TK) ck[threadIdx.x] = coords_of(a, p, k0 + threadIdx.x, nv);
      __syncthreads();
      k_next.load(kb, a.sk.row, k0 + TK, nv);
      v_next.load(vb, a.sv.row, k0 + TK, nv);
      float s[4][4] = {};
      product<D>(qt, kt, ty, tx, s);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float mx = m[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = tx + 16 * j;
          s[i][j] = k0 + c < nv ? fmaf(s[i][j], scale, tab[entry_of(a, cq[i], ck[c])]) : -INFINITY;
          mx = fmaxf(mx, s[i][j]);
        }
#pragma unroll
        for (int w = 8; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
        const float ref = mx == -INFINITY ? 0.f : mx;
        const float f = exp2f(m[i] - ref);
        m[i] = mx;
        l[i] *= f;
#pragma unroll
        for (int c = 0; c < C; ++c) o[i][c] *= f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float e = exp2f(s[i][j] - ref);
          l[i] += e;
          pt[(tx + 16 * j) * PITCH + 4 * ty + i] = e;
        }
      }
      __syncthreads();
      product_rows<C>(pt, vt, ty, tx, o);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float tot = l[i];
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) tot += __shfl_xor_sync(0xffffffffu, tot, w);
    const int row = q0 + 4 * ty + i;
    if (row >= a.length) continue;
    const bool live = row < nv && !(tot == 0.f);
    const float inv = live ? 1.f / tot : 0.f;
    T* orow = (T*)a.out + p * a.so.pos + h * a.so.head + row * a.so.row;
    const int64_t at = (p * a.heads + h) * a.length + row;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const float x = live ? o[i][c] * inv : 0.f;
      orow[column<C>(tx, c)] = from_f<T>(x);
      if (a.full) a.full[at * D + column<C>(tx, c)] = x;
    }
    if (a.lse && tx == 0) a.lse[at] = live ? (m[i] + log2f(tot)) * kLn2 : -INFINITY;
  }
}

// delta_i = dO_i . out_i (out before its rounding), one warp per (position, head, row).
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) delta_kernel(const Args a) {
  const int lane = threadIdx.x & 31;
  const int64_t at = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 5;
  if (at >= a.n_pos * a.heads * a.length) return;
  const int64_t row = at % a.length, h = at / a.length % a.heads, p = at / a.length / a.heads;
  float s = 0.f;
  if (a.lse_in[at] != -INFINITY) {
    const T* g = (const T*)a.grad + p * a.sg.pos + h * a.sg.head + row * a.sg.row;
    const T* o = (const T*)a.out + p * a.so.pos + h * a.so.head + row * a.so.row;
    for (int d = lane; d < D; d += 32) s = fmaf(to_f(g[d]), a.full ? a.full[at * D + d] : to_f(o[d]), s);
  }
  s = warp_sum(s);
  if (lane == 0) a.delta[at] = s;
}

// P and dS of the thread's 4 x 4 pairs (queries 4 ty + i, keys tx + 16 j).
template <int D>
__device__ __forceinline__ void pair_grads(const Args& a, const float* qt, const float* kt, const float* gt,
                                           const float* vt, const int2* cq, const int2* ck, const float* tab,
                                           const float* lse, const float* delta, int k0, int nv, int ty, int tx,
                                           float pr[4][4], float ds[4][4]) {
  float s[4][4] = {}, dp[4][4] = {};
  product<D>(qt, kt, ty, tx, s);
  product<D>(gt, vt, ty, tx, dp);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float z = lse[4 * ty + i], dl = delta[4 * ty + i];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = tx + 16 * j;
      const float x = fmaf(s[i][j], a.scale * kLog2e, tab[entry_of(a, cq[4 * ty + i], ck[c])]) - z;
      // a row without a key has z = +inf here
      const float e = k0 + c < nv ? exp2f(x) : 0.f;
      pr[i][j] = e;
      // a key with P = 0 adds nothing (a NaN stays); the only token of a position
      // has P = 1 whatever its score
      ds[i][j] = nv == 1 ? 0.f : e > 0.f ? e * (dp[i][j] - dl) : e;
    }
  }
}

// The query tile's lse (log2 units; +inf for a row without a key) and delta.
__device__ __forceinline__ void stage_rows(const Args& a, int64_t p, int h, int q0, int nv, float* lse, float* delta) {
  if (threadIdx.x < TQ) {
    const int row = q0 + threadIdx.x;
    const int64_t at = (p * a.heads + h) * a.length + row;
    const float z = row < nv ? a.lse_in[at] : -INFINITY;
    lse[threadIdx.x] = z == -INFINITY ? INFINITY : z * kLog2e;
    delta[threadIdx.x] = row < nv ? a.delta[at] : 0.f;
  }
}

template <typename T, int D>
__device__ __forceinline__ void key_grads(const Args& a, float* sm, int64_t cta) {
  float* qt = sm;
  float* kt = qt + 64 * kRow<D>;
  float* vt = kt + 64 * kRow<D>;
  float* gt = vt + 64 * kRow<D>;
  float* ps = gt + 64 * kRow<D>;         // [query][68]
  float* dss = ps + 64 * PITCH;       // [query][68]
  float* lse = dss + 64 * PITCH;
  float* delta = lse + TQ;
  int2* cq = reinterpret_cast<int2*>(delta + TQ);
  int2* ck = cq + TQ;
  float* tab = reinterpret_cast<float*>(ck + TK);
  const int n_tiles = (int)((a.length + TK - 1) / TK);
  const int tile = (int)(cta % n_tiles), kvh = (int)(cta / n_tiles % a.kv_heads);
  const int64_t p = cta / n_tiles / a.kv_heads;
  const int group = a.heads / a.kv_heads;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const int nv = valid_of(a, p), k0 = tile * TK;
  constexpr int C = D / 16;
  float dk[4][C] = {}, dv[4][C] = {};
  if (k0 < nv) {
    stage<T, D>(kt, (const T*)a.k + p * a.sk.pos + kvh * a.sk.head, a.sk.row, k0, nv);
    stage<T, D>(vt, (const T*)a.v + p * a.sv.pos + kvh * a.sv.head, a.sv.row, k0, nv);
    if (threadIdx.x < TK) ck[threadIdx.x] = coords_of(a, p, k0 + threadIdx.x, nv);
    for (int h = kvh * group; h < (kvh + 1) * group; ++h) {
      __syncthreads();
      stage_bias(a, h, tab);
      const T* qb = (const T*)a.q + p * a.sq.pos + h * a.sq.head;
      const T* gb = (const T*)a.grad + p * a.sg.pos + h * a.sg.head;
      Rows<T, D> q_next, g_next;
      q_next.load(qb, a.sq.row, 0, nv);
      g_next.load(gb, a.sg.row, 0, nv);
      for (int q0 = 0; q0 < nv; q0 += TQ) {
        __syncthreads();
        q_next.store(qt);
        g_next.store(gt);
        stage_rows(a, p, h, q0, nv, lse, delta);
        if (threadIdx.x < TQ) cq[threadIdx.x] = coords_of(a, p, q0 + threadIdx.x, nv);
        __syncthreads();
        q_next.load(qb, a.sq.row, q0 + TQ, nv);
        g_next.load(gb, a.sg.row, q0 + TQ, nv);
        float pr[4][4], ds[4][4];
        pair_grads<D>(a, qt, kt, gt, vt, cq, ck, tab, lse, delta, k0, nv, ty, tx, pr, ds);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            ps[(4 * ty + i) * PITCH + tx + 16 * j] = pr[i][j];
            dss[(4 * ty + i) * PITCH + tx + 16 * j] = ds[i][j];
          }
        __syncthreads();
        product_rows<C>(ps, gt, ty, tx, dv);  // rows of the result: keys 4 ty + i
        product_rows<C>(dss, qt, ty, tx, dk);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = k0 + 4 * ty + i;
    if (row >= a.length) continue;
    const int64_t at = ((p * a.kv_heads + kvh) * a.length + row) * D;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      ((T*)a.dk)[at + column<C>(tx, c)] = from_f<T>(dk[i][c] * a.scale);
      ((T*)a.dv)[at + column<C>(tx, c)] = from_f<T>(dv[i][c]);
    }
  }
}

template <typename T, int D>
__device__ __forceinline__ void query_grads(const Args& a, float* sm, int64_t cta) {
  float* qt = sm;
  float* kt = qt + 64 * kRow<D>;
  float* vt = kt + 64 * kRow<D>;
  float* gt = vt + 64 * kRow<D>;
  float* dst = gt + 64 * kRow<D>;        // [key][68]
  float* lse = dst + 64 * PITCH;
  float* delta = lse + TQ;
  int2* cq = reinterpret_cast<int2*>(delta + TQ);
  int2* ck = cq + TQ;
  float* hist = reinterpret_cast<float*>(ck + TK);  // [bucket][query]
  float* tab = hist + a.n_buckets * TQ;
  const int n_tiles = (int)((a.length + TQ - 1) / TQ);
  const int tile = (int)(cta % n_tiles), h = (int)(cta / n_tiles % a.heads);
  const int64_t p = cta / n_tiles / a.heads;
  const int kvh = h / (a.heads / a.kv_heads);
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const int nv = valid_of(a, p), q0 = tile * TQ;
  constexpr int C = D / 16;
  float dq[4][C] = {};
  for (int i = threadIdx.x; i < a.n_buckets * TQ; i += kThreads) hist[i] = 0.f;
  if (q0 < nv) {
    stage<T, D>(qt, (const T*)a.q + p * a.sq.pos + h * a.sq.head, a.sq.row, q0, nv);
    stage<T, D>(gt, (const T*)a.grad + p * a.sg.pos + h * a.sg.head, a.sg.row, q0, nv);
    stage_rows(a, p, h, q0, nv, lse, delta);
    if (threadIdx.x < TQ) cq[threadIdx.x] = coords_of(a, p, q0 + threadIdx.x, nv);
    stage_bias(a, h, tab);
    const T* kb = (const T*)a.k + p * a.sk.pos + kvh * a.sk.head;
    const T* vb = (const T*)a.v + p * a.sv.pos + kvh * a.sv.head;
    Rows<T, D> k_next, v_next;
    k_next.load(kb, a.sk.row, 0, nv);
    v_next.load(vb, a.sv.row, 0, nv);
    for (int k0 = 0; k0 < nv; k0 += TK) {
      __syncthreads();
      k_next.store(kt);
      v_next.store(vt);
      if (threadIdx.x < TK) ck[threadIdx.x] = coords_of(a, p, k0 + threadIdx.x, nv);
      __syncthreads();
      k_next.load(kb, a.sk.row, k0 + TK, nv);
      v_next.load(vb, a.sv.row, k0 + TK, nv);
      float pr[4][4], ds[4][4];
      pair_grads<D>(a, qt, kt, gt, vt, cq, ck, tab, lse, delta, k0, nv, ty, tx, pr, ds);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<float4*>(dst + (tx + 16 * j) * PITCH + 4 * ty) =
            make_float4(ds[0][j], ds[1][j], ds[2][j], ds[3][j]);
      __syncthreads();
      product_rows<C>(dst, kt, ty, tx, dq);
      if (a.dbias && threadIdx.x < TQ) {  // the row's pairs, in key order
        const int2 c = cq[threadIdx.x];
        for (int j = 0; j < min(TK, nv - k0); ++j) {
          const int b = bucket_of(a, entry_of(a, c, ck[j]));
          if (b >= 0) hist[b * TQ + threadIdx.x] += dst[j * PITCH + threadIdx.x];
        }
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = q0 + 4 * ty + i;
    if (row >= a.length) continue;
    const int64_t at = ((p * a.heads + h) * a.length + row) * D;
#pragma unroll
    for (int c = 0; c < C; ++c) ((T*)a.dq)[at + column<C>(tx, c)] = from_f<T>(dq[i][c] * a.scale);
  }
  if (a.dbias) {
    const int64_t parts = a.n_pos * n_tiles, part = p * n_tiles + tile;
    for (int b = threadIdx.x; b < a.n_buckets; b += kThreads) {
      float s = 0.f;
      for (int r = 0; r < TQ; ++r) s += hist[b * TQ + r];
      a.bias_part[((int64_t)h * a.n_buckets + b) * parts + part] = s;
    }
  }
}

// The key tiles' CTAs, then the query tiles' in one launch: the two are
// independent and fill the GPU together.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads, kCtas<D>) backward_kernel(const Args a, int64_t key_ctas) {
  extern __shared__ float sm[];
  if (blockIdx.x < key_ctas) key_grads<T, D>(a, sm, blockIdx.x);
  else query_grads<T, D>(a, sm, blockIdx.x - key_ctas);
}

// dbias[b, h] = the sum of its CTAs' parts: fixed strides and a fixed tree.
__global__ void __launch_bounds__(kThreads) bias_sum_kernel(const float* __restrict__ part, int64_t ctas, int heads,
                                                            int n_buckets, float* __restrict__ dbias) {
  __shared__ double ws[kThreads];
  const int h = blockIdx.x / n_buckets, b = blockIdx.x % n_buckets;
  const float* src = part + (int64_t)blockIdx.x * ctas;
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < ctas; i += kThreads) s += (double)src[i];
  ws[threadIdx.x] = s;
  for (int w = kThreads / 2; w > 0; w >>= 1) {
    __syncthreads();
    if (threadIdx.x < w) ws[threadIdx.x] += ws[threadIdx.x + w];
  }
  if (threadIdx.x == 0) dbias[(int64_t)b * heads + h] = (float)ws[0];
}

inline size_t map_bytes(const Args& a) {
  return ((size_t)(2 * a.rq + 1) * (2 * a.rr + 1) + a.n_buckets) * 4;
}

template <typename T, int D>
int simt_forward(const Args& a, cudaStream_t s) {
  const size_t smem = (3 * 64 * kRow<D> + 64 * PITCH) * 4 + TK * 8 + map_bytes(a);
  auto kern = forward_kernel<T, D>;
  if (int rc = configure(kern, smem, "bucket_attention")) return rc;
  const int64_t ctas = a.n_pos * a.heads * cdiv(a.length, TQ);
  kern<<<(unsigned)ctas, kThreads, smem, s>>>(a);
  return launch_status("bucket_attention");
}

template <typename T, int D>
int simt_delta(const Args& a, cudaStream_t s) {
  delta_kernel<T, D><<<(unsigned)cdiv(a.n_pos * a.heads * a.length, kThreads / 32), kThreads, 0, s>>>(a);
  return launch_status("bucket_attention_backward");
}

template <typename T, int D>
int simt_backward(const Args& a, cudaStream_t s) {
  const size_t common = 4 * 64 * kRow<D> * 4 + 2 * TQ * 4 + (TQ + TK) * 8 + map_bytes(a);
  const size_t keys = common + 2 * 64 * PITCH * 4, queries = common + 64 * PITCH * 4 + (size_t)a.n_buckets * TQ * 4;
  const size_t smem = std::max(keys, queries);
  auto kern = backward_kernel<T, D>;
  if (int rc = configure(kern, smem, "bucket_attention_backward")) return rc;
  if (int rc = simt_delta<T, D>(a, s)) return rc;
  const int64_t tiles = cdiv(a.length, TQ), key_ctas = a.n_pos * a.kv_heads * tiles;
  kern<<<(unsigned)(key_ctas + a.n_pos * a.heads * tiles), kThreads, smem, s>>>(a, key_ctas);
  return launch_status("bucket_attention_backward");
}

inline int bias_sum(const Args& a, int64_t ctas, cudaStream_t s) {
  bias_sum_kernel<<<(unsigned)(a.heads * a.n_buckets), kThreads, 0, s>>>(a.bias_part, ctas, a.heads, a.n_buckets,
                                                                        a.dbias);
  return launch_status("bucket_attention_backward");
}

// The workspace's words ahead of delta: on the tensor cores the dQ and dK / dV
// parts and the bias sums of the plan's CTAs; on the CUDA cores, which serve bf16
// rows off 16 bytes too, the bias sums of every query tile and no parts.
inline int64_t front_words(const BackwardPlan& plan, bool tensor_cores, int64_t n_pos, int heads, int64_t length,
                           int n_buckets) {
  const int64_t sums = (int64_t)heads * n_buckets;
  return tensor_cores ? plan.dq_words + plan.dkv_words + plan.ctas * sums : n_pos * cdiv(length, TQ) * sums;
}

inline int check(const Args& a, int dtype, const char* what) {
  MB_REQUIRE(valid_dtype(dtype), "%s: bad dtype", what);
  MB_REQUIRE(a.n_pos >= 0 && a.length >= 0 && a.heads > 0 && a.kv_heads > 0 && a.heads % a.kv_heads == 0,
             "%s: bad sizes (heads must be a multiple of kv_heads)", what);
  MB_REQUIRE(a.dim == 16 || a.dim == 32 || a.dim == 64 || a.dim == 128, "%s: head_dim %d unsupported", what, a.dim);
  MB_REQUIRE(a.n_buckets > 0 && a.n_buckets <= kMaxBuckets, "%s: n_buckets must be in [1, %d] (got %d)", what,
             kMaxBuckets, a.n_buckets);
  MB_REQUIRE(a.rq >= 0 && a.rr >= 0 && a.rq <= kMaxMap && a.rr <= kMaxMap &&
                 (int64_t)(2 * a.rq + 1) * (2 * a.rr + 1) <= kMaxMap,
             "%s: the bucket map must have at most %d entries", what, kMaxMap);
  MB_REQUIRE(a.length <= (1 << 24) && (a.length == 0 || a.n_pos <= INT32_MAX / 2 / a.heads / cdiv(a.length, TQ)),
             "%s: too many tiles", what);
  return MB_OK;
}

// A body over the tensors' type and head size.
#define MB_BUCKET_DISPATCH(dtype, dim, fn, ...)               \
  [&]() -> int {                                              \
    int rc_ = MB_OK;                                          \
    MB_DISPATCH_T(dtype, T, [&] {                             \
      if ((dim) == 16) rc_ = fn<T, 16>(__VA_ARGS__);          \
      else if ((dim) == 32) rc_ = fn<T, 32>(__VA_ARGS__);     \
      else if ((dim) == 64) rc_ = fn<T, 64>(__VA_ARGS__);     \
      else rc_ = fn<T, 128>(__VA_ARGS__);                     \
    });                                                       \
    return rc_;                                               \
  }()

}  // namespace bucket
}  // namespace mb

using namespace mb;

extern "C" {

int mb_bucket_attention(const void* q, const void* k, const void* v, int dtype, int64_t n_pos, int heads, int kv_heads,
                        int head_dim, int64_t length, int64_t q_pos, int64_t q_head, int64_t q_row, int64_t k_pos,
                        int64_t k_head, int64_t k_row, int64_t v_pos, int64_t v_head, int64_t v_row, float scale,
                        const float* bias, int n_buckets, const int32_t* bucket_map, int radius_q, int radius_r,
                        const int32_t* coords, int64_t c_pos, const int32_t* valid, void* out, int64_t o_pos,
                        int64_t o_head, int64_t o_row, float* full, float* lse, void* stream) {
  bucket::Args a = {};
  a.q = q, a.k = k, a.v = v;
  a.sq = {q_pos, q_head, q_row}, a.sk = {k_pos, k_head, k_row}, a.sv = {v_pos, v_head, v_row};
  a.n_pos = n_pos, a.length = length, a.heads = heads, a.kv_heads = kv_heads, a.dim = head_dim;
  a.scale = scale, a.bias = bias, a.n_buckets = n_buckets, a.map = bucket_map, a.rq = radius_q, a.rr = radius_r;
  a.coords = coords, a.c_pos = c_pos, a.valid = valid;
  a.out = out, a.so = {o_pos, o_head, o_row}, a.full = full, a.lse = lse;
  if (int rc = bucket::check(a, dtype, "bucket_attention")) return rc;
  if (n_pos == 0 || length == 0) return MB_OK;
  MB_REQUIRE(q && k && v && bias && bucket_map && coords && out, "bucket_attention: null pointer");
  cudaStream_t s = as_stream(stream);
  if (bucket::tc_serves(a, dtype)) return bucket::tc_forward(a, s);
  return MB_BUCKET_DISPATCH(dtype, head_dim, bucket::simt_forward, a, s);
}

int mb_bucket_attention_limit_parts(int64_t bytes) {
  MB_REQUIRE(bytes >= 0, "bucket_attention_limit_parts: negative size");
  bucket::part_limit.store(bytes / 4 + (bytes % 4 != 0), std::memory_order_relaxed);
  return MB_OK;
}

int mb_bucket_attention_workspace(int dtype, int64_t n_pos, int heads, int kv_heads, int head_dim, int64_t length,
                                  int n_buckets, int64_t* bytes) {
  MB_REQUIRE(bytes, "bucket_attention_workspace: null pointer");
  MB_REQUIRE(valid_dtype(dtype) && n_pos >= 0 && heads > 0 && kv_heads > 0 && head_dim > 0 && length >= 0 &&
                 n_buckets > 0,
             "bucket_attention_workspace: bad sizes");
  const bucket::BackwardPlan plan = bucket::backward_plan(n_pos, heads, kv_heads, head_dim, length, dtype);
  *bytes = 4 * (std::max(bucket::front_words(plan, false, n_pos, heads, length, n_buckets),
                         bucket::front_words(plan, true, n_pos, heads, length, n_buckets)) +
                n_pos * heads * length);
  return MB_OK;
}

int mb_bucket_attention_backward(const void* q, const void* k, const void* v, int dtype, int64_t n_pos, int heads,
                                 int kv_heads, int head_dim, int64_t length, int64_t q_pos, int64_t q_head,
                                 int64_t q_row, int64_t k_pos, int64_t k_head, int64_t k_row, int64_t v_pos,
                                 int64_t v_head, int64_t v_row, float scale, const float* bias, int n_buckets,
                                 const int32_t* bucket_map, int radius_q, int radius_r, const int32_t* coords,
                                 int64_t c_pos, const int32_t* valid, const void* out, int64_t o_pos, int64_t o_head,
                                 int64_t o_row, const float* full, const float* lse, const void* grad_out,
                                 int64_t g_pos, int64_t g_head, int64_t g_row, void* workspace,
                                 int64_t workspace_bytes, void* dq, void* dk, void* dv, float* dbias, void* stream) {
  bucket::Args a = {};
  a.q = q, a.k = k, a.v = v;
  a.sq = {q_pos, q_head, q_row}, a.sk = {k_pos, k_head, k_row}, a.sv = {v_pos, v_head, v_row};
  a.n_pos = n_pos, a.length = length, a.heads = heads, a.kv_heads = kv_heads, a.dim = head_dim;
  a.scale = scale, a.bias = bias, a.n_buckets = n_buckets, a.map = bucket_map, a.rq = radius_q, a.rr = radius_r;
  a.coords = coords, a.c_pos = c_pos, a.valid = valid;
  a.out = const_cast<void*>(out), a.so = {o_pos, o_head, o_row}, a.full = const_cast<float*>(full), a.lse_in = lse;
  a.grad = grad_out, a.sg = {g_pos, g_head, g_row};
  a.dq = dq, a.dk = dk, a.dv = dv, a.dbias = dbias;
  if (int rc = bucket::check(a, dtype, "bucket_attention_backward")) return rc;
  cudaStream_t s = as_stream(stream);
  if (n_pos == 0 || length == 0) {
    if (dbias && cudaMemsetAsync(dbias, 0, sizeof(float) * n_buckets * heads, s) != cudaSuccess)
      return launch_status("bucket_attention_backward");
    return MB_OK;
  }
  MB_REQUIRE(q && k && v && bias && bucket_map && coords && out && lse && grad_out && workspace && dq && dk && dv,
             "bucket_attention_backward: null pointer");
  // one plan for the whole call: the limit on parts may change beside it
  const bucket::BackwardPlan plan = bucket::backward_plan(n_pos, heads, kv_heads, head_dim, length, dtype);
  const bool tensor_cores = bucket::tc_serves(a, dtype);
  const int64_t front = bucket::front_words(plan, tensor_cores, n_pos, heads, length, n_buckets);
  const int64_t need = 4 * (front + n_pos * heads * length);
  MB_REQUIRE(workspace_bytes >= need && aligned(workspace, 16),
             "bucket_attention_backward: the workspace needs %lld bytes, 16-byte aligned", (long long)need);
  a.dq_part = (float*)workspace;
  a.dkv_part = a.dq_part + plan.dq_words;
  a.bias_part = tensor_cores ? a.dkv_part + plan.dkv_words : a.dq_part;
  a.delta = (float*)workspace + front;
  int64_t parts = n_pos * cdiv(length, bucket::TQ);  // of a bias sum
  if (tensor_cores) {
    if (int rc = bucket::tc_backward(a, plan, s)) return rc;
    parts = plan.ctas;
  } else {
    if (int rc = MB_BUCKET_DISPATCH(dtype, head_dim, bucket::simt_backward, a, s)) return rc;
  }
  return dbias ? bucket::bias_sum(a, parts, s) : MB_OK;
}

}  // extern "C"
