// muon.cu -- the Muon update of adapter matrices: momentum, then the update
// orthogonalised by Newton-Schulz steps.
//
//   buf = mu buf + g;  u = g + mu buf (Nesterov) or buf
//   X_0 = u / (|u|_F + eps);  X_{i+1} = a X_i + (b A + c A^2) X_i,  A = X_i X_i^T
//   w = w (1 - lr wd) - lr s X_n
//
// Adapters have one side of at most 16 (the rank).  With k that side and
// G = X_0 X_0^T (k x k), every X_i is P_i X_0 with P_i a polynomial of G, so
// all steps happen on k x k matrices:
//   Q = a I + b G_i + c G_i^2,  P_{i+1} = Q P_i,  G_{i+1} = Q G_i Q
// (polynomials of one matrix commute), and the long side is met twice: once
// for G and once for P_n X_0.  In between u stays in shared memory, so that
// g, buf and w are read once and buf and w written once: 20 bytes an element.
//
// A step raises a small direction by a = 3.44, five by hundreds, and G holds
// the directions' squares: in 32 bits a direction at 1e-3 of the largest would
// drown in G's rounding.  So G and P are formed in 64 bits, with the
// m8n8k4 products of the tensor pipe (3 for each 4 columns of a 16-row
// matrix, the lower left block being the upper right one's mirror image).
//
// A cluster of CTAs takes a matrix, each a share of the long side; G's parts
// meet over distributed shared memory in rank order and every CTA runs the
// small steps for itself.  Sides too long for the cluster's shared memory go
// in several tiles a CTA, and the second pass forms u again from g and buf.
#include <algorithm>
#include <cmath>

#include "common.cuh"

namespace llmcu {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kLd = 20;  // row stride of the small matrices: a fragment's 16 lanes meet 16 different bank pairs
constexpr int kMaxTile = 1536;
constexpr float kNsA = 3.4445f, kNsB = -4.7750f, kNsC = 2.0315f;

// d (8x8) += a (8x4) . b (4x8): lane l holds a[l / 4][l % 4], b[l % 4][l / 4]
// and d[l / 4][2 (l % 4) + {0, 1}].
__device__ __forceinline__ void mma_f64(double (&d)[2], double a, double b) {
  asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};"
               : "+d"(d[0]), "+d"(d[1])
               : "d"(a), "d"(b));
}

// 8 x 8 block (bi, bj) of A . B, both [8 KB, 8 KB] with row stride kLd and B
// symmetric (so that both operands' fragments are read the same way).
template <int KB>
__device__ __forceinline__ void small_product(const double* A, const double* B, int bi, int bj, int lane,
                                              double (&d)[2]) {
  d[0] = d[1] = 0.0;
  const double* pa = A + (8 * bi + (lane >> 2)) * kLd + (lane & 3);
  const double* pb = B + (8 * bj + (lane >> 2)) * kLd + (lane & 3);
#pragma unroll
  for (int s = 0; s < 2 * KB; ++s) mma_f64(d, pa[4 * s], pb[4 * s]);
}

struct Tile {
  float* u;
  int pitch;
  int k, len;        // rows, columns of this tile
  int64_t base;      // first element of the tile in the buffers (tall) / of row 0 (wide)
  int64_t row;       // wide: elements between rows
  bool tall, vec;
};

// Calls f(offset, smem index) for every element of the tile, and f4 for four
// elements that lie together in memory where the layout allows it (i[] their
// places in shared memory).
template <class F, class F4>
__device__ __forceinline__ void for_tile(const Tile& t, F f, F4 f4) {
  if (!t.tall) {
    if (t.vec) {
      const int l4 = t.len >> 2;
      for (int e = threadIdx.x; e < t.k * l4; e += kThreads) {
        const int r = e / l4, c = (e - r * l4) << 2;
        const int s = r * t.pitch + c;
        const int i[4] = {s, s + 1, s + 2, s + 3};
        f4(t.base + r * t.row + c, i);
      }
    } else {
      for (int e = threadIdx.x; e < t.k * t.len; e += kThreads) {
        const int r = e / t.len, c = e - r * t.len;
        f(t.base + r * t.row + c, r * t.pitch + c);
      }
    }
  } else {
    const int n = t.k * t.len;
    const int n4 = t.vec ? n >> 2 : 0;
    for (int e = threadIdx.x; e < n4; e += kThreads) {
      int i[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = (4 * e + j) / t.k;
        i[j] = (4 * e + j - c * t.k) * t.pitch + c;
      }
      f4(t.base + 4 * e, i);
    }
    for (int e = 4 * n4 + threadIdx.x; e < n; e += kThreads) {
      const int c = e / t.k;
      f(t.base + e, (e - c * t.k) * t.pitch + c);
    }
  }
}

template <int KB>
__global__ void __launch_bounds__(kThreads) muon_kernel(const MuonArgs a) {
  constexpr int K = 8 * KB;
  constexpr int kBlocks = KB == 2 ? 3 : 1;  // 8 x 8 blocks of G's upper half
  extern __shared__ float u[];
  __shared__ double gw[kWarps][kBlocks * 64];
  __shared__ double gpart[kBlocks * 64];
  __shared__ double G[K * kLd], Q[K * kLd], T[K * kLd], P[2][K * kLd];
  const int C = a.cluster;
  const int rank = C > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int id = blockIdx.x / C;
  const int layer = id / a.n_slots;
  const MuonSlot& sl = a.slot[id - layer * a.n_slots];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;

  Tile t;
  t.u = u;
  t.pitch = a.pitch;
  t.tall = sl.rows > sl.cols;
  t.k = min(sl.rows, sl.cols);
  const int m = max(sl.rows, sl.cols);
  t.row = sl.cols;
  const int64_t origin = layer * a.layer_stride + sl.off;
  const int tile = min(a.tile, ((m + C - 1) / C + 31) & ~31);
  const int n_tiles = (m + tile - 1) / tile;
  const bool resident = n_tiles <= C;
  const bool base_ok = ((reinterpret_cast<uintptr_t>(a.w + origin) | reinterpret_cast<uintptr_t>(a.grad + origin) |
                         reinterpret_cast<uintptr_t>(a.mom + origin)) & 15) == 0;
  auto set_tile = [&](int i) {
    const int j0 = i * tile;
    t.len = min(tile, m - j0);
    t.base = origin + static_cast<int64_t>(j0) * (t.tall ? t.k : 1);
    t.vec = base_ok && (t.tall || ((sl.cols & 3) == 0));
  };
  const float mu = a.momentum;
  const bool nesterov = a.nesterov != 0;
  // u of the tile into shared memory, zeros around it up to K rows and a
  // multiple of 8 columns
  auto load_u = [&](bool first) {
    const int l8 = (t.len + 7) & ~7;
    for (int e = threadIdx.x; e < (K - t.k) * l8; e += kThreads) {
      const int r = e / l8;
      u[(t.k + r) * t.pitch + e - r * l8] = 0.f;
    }
    for (int e = threadIdx.x; e < t.k * (l8 - t.len); e += kThreads) {
      const int r = e / (l8 - t.len);
      u[r * t.pitch + t.len + e - r * (l8 - t.len)] = 0.f;
    }
    for_tile(
        t,
        [&](int64_t o, int i) {
          const float g = a.grad[o];
          float b = a.mom[o];
          if (first) a.mom[o] = b = fmaf(mu, b, g);
          u[i] = nesterov ? fmaf(mu, b, g) : b;
        },
        [&](int64_t o, const int(&i)[4]) {
          const float4 g4 = *reinterpret_cast<const float4*>(a.grad + o);
          float4 b4 = *reinterpret_cast<const float4*>(a.mom + o);
          const float g[4] = {g4.x, g4.y, g4.z, g4.w};
          float b[4] = {b4.x, b4.y, b4.z, b4.w};
          if (first) {
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = fmaf(mu, b[j], g[j]);
            *reinterpret_cast<float4*>(a.mom + o) = make_float4(b[0], b[1], b[2], b[3]);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) u[i[j]] = nesterov ? fmaf(mu, b[j], g[j]) : b[j];
        });
  };

  // ------------------------------------------------------------ G = u u^T
  double acc[kBlocks][2];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) acc[b][0] = acc[b][1] = 0.0;
  for (int i = rank; i < n_tiles; i += C) {
    set_tile(i);
    __syncthreads();
    load_u(true);
    __syncthreads();
    const float* p0 = u + (lane >> 2) * t.pitch + (lane & 3);
    const float* p1 = p0 + 8 * t.pitch;
#pragma unroll 4
    for (int c = 4 * w; c < t.len; c += 4 * kWarps) {
      const double x0 = static_cast<double>(p0[c]);
      mma_f64(acc[0], x0, x0);
      if constexpr (KB == 2) {
        const double x1 = static_cast<double>(p1[c]);
        mma_f64(acc[1], x0, x1);
        mma_f64(acc[2], x1, x1);
      }
    }
  }
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
    gw[w][b * 64 + 2 * lane] = acc[b][0];
    gw[w][b * 64 + 2 * lane + 1] = acc[b][1];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < kBlocks * 64; e += kThreads) {
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) s += gw[i][e];
    gpart[e] = s;
  }
  if (C > 1)
    cluster_sync_all();
  else
    __syncthreads();
  for (int e = threadIdx.x; e < kBlocks * 64; e += kThreads) {
    double s = gpart[e];
    if (C > 1) {
      s = 0.0;
      const uint32_t mine = smem_u32(gpart + e);
      for (int c = 0; c < C; ++c) s += ld_cluster_f64(mapa_shared(mine, c));
    }
    // element e of block b: row e / 8, column e % 8 (lane l held d[l / 4][2 (l % 4) + {0, 1}])
    const int b = e >> 6, r = (e >> 3) & 7, c = e & 7;
    const int bi = b == 2 ? 1 : 0, bj = b == 0 ? 0 : 1;
    G[(8 * bi + r) * kLd + 8 * bj + c] = s;
    if (bi != bj) G[(8 * bj + c) * kLd + 8 * bi + r] = s;
  }
  if (C > 1)
    cluster_sync_all();  // nobody leaves while its part is read
  else
    __syncthreads();

  // ------------------------------------------------- the steps, on K x K
  double norm2 = 0.0;
  for (int i = 0; i < t.k; ++i) norm2 += G[i * kLd + i];
  const double scale = 1.0 / (sqrt(norm2) + static_cast<double>(a.eps));
  __syncthreads();
  for (int e = threadIdx.x; e < K * K; e += kThreads) G[(e / K) * kLd + e % K] *= scale * scale;
  __syncthreads();
  const int blk = w & (KB * KB - 1), bi = blk / KB, bj = blk % KB;
  const bool first_set = w < KB * KB, second_set = w >= KB * KB && w < 2 * KB * KB;
  const int at = (8 * bi + (lane >> 2)) * kLd + 8 * bj + 2 * (lane & 3);
  double d[2];
  int cur = 0;
  for (int step = 0; step < a.steps; ++step) {
    const bool last = step + 1 == a.steps;
    if (first_set) {
      small_product<KB>(G, G, bi, bj, lane, d);
      const bool diag = bi == bj;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const double one = diag && (lane >> 2) == 2 * (lane & 3) + j ? static_cast<double>(kNsA) : 0.0;
        const double q = one + static_cast<double>(kNsB) * G[at + j] + static_cast<double>(kNsC) * d[j];
        Q[at + j] = q;
        if (step == 0) P[0][at + j] = q;
      }
    }
    __syncthreads();
    if (first_set && !last) {
      small_product<KB>(Q, G, bi, bj, lane, d);
      T[at] = d[0];
      T[at + 1] = d[1];
    } else if (second_set && step > 0) {
      small_product<KB>(Q, P[cur], bi, bj, lane, d);
      P[cur ^ 1][at] = d[0];
      P[cur ^ 1][at + 1] = d[1];
    }
    if (step > 0) cur ^= 1;
    __syncthreads();
    if (first_set && !last) {
      small_product<KB>(Q, T, bi, bj, lane, d);
      G[at] = d[0];
      G[at + 1] = d[1];
    }
    __syncthreads();
  }

  // ---------------------------------------------------- w from P X_0
  double pf[KB][2 * KB];
#pragma unroll
  for (int b = 0; b < KB; ++b)
#pragma unroll
    for (int s = 0; s < 2 * KB; ++s) pf[b][s] = P[cur][(8 * b + (lane >> 2)) * kLd + 4 * s + (lane & 3)] * scale;
  const float adjust = a.match_rms ? 0.2f * sqrtf(static_cast<float>(m))
                                   : sqrtf(fmaxf(1.f, static_cast<float>(sl.rows) / static_cast<float>(sl.cols)));
  const float step_size = a.lr * adjust, keep = 1.f - a.lr * a.weight_decay;
  for (int i = rank; i < n_tiles; i += C) {
    if (!resident) {
      set_tile(i);
      __syncthreads();
      load_u(false);
      __syncthreads();
    }
    for (int c = 8 * w; c < t.len; c += 8 * kWarps) {
      double x[2 * KB];
#pragma unroll
      for (int s = 0; s < 2 * KB; ++s) x[s] = static_cast<double>(u[(4 * s + (lane & 3)) * t.pitch + c + (lane >> 2)]);
      __syncwarp();  // the warp's 8 columns are read before they are overwritten
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        double o[2] = {0.0, 0.0};
#pragma unroll
        for (int s = 0; s < 2 * KB; ++s) mma_f64(o, pf[b][s], x[s]);
        *reinterpret_cast<float2*>(u + (8 * b + (lane >> 2)) * t.pitch + c + 2 * (lane & 3)) =
            make_float2(static_cast<float>(o[0]), static_cast<float>(o[1]));
      }
    }
    __syncthreads();
    for_tile(
        t, [&](int64_t o, int s) { a.w[o] = fmaf(-step_size, u[s], keep * a.w[o]); },
        [&](int64_t o, const int(&s)[4]) {
          float4 v = *reinterpret_cast<const float4*>(a.w + o);
          v.x = fmaf(-step_size, u[s[0]], keep * v.x);
          v.y = fmaf(-step_size, u[s[1]], keep * v.y);
          v.z = fmaf(-step_size, u[s[2]], keep * v.z);
          v.w = fmaf(-step_size, u[s[3]], keep * v.w);
          *reinterpret_cast<float4*>(a.w + o) = v;
        });
  }
}

template <int KB>
cudaError_t launch(const MuonArgs& a, cudaStream_t st) {
  static std::atomic<unsigned long long> attr_set{0};
  cudaError_t e = once_per_device(attr_set, [] {
    return cudaFuncSetAttribute(muon_kernel<KB>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                8 * KB * (kMaxTile + 4) * static_cast<int>(sizeof(float)));
  });
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.layers) * a.n_slots * a.cluster);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(float) * 8 * KB * a.pitch;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = a.cluster;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = a.cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, muon_kernel<KB>, a);
}

}  // namespace

cudaError_t muon_update(MuonArgs a, cudaStream_t st) {
  if (a.n_slots < 1 || a.n_slots > kMuonMaxSlots || a.layers < 1 || a.steps < 1) return cudaErrorInvalidValue;
  int k = 0, m = 0;
  for (int i = 0; i < a.n_slots; ++i) {
    k = std::max(k, std::min(a.slot[i].rows, a.slot[i].cols));
    m = std::max(m, std::max(a.slot[i].rows, a.slot[i].cols));
  }
  if (k > kMuonMaxRank) return cudaErrorInvalidValue;
  // CTAs a matrix: as many as give each 128 columns, fewer once there are more
  // than four CTAs an SM (then a wider tile costs nothing and the small steps,
  // which every CTA runs, are run less often)
  const int64_t count = static_cast<int64_t>(a.layers) * a.n_slots;
  auto tile_of = [&](int c) { return ((m + c - 1) / c + 31) & ~31; };
  int C = 8;
  while (C > 1 && (m + C - 1) / C < 128) C /= 2;
  while (C > 1 && count * C > 4LL * gemm_num_sms() && tile_of(C / 2) <= 1024) C /= 2;
  a.cluster = C;
  a.tile = std::min(kMaxTile, tile_of(C));
  a.pitch = a.tile + 4;
  if (count * C >= (1LL << 31)) return cudaErrorInvalidValue;
  return k <= 8 ? launch<1>(a, st) : launch<2>(a, st);
}

}  // namespace llmcu
