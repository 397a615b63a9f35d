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
//
// 112 matrices of 16 x 2048 (73 MB) take 26 us, 11 at the copy rate: a CTA's
// two passes take 7 us each, half of it the 64-bit products (7 us of an SM's
// tensor pipe in all, 16 cycles each), the small steps 2 us of dependent
// products (about 55 cycles each) and the exchange of G's parts 1 us.  Loading
// a chunk ahead, or w into L2 beforehand, made neither pass faster.  All 224
// matrices of a 28-layer model's attention adapters take 47 us, where AdamW's
// seven passes take 43.
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
  double d2[2] = {0.0, 0.0};  // a second chain: a product's latency is several times its issue time
  const double* pa = A + (8 * bi + (lane >> 2)) * kLd + (lane & 3);
  const double* pb = B + (8 * bj + (lane >> 2)) * kLd + (lane & 3);
#pragma unroll
  for (int s = 0; s < 2 * KB; s += 2) {
    mma_f64(d, pa[4 * s], pb[4 * s]);
    mma_f64(d2, pa[4 * s + 4], pb[4 * s + 4]);
  }
  d[0] += d2[0];
  d[1] += d2[1];
}

// 32 columns of a matrix (fewer at its end), which one warp takes through every
// step: loading, G, the product with P and the update of w, without a word to
// the other warps, so that the warps' loads and products overlap.
constexpr int kCols = 32;
template <int kScalar>  // single elements a lane loads at once where it loads single ones
struct ChunkOf {
  int64_t base;  // its first element in the buffers
  int64_t row;   // wide: elements between rows
  float* u;      // its first column in shared memory, rows `pitch` apart
  int pitch;
  int k, len;    // rows, columns
  bool tall, vec;
  uint32_t inv;  // ceil(2^32 / k) for the tall layout's divisions; 0 for k = 1

  // x / k for x < 512
  __device__ __forceinline__ int div_k(int x) const {
    return inv ? static_cast<int>(__umulhi(static_cast<uint32_t>(x), inv)) : x;
  }
  // vec: group e < 8 k is four elements that lie together in memory
  __device__ __forceinline__ int64_t offset4(int e) const {
    return tall ? base + 4 * e : base + (e >> 3) * row + 4 * (e & 7);
  }
  __device__ __forceinline__ void put4(int e, float4 v) const {
    if (tall) {
      const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = div_k(4 * e + j);
        u[(4 * e + j - c * k) * pitch + c] = x[j];
      }
    } else {
      *reinterpret_cast<float4*>(u + (e >> 3) * pitch + 4 * (e & 7)) = v;
    }
  }
  __device__ __forceinline__ float4 get4(int e) const {
    if (tall) {
      float x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = div_k(4 * e + j);
        x[j] = u[(4 * e + j - c * k) * pitch + c];
      }
      return make_float4(x[0], x[1], x[2], x[3]);
    }
    return *reinterpret_cast<const float4*>(u + (e >> 3) * pitch + 4 * (e & 7));
  }
  // Single elements, kScalar of them at a time for each lane: turn h < turns().
  // Wide: rows kScalar h, ..., the lane's column.  Tall: in memory's order.
  __device__ __forceinline__ int turns() const {
    return tall ? (k * len + 32 * kScalar - 1) / (32 * kScalar) : (k + kScalar - 1) / kScalar;
  }
  __device__ __forceinline__ bool has(int h, int j, int lane) const {
    return tall ? (h * kScalar + j) * 32 + lane < k * len : h * kScalar + j < k && lane < len;
  }
  __device__ __forceinline__ int64_t offset(int h, int j, int lane) const {
    return tall ? base + (h * kScalar + j) * 32 + lane : base + (h * kScalar + j) * row + lane;
  }
  __device__ __forceinline__ int place(int h, int j, int lane) const {
    if (!tall) return (h * kScalar + j) * pitch + lane;
    const int e = (h * kScalar + j) * 32 + lane, c = div_k(e);
    return (e - c * k) * pitch + c;
  }
};

// VEC: every matrix can be read four elements at a time (but for the columns
// behind a multiple of 32).
template <int KB, bool VEC>
__global__ void __launch_bounds__(kThreads, 2) muon_kernel(const MuonArgs a) {
  // where single elements are the exception, fewer at once: 8 cost the others 5 us in 25
  constexpr int kScalar = VEC ? 2 : 8;
  using Chunk = ChunkOf<kScalar>;
  constexpr int K = 8 * KB;
  constexpr int kBlocks = KB == 2 ? 3 : 1;  // 8 x 8 blocks of G's upper half
  extern __shared__ __align__(16) float u[];
  __shared__ double gw[kWarps / 2][kBlocks * 64];
  __shared__ double slots[8][kBlocks * 64];  // G's parts, every CTA's
  __shared__ double G[K * kLd], Q[K * kLd], T[K * kLd], P[2][K * kLd];
  __shared__ double s_scale;
  const int C = a.cluster;
  const int rank = C > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  if (C > 1) cluster_arrive();
  pdl_trigger();
  const int id = blockIdx.x / C;
  const int layer = id / a.n_slots;
  const MuonSlot& sl = a.slot[id - layer * a.n_slots];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;

  const bool tall = sl.rows > sl.cols;
  const int k = min(sl.rows, sl.cols), m = max(sl.rows, sl.cols);
  const int64_t origin = layer * a.layer_stride + sl.off;
  const int tile = min(a.tile, ((m + C - 1) / C + 31) & ~31);
  const int n_tiles = (m + tile - 1) / tile;
  const bool resident = n_tiles <= C;
  const float mu = a.momentum;
  const bool nesterov = a.nesterov != 0;
  // chunk at column c0 of tile i
  auto chunk = [&](int i, int c0) {
    Chunk q;
    const int j0 = i * tile + c0;
    q.base = origin + static_cast<int64_t>(j0) * (tall ? k : 1);
    q.row = sl.cols;
    q.u = u + c0;
    q.pitch = a.pitch;
    q.k = k;
    q.len = min(kCols, min(m - j0, tile - c0));
    q.tall = tall;
    q.vec = VEC && q.len == kCols;
    q.inv = k > 1 ? 0xffffffffu / static_cast<uint32_t>(k) + 1u : 0u;
    return q;
  };
  auto columns = [&](int i) { return min(tile, m - i * tile); };
  // u of the chunk into shared memory, zeros behind its columns.  A lane's
  // loads are all issued before the first is used.
  auto load_u = [&](const Chunk& q, bool first) {
    if (q.vec) {
      const int n = 8 * k;
      float4 g[4], b[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = lane + 32 * j;
        if (e < n) {
          const int64_t o = q.offset4(e);
          g[j] = __ldg(reinterpret_cast<const float4*>(a.grad + o));
          b[j] = *reinterpret_cast<const float4*>(a.mom + o);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = lane + 32 * j;
        if (e < n) {
          float4 v = b[j];
          if (first) {
            v = make_float4(fmaf(mu, v.x, g[j].x), fmaf(mu, v.y, g[j].y), fmaf(mu, v.z, g[j].z),
                            fmaf(mu, v.w, g[j].w));
            *reinterpret_cast<float4*>(a.mom + q.offset4(e)) = v;
          }
          if (nesterov)
            v = make_float4(fmaf(mu, v.x, g[j].x), fmaf(mu, v.y, g[j].y), fmaf(mu, v.z, g[j].z),
                            fmaf(mu, v.w, g[j].w));
          q.put4(e, v);
        }
      }
    } else {
#pragma unroll 1
      for (int h = 0; h < q.turns(); ++h) {
        float g[kScalar], b[kScalar];
#pragma unroll
        for (int j = 0; j < kScalar; ++j) {
          if (q.has(h, j, lane)) {
            const int64_t o = q.offset(h, j, lane);
            g[j] = __ldg(a.grad + o);
            b[j] = a.mom[o];
          }
        }
#pragma unroll
        for (int j = 0; j < kScalar; ++j) {
          if (q.has(h, j, lane)) {
            float v = b[j];
            if (first) a.mom[q.offset(h, j, lane)] = v = fmaf(mu, v, g[j]);
            q.u[q.place(h, j, lane)] = nesterov ? fmaf(mu, v, g[j]) : v;
          }
        }
      }
      if (lane >= q.len)
        for (int r = 0; r < k; ++r) q.u[r * q.pitch + lane] = 0.f;
    }
    __syncwarp();
  };
  // rows k .. K - 1 stay zero: P's last rows and columns are a multiple of the identity's
  for (int e = threadIdx.x; e < (K - k) * a.pitch; e += kThreads) u[k * a.pitch + e] = 0.f;
  __syncthreads();

  // ------------------------------------------------------------ G = u u^T
  double acc[kBlocks][2];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) acc[b][0] = acc[b][1] = 0.0;
  for (int i = rank; i < n_tiles; i += C) {
    const int cols = columns(i);
    for (int c0 = kCols * w; c0 < cols; c0 += kCols * kWarps) {
      const Chunk q = chunk(i, c0);
      load_u(q, true);
      const float* p0 = q.u + (lane >> 2) * q.pitch + (lane & 3);
      const float* p1 = p0 + 8 * q.pitch;
#pragma unroll
      for (int c = 0; c < kCols; c += 4) {
        const double x0 = static_cast<double>(p0[c]);
        mma_f64(acc[0], x0, x0);
        if constexpr (KB == 2) {
          const double x1 = static_cast<double>(p1[c]);
          mma_f64(acc[1], x0, x1);
          mma_f64(acc[2], x1, x1);
        }
      }
      __syncwarp();  // a later tile's chunk lands in the same place
    }
  }
  // the warps' parts: the upper half's first, then the lower half's on top
#pragma unroll
  for (int h = 1; h >= 0; --h) {
    if ((w >= kWarps / 2) == (h == 1)) {
      double* mine = gw[w & (kWarps / 2 - 1)];
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          double& x = mine[b * 64 + 2 * lane + j];
          x = h ? acc[b][j] : x + acc[b][j];
        }
    }
    __syncthreads();
  }
  // this CTA's part to every CTA of the cluster (all of them run: they arrived
  // at the start); after the barrier all reads are local, and a CTA may leave
  // at any time
  if (C > 1) cluster_wait();
  for (int e = threadIdx.x; e < kBlocks * 64; e += kThreads) {
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < kWarps / 2; ++i) s += gw[i][e];
    if (C > 1) {
      const uint32_t to = smem_u32(&slots[rank][e]);
      for (int c = 0; c < C; ++c) st_cluster_f64(mapa_shared(to, c), s);
    } else {
      slots[0][e] = s;
    }
  }
  if (C > 1)
    cluster_sync_all();
  else
    __syncthreads();
  for (int e = threadIdx.x; e < kBlocks * 64; e += kThreads) {
    double s = 0.0;
    for (int c = 0; c < C; ++c) s += slots[c][e];
    // element e of block b: row e / 8, column e % 8 (lane l held d[l / 4][2 (l % 4) + {0, 1}])
    const int b = e >> 6, r = (e >> 3) & 7, c = e & 7;
    const int bi = b == 2 ? 1 : 0, bj = b == 0 ? 0 : 1;
    G[(8 * bi + r) * kLd + 8 * bj + c] = s;
    if (bi != bj) G[(8 * bj + c) * kLd + 8 * bi + r] = s;
  }
  __syncthreads();

  // ------------------------------------------------- the steps, on K x K
  if (w == 0) {  // |u|_F^2 is G's trace
    double d = lane < k ? G[lane * kLd + lane] : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    if (lane == 0) s_scale = 1.0 / (sqrt(d) + static_cast<double>(a.eps));
  }
  __syncthreads();
  const double scale = s_scale;
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
    const int cols = columns(i);
    for (int c0 = kCols * w; c0 < cols; c0 += kCols * kWarps) {
      const Chunk q = chunk(i, c0);
      if (!resident) load_u(q, false);
      float4 v[4];  // w of the chunk, on its way while the products are formed
      if (q.vec) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (lane + 32 * j < 8 * k) v[j] = *reinterpret_cast<const float4*>(a.w + q.offset4(lane + 32 * j));
      }
#pragma unroll
      for (int c = 0; c < kCols; c += 8) {
        double x[2 * KB];
#pragma unroll
        for (int s = 0; s < 2 * KB; ++s)
          x[s] = static_cast<double>(q.u[(4 * s + (lane & 3)) * q.pitch + c + (lane >> 2)]);
        __syncwarp();  // the 8 columns are read before they are overwritten
#pragma unroll
        for (int b = 0; b < KB; ++b) {
          double o[2] = {0.0, 0.0};
#pragma unroll
          for (int s = 0; s < 2 * KB; ++s) mma_f64(o, pf[b][s], x[s]);
          *reinterpret_cast<float2*>(q.u + (8 * b + (lane >> 2)) * q.pitch + c + 2 * (lane & 3)) =
              make_float2(static_cast<float>(o[0]), static_cast<float>(o[1]));
        }
      }
      __syncwarp();
      if (q.vec) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int e = lane + 32 * j;
          if (e < 8 * k) {
            const float4 x = q.get4(e);
            *reinterpret_cast<float4*>(a.w + q.offset4(e)) =
                make_float4(fmaf(-step_size, x.x, keep * v[j].x), fmaf(-step_size, x.y, keep * v[j].y),
                            fmaf(-step_size, x.z, keep * v[j].z), fmaf(-step_size, x.w, keep * v[j].w));
          }
        }
      } else {
#pragma unroll 1
        for (int h = 0; h < q.turns(); ++h) {
          float x[kScalar];
#pragma unroll
          for (int j = 0; j < kScalar; ++j)
            if (q.has(h, j, lane)) x[j] = a.w[q.offset(h, j, lane)];
#pragma unroll
          for (int j = 0; j < kScalar; ++j)
            if (q.has(h, j, lane))
              a.w[q.offset(h, j, lane)] = fmaf(-step_size, q.u[q.place(h, j, lane)], keep * x[j]);
        }
      }
      __syncwarp();
    }
  }
  // whoever waits for this launch waits for the ones before it
  if (a.chained) pdl_wait();
}

template <int KB, bool VEC>
cudaError_t launch(const MuonArgs& a, cudaStream_t st) {
  static std::atomic<unsigned long long> attr_set{0};
  cudaError_t e = once_per_device(attr_set, [] {
    return cudaFuncSetAttribute(muon_kernel<KB, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                8 * KB * (kMaxTile + 4) * static_cast<int>(sizeof(float)));
  });
  if (e != cudaSuccess) return e;
  return launch_cluster(muon_kernel<KB, VEC>, static_cast<unsigned>(a.layers) * a.n_slots * a.cluster, kThreads,
                        a.cluster, sizeof(float) * 8 * KB * a.pitch, st, a.chained, a);
}

// Four elements at a time: 16-byte aligned bases and strides, and for the wide
// layout rows of a multiple of four.
bool vectors(const MuonArgs& a) {
  uintptr_t bits = reinterpret_cast<uintptr_t>(a.w) | reinterpret_cast<uintptr_t>(a.grad) |
                   reinterpret_cast<uintptr_t>(a.mom);
  if (a.layers > 1) bits |= static_cast<uintptr_t>(a.layer_stride) * sizeof(float);
  for (int i = 0; i < a.n_slots; ++i) {
    bits |= static_cast<uintptr_t>(a.slot[i].off) * sizeof(float);
    if (a.slot[i].rows <= a.slot[i].cols) bits |= static_cast<uintptr_t>(a.slot[i].cols) * sizeof(float);
  }
  return bits % 16 == 0;
}

}  // namespace

cudaError_t muon_update(MuonArgs all, cudaStream_t st, int* launches) {
  if (all.n_slots < 1 || all.n_slots > kMuonMaxSlots || all.layers < 1 || all.steps < 1) return cudaErrorInvalidValue;
  auto long_side = [](const MuonSlot& s) { return std::max(s.rows, s.cols); };
  for (int i = 0; i < all.n_slots; ++i)
    if (std::min(all.slot[i].rows, all.slot[i].cols) > kMuonMaxRank) return cudaErrorInvalidValue;
  // columns a CTA: 1024, less while that leaves SMs without one (every CTA of a
  // matrix runs the small steps, so wide tiles are cheaper: 112 matrices of 16 x
  // 2048 take 26 us in pairs of CTAs and 32 in fours), down to 128
  int want = 1024;
  for (;; want /= 2) {
    int64_t ctas = 0;
    for (int i = 0; i < all.n_slots; ++i) ctas += (long_side(all.slot[i]) + want - 1) / want;
    if (want == 128 || ctas * all.layers >= gemm_num_sms()) break;
  }
  // A launch for each cluster size, a power of two of at most eight, the largest
  // first.  They work on different matrices: each may start as soon as the one
  // before it has started everywhere, and waits for its end before its own.
  bool first = true;
  for (int C = 8; C >= 1; C /= 2) {
    MuonArgs a = all;
    a.n_slots = 0;
    int k = 0, m = 0;
    for (int i = 0; i < all.n_slots; ++i) {
      const int tiles = (long_side(all.slot[i]) + want - 1) / want;
      if ((C == 1 || tiles > C / 2) && (C == 8 || tiles <= C)) {
        a.slot[a.n_slots++] = all.slot[i];
        k = std::max(k, std::min(all.slot[i].rows, all.slot[i].cols));
        m = std::max(m, long_side(all.slot[i]));
      }
    }
    if (!a.n_slots) continue;
    a.cluster = C;
    a.tile = std::min(kMaxTile, ((m + C - 1) / C + 31) & ~31);
    a.pitch = a.tile + 4;
    if (static_cast<int64_t>(a.layers) * a.n_slots * C >= (1LL << 31)) return cudaErrorInvalidValue;
    a.chained = !first;
    const bool vec = vectors(a);
    const cudaError_t e = k <= 8 ? (vec ? launch<1, true>(a, st) : launch<1, false>(a, st))
                                 : (vec ? launch<2, true>(a, st) : launch<2, false>(a, st));
    if (e != cudaSuccess) return e;
    if (launches) ++*launches;
    first = false;
  }
  return cudaSuccess;
}

}  // namespace llmcu
