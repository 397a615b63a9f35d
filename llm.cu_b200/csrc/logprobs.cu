// logprobs.cu -- token log-probabilities straight from hidden states and the
// (frozen) output head, and their gradient with respect to the hidden states:
//
//   l[m, v] = x[m] . E[v],  lse[m] = log sum_v exp l[m, v],
//   logp[m] = l[m, t_m] - lse[m]
//   dx[m]   = scale * dlogp[m] * ((1 - p_t) E[t_m] - sum_{v != t} p_v E[v]),  p = exp(l - lse)
//
// No [M, V] logits are formed.  The forward is one GEMM over the whole
// vocabulary whose epilogue keeps a maximum and a sum per 128 columns; the
// backward forms the probabilities again a vocabulary chunk at a time and
// multiplies each chunk with its rows of E.
#include <algorithm>
#include <cmath>

#include "common.cuh"

namespace llmcu {

namespace {

// Two (max, sum of exp(l - max)) pairs as one.
__device__ __forceinline__ float2 join_pairs(float2 a, float2 b) {
  const float n = fmaxf(a.x, b.x);
  // both maxima -inf: the sums are 0, or a NaN
  const float s = n > -INFINITY ? a.y * exp2f((a.x - n) * kLog2e) + b.y * exp2f((b.x - n) * kLog2e) : a.y + b.y;
  return make_float2(n, s);
}

// x . e in fp32 by one warp (the same order of sums wherever it is called):
// the target's logit.  The tensor cores cut what they add to the accumulator,
// which leaves a logit of 10 about 3e-5 short after 128 steps of K; over the
// sum of the exponentials that hardly shows, in l_t - lse it does.
__device__ __forceinline__ float target_logit(const __half* __restrict__ x, const __half* __restrict__ e, int H,
                                              int lane) {
  float s = 0.f;
  const int h8 = H & ~7;  // rows start on 16 bytes
  for (int c = lane * 8; c < h8; c += 256) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(x + c));
    const uint4 b = __ldg(reinterpret_cast<const uint4*>(e + c));
    const __half2* ha = reinterpret_cast<const __half2*>(&a);
    const __half2* hb = reinterpret_cast<const __half2*>(&b);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 u = __half22float2(ha[j]), v = __half22float2(hb[j]);
      s = fmaf(u.x, v.x, fmaf(u.y, v.y, s));
    }
  }
  if (h8 + lane < H) s = fmaf(__half2float(x[h8 + lane]), __half2float(e[h8 + lane]), s);
  return warp_sum(s);
}

// The pair p with one of its terms, the logit `rough`, replaced by `exact`.
__device__ __forceinline__ float2 replace_term(float2 p, float rough, float exact) {
  const float d = exact - rough;
  if (fabsf(d) < 1.f) {
    p.y = fmaf(exp2f((rough - p.x) * kLog2e), expm1f(d), p.y);
  } else if (isfinite(d)) {
    // logits of 1e5 and more, whose roundings pass 1: what is left without the
    // term (nothing, where it was nearly all), joined with it
    const float rest = p.y - exp2f((rough - p.x) * kLog2e);
    p = rest > 1e-6f * p.y ? join_pairs(make_float2(p.x, rest), make_float2(exact, 1.f)) : make_float2(exact, 1.f);
  }
  return p;
}

constexpr int kWarps = 32;  // of the forward's finishing kernel: they share the slots

// One row: the vocabulary is read once by plain loads and multiplied on the
// CUDA cores, in fp32.  What bounds it is reading E: 622 MB for 151936 x 2048
// is 95 us at the measured copy rate; with its finishing kernel it takes 103,
// where the GEMM takes 120.  Smaller heads go the same way: 6.4 us against 7.2
// for 128 x 64, 6.7 / 8.2 for 4096 x 256, 9.0 / 11.5 for 32000 x 256, 18.4 / 19.7
// for 8192 x 2048, 35 / 44 for 40000 x 2048 (4096 x 2048 alone is 17.8 / 17.2).
// From two rows on the GEMM takes all: there the products outweigh the loads (a
// kernel like this one took 113 us for two rows and 148 for four at 151936 x
// 2048, the GEMM 110).
//
// A warp takes four rows of E at a time, a lane eight elements of each every
// 256; x lies in shared memory as fp32, its halves of eight apart, so that a
// warp's 16-byte reads meet every bank once.  The four logits meet in all
// lanes, which keep the running maximum and sum.
constexpr int kOneThreads = 512;
constexpr int kOneBlocks = 2;  // CTAs an SM
constexpr int kOneSmem = 96 * 1024;
constexpr int kVecRows = 4;    // rows of E a warp takes at once

__global__ void __launch_bounds__(kOneThreads, kOneBlocks)
    one_row_kernel(const __half* __restrict__ x, const __half* __restrict__ E, const int* __restrict__ targets, int H,
                   int V, int lde, float2* __restrict__ part, float* __restrict__ tgt_logit) {
  extern __shared__ __align__(16) float xs[];  // [h256]
  __shared__ float2 red[kOneThreads / 32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int h256 = (H + 255) & ~255;
  for (int k = threadIdx.x; k < h256; k += kOneThreads)
    xs[(k & ~255) + (k & 4) * 32 + ((k & 255) >> 3) * 4 + (k & 3)] = k < H ? __half2float(x[k]) : 0.f;
  pdl_trigger();
  __syncthreads();
  float2 p = make_float2(-INFINITY, 0.f);
  const int t = *targets;
  // a run of E's rows for each warp of the grid
  const int warps = gridDim.x * (kOneThreads / 32);
  const int me = blockIdx.x * (kOneThreads / 32) + w;
  const int v_end = static_cast<int>(static_cast<int64_t>(V) * (me + 1) / warps);
  for (int v0 = static_cast<int>(static_cast<int64_t>(V) * me / warps); v0 < v_end; v0 += kVecRows) {
    float acc[kVecRows] = {};
    const __half* row[kVecRows];  // past the run: its last row again, not used
#pragma unroll
    for (int r = 0; r < kVecRows; ++r) row[r] = E + static_cast<size_t>(min(v0 + r, v_end - 1)) * lde;
#pragma unroll 2
    for (int k0 = 0; k0 < h256; k0 += 256) {
      const int k = k0 + lane * 8;
      uint4 e[kVecRows];
#pragma unroll
      for (int r = 0; r < kVecRows; ++r) {
        e[r] = make_uint4(0u, 0u, 0u, 0u);
        if (k + 8 <= H) {
          e[r] = __ldcs(reinterpret_cast<const uint4*>(row[r] + k));
        } else if (k < H) {
          __half* h = reinterpret_cast<__half*>(&e[r]);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (k + j < H) h[j] = row[r][k + j];
        }
      }
      const float4 a = *reinterpret_cast<const float4*>(xs + k0 + lane * 4);
      const float4 b = *reinterpret_cast<const float4*>(xs + k0 + 128 + lane * 4);
#pragma unroll
      for (int r = 0; r < kVecRows; ++r) {
        const __half2* h = reinterpret_cast<const __half2*>(&e[r]);
        const float2 f0 = __half22float2(h[0]), f1 = __half22float2(h[1]), f2 = __half22float2(h[2]),
                     f3 = __half22float2(h[3]);
        float c = acc[r];
        c = fmaf(a.x, f0.x, c);
        c = fmaf(a.y, f0.y, c);
        c = fmaf(a.z, f1.x, c);
        c = fmaf(a.w, f1.y, c);
        c = fmaf(b.x, f2.x, c);
        c = fmaf(b.y, f2.y, c);
        c = fmaf(b.z, f3.x, c);
        acc[r] = fmaf(b.w, f3.y, c);
      }
    }
    float l[kVecRows];
    float n = p.x;
#pragma unroll
    for (int r = 0; r < kVecRows; ++r) {
      const float v = warp_sum(acc[r]);
      l[r] = v0 + r < v_end ? v : -INFINITY;
      if (v0 + r == t && v0 + r < v_end && lane == 0) *tgt_logit = v;
      n = fmaxf(n, l[r]);
    }
    if (n > -INFINITY) {
      float s = p.y * exp2f((p.x - n) * kLog2e);
#pragma unroll
      for (int r = 0; r < kVecRows; ++r) s += exp2f((l[r] - n) * kLog2e);
      p = make_float2(n, s);
    } else {  // -inf so far, or NaN: the sum keeps the NaN
#pragma unroll
      for (int r = 0; r < kVecRows; ++r) p.y += l[r] == -INFINITY ? 0.f : l[r];
    }
  }
  if (lane == 0) red[w] = p;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kOneThreads / 32; ++i) p = join_pairs(p, red[i]);
    part[blockIdx.x] = p;
  }
}

cudaError_t one_row(const __half* x, const __half* E, const int* targets, int H, int V, int lde, float2* part,
                    float* tgt_logit, int blocks, cudaStream_t st) {
  static std::atomic<unsigned long long> attr_set{0};
  cudaError_t e = once_per_device(attr_set, [] {
    return cudaFuncSetAttribute(one_row_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kOneSmem);
  });
  if (e != cudaSuccess) return e;
  return launch_pdl(one_row_kernel, blocks, kOneThreads, sizeof(float) * ((H + 255) & ~255), st, x, E, targets, H, V,
                    lde, part, tgt_logit);
}

// Joins the slots' (max, sum) pairs, RB rows a CTA: lane l of warp w takes row
// l % RB of slots w * (32 / RB) + l / RB, and every 32 * (32 / RB)th on.  Before
// that, while the GEMM still runs, warp w forms row w's target logit (x, E and
// the targets are complete before the GEMM starts); it also replaces the GEMM's
// value in the sum.  Four rows a CTA (32-byte pieces of the pairs, [slot][row])
// while that is at most two CTAs an SM, else 32; at most 32 warps a CTA, fewer
// where there are fewer slots to share.
template <int RB>
__global__ void __launch_bounds__(32 * kWarps)
    logprob_finish_kernel(const float2* __restrict__ part, const float* __restrict__ tgt_logit,
                          const int* __restrict__ targets, const __half* __restrict__ x, const __half* __restrict__ E,
                          int M, int H, int V, int ldx, int lde, int slots, float* __restrict__ logp,
                          float* __restrict__ lse) {
  pdl_trigger();
  __shared__ float2 red[kWarps][RB + 1];  // + 1: read down its columns
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  const int row = blockIdx.x * RB + w;
  const int t = w < RB && row < M ? targets[row] : -1;
  const bool ok = t >= 0 && t < V;
  float exact = 0.f;
  if (ok) exact = target_logit(x + static_cast<size_t>(row) * ldx, E + static_cast<size_t>(t) * lde, H, lane);
  pdl_wait();
  const int m = blockIdx.x * RB + lane % RB;
  float2 p = make_float2(-INFINITY, 0.f);
  if (m < M) {
#pragma unroll 4
    for (int i = w * (32 / RB) + lane / RB; i < slots; i += nw * (32 / RB))
      p = join_pairs(p, part[static_cast<size_t>(i) * M + m]);
  }
#pragma unroll
  for (int o = 16; o >= RB; o >>= 1)
    p = join_pairs(p, make_float2(__shfl_xor_sync(0xffffffffu, p.x, o), __shfl_xor_sync(0xffffffffu, p.y, o)));
  if (lane < RB) red[w][lane] = p;
  __syncthreads();
  if (w >= RB || row >= M) return;
  p = lane < nw ? red[lane][w] : make_float2(-INFINITY, 0.f);  // the warps' parts of row w
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    p = join_pairs(p, make_float2(__shfl_xor_sync(0xffffffffu, p.x, o), __shfl_xor_sync(0xffffffffu, p.y, o)));
  if (lane == 0) {
    if (ok) p = replace_term(p, tgt_logit[row], exact);
    const float ls = logf(p.y);
    lse[row] = p.x + ls;
    logp[row] = ok ? (exact - p.x) - ls : 0.f;  // not through lse, whose rounding a confident token would show
  }
}

// The same for the training step's streamed head, whose partials lie [row][slot]
// as separate references and sums: a warp a row.
constexpr int kStreamWarps = 8;
__global__ void __launch_bounds__(32 * kStreamWarps)
    stream_logp_kernel(const float* __restrict__ part_ref, const float* __restrict__ part_sum,
                       const float* __restrict__ tgt_logit, const int* __restrict__ targets,
                       const __half* __restrict__ x, const __half* __restrict__ E, int M, int H, int V, int slots,
                       float* __restrict__ logp) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int m = blockIdx.x * kStreamWarps + (threadIdx.x >> 5);
  if (m >= M) return;
  const int t = targets[m];
  if (t < 0 || t >= V) {
    if (lane == 0) logp[m] = 0.f;
    return;
  }
  const float exact = target_logit(x + static_cast<size_t>(m) * H, E + static_cast<size_t>(t) * H, H, lane);
  const float* pr = part_ref + static_cast<size_t>(m) * slots;
  const float* ps = part_sum + static_cast<size_t>(m) * slots;
  float mx = -INFINITY;
  for (int i = lane; i < slots; i += 32) mx = fmaxf(mx, pr[i]);
  mx = warp_max(mx);
  float s = 0.f;
  for (int i = lane; i < slots; i += 32) s += ps[i] * exp2f((pr[i] - mx) * kLog2e);
  s = warp_sum(s);
  if (lane == 0) {
    const float2 p = replace_term(make_float2(mx, s), tgt_logit[m], exact);
    logp[m] = (exact - p.x) - logf(p.y);
  }
}

// The rows that have a gradient -- their target lies in the vocabulary and
// their upstream gradient is not 0 -- in order: list[0 .. *count), and each
// row's place there (or -1).  One CTA.
__global__ void __launch_bounds__(1024)
    live_rows_kernel(const int* __restrict__ targets, const float* __restrict__ dlogp, int M, int V,
                     int* __restrict__ list, int* __restrict__ place, int* __restrict__ count) {
  pdl_trigger();
  __shared__ int warps[32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int base = 0;
  for (int m0 = 0; m0 < M; m0 += 4 * 1024) {
    bool live[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // the loads of four turns at once
      const int m = m0 + j * 1024 + threadIdx.x;
      live[j] = m < M && targets[m] >= 0 && targets[m] < V && dlogp[m] != 0.f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + j * 1024 + threadIdx.x;
      if (m0 + j * 1024 >= M) break;
      const uint32_t b = __ballot_sync(0xffffffffu, live[j]);
      if (lane == 0) warps[w] = __popc(b);
      __syncthreads();
      const int mine = warps[lane];
      const int total = __reduce_add_sync(0xffffffffu, mine);
      const int before = __reduce_add_sync(0xffffffffu, lane < w ? mine : 0);
      const int at = base + before + __popc(b & ((1u << lane) - 1u));
      if (live[j]) list[at] = m;
      if (m < M) place[m] = live[j] ? at : -1;
      base += total;
      __syncthreads();
    }
  }
  if (threadIdx.x == 0) *count = base;
}

// x, lse and targets of those rows, one after another (a warp a row).
__global__ void __launch_bounds__(256)
    gather_rows_kernel(const __half* __restrict__ x, int ldx, const float* __restrict__ lse,
                       const int* __restrict__ targets, const int* __restrict__ list, const int* __restrict__ count,
                       int H, __half* __restrict__ xc, int ldc, float* __restrict__ lsec, int* __restrict__ tc) {
  pdl_trigger();
  pdl_wait();
  const int i = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (i >= *count) return;
  const int m = list[i];
  const __half* src = x + static_cast<size_t>(m) * ldx;  // rows start on 16 bytes
  __half* dst = xc + static_cast<size_t>(i) * ldc;
  for (int c = lane * 8; c < H; c += 256) {
    if (c + 8 <= H) {
      *reinterpret_cast<uint4*>(dst + c) = __ldg(reinterpret_cast<const uint4*>(src + c));
    } else {
      for (int j = c; j < H; ++j) dst[j] = src[j];
    }
  }
  if (lane == 0) {
    lsec[i] = lse[m];
    tc[i] = targets[m];
  }
}

// dx row m from the K slices' partial sums (slab k: rows [k * slab_rows, ...)
// of acc), in slice order, and the target's own term in fp32.  A warp takes
// `cols` columns of a row (parts of them for each row).
__global__ void __launch_bounds__(256)
    logprob_dx_kernel(const float* __restrict__ acc, int slabs, int slab_rows, int ld_acc,
                      const int* __restrict__ place, const __half* __restrict__ x, int ldx,
                      const __half* __restrict__ E, int lde, const float* __restrict__ lse,
                      const float* __restrict__ dlogp, const int* __restrict__ targets, int M, int H, int V,
                      float scale, __half* __restrict__ dx, int lddx, int cols, int parts) {
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int64_t item = blockIdx.x * static_cast<int64_t>(8) + (threadIdx.x >> 5);
  const int m = static_cast<int>(item / parts);
  if (m >= M) return;
  const int c0 = static_cast<int>(item - static_cast<int64_t>(m) * parts) * cols;
  const int t = targets[m];
  const bool ok = t >= 0 && t < V;
  const __half* et = E + static_cast<size_t>(ok ? t : 0) * lde;
  // inputs alone: while the last GEMM still runs
  const float exact = ok ? target_logit(x + static_cast<size_t>(m) * ldx, et, H, lane) : 0.f;
  const float up = dlogp[m];
  // 1 - p_t without cancellation for a confident token
  const float one_minus = ok ? -expm1f(exact - lse[m]) : 0.f;
  pdl_wait();
  const int at = place ? place[m] : m;  // the row of the partial sums; -1: it has no gradient
  const bool live = ok && at >= 0 && up != 0.f;  // else 0, whatever x and the sums hold
  const float g = scale * up;
  const float unshift = exp2f(-kProbShift);
  const float* a0 = acc + static_cast<size_t>(max(at, 0)) * ld_acc;
  const size_t slab = static_cast<size_t>(slab_rows) * ld_acc;
  __half* out = dx + static_cast<size_t>(m) * lddx;
  const bool vec = (reinterpret_cast<uintptr_t>(dx) & 7) == 0 && (lddx & 3) == 0;
  const int end = min(H, c0 + cols);
  for (int c = c0 + lane * 4; c < end; c += 128) {
    float r[4] = {0.f, 0.f, 0.f, 0.f};
    if (live) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
      for (int k = 0; k < slabs; ++k) {  // ld_acc is a multiple of 4; what lies past H is not used
        const float4 o = *reinterpret_cast<const float4*>(a0 + k * slab + c);
        v.x += o.x;
        v.y += o.y;
        v.z += o.z;
        v.w += o.w;
      }
      const float sum[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < H) r[j] = g * fmaf(one_minus, __half2float(et[c + j]), -unshift * sum[j]);
    }
    if (vec && c + 4 <= H) {
      uint2 u;
      u.x = pack_half2(r[0], r[1]);
      u.y = pack_half2(r[2], r[3]);
      *reinterpret_cast<uint2*>(out + c) = u;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < H) out[c + j] = __float2half_rn(r[j]);
    }
  }
}

// The backward's split of the vocabulary.
struct BwdPlan {
  int vc;         // columns per chunk: a multiple of 1024, or all of V
  int ksplit;     // K slices asked of each chunk's dx GEMM
  int slabs;      // slices the widest chunk really has
  int slab_rows;  // rows of one slice's partial sums
  int ld_acc;
};

// 128 MiB of fp16 probabilities a chunk, as for the training step's head
// (16384 columns at 4096 rows).  Few rows take the whole vocabulary at once:
// 130 rows in 16384-column chunks, whose rows of E the second product would
// find in L2, ran 525 us against 294 in one chunk.
constexpr size_t kChunkElems = static_cast<size_t>(64) << 20;

BwdPlan bwd_plan(int M, int H, int V) {
  BwdPlan p;
  p.ld_acc = (H + 3) / 4 * 4;
  p.slab_rows = (M + 255) / 256 * 256;
  const size_t fit = std::max<size_t>(1024, kChunkElems / static_cast<size_t>(M) / 1024 * 1024);
  p.vc = static_cast<int>(std::min<size_t>(fit, (static_cast<size_t>(V) + 1023) / 1024 * 1024));
  // K slices of the dx GEMM: the count whose waves of tiles waste least (74
  // CTA pairs, or 148 CTAs up to 128 rows), each slice adding a little for its
  // partial sums
  const int tiles = (M > 128 ? (M + 255) / 256 : 1) * ((H + 255) / 256);
  const int slots = std::max(1, M > 128 ? gemm_num_sms() / 2 : gemm_num_sms());
  const int nk = (std::min(p.vc, V) + 63) / 64;
  double best = 1e30;
  p.ksplit = 1;
  for (int k = 1; k <= 32 && 4 * k <= std::max(4, nk); ++k) {
    const double cost = static_cast<double>((tiles * static_cast<int64_t>(k) + slots - 1) / slots) / k * (1 + 0.004 * k);
    if (cost < best) {
      best = cost;
      p.ksplit = k;
    }
  }
  const int per = (nk + p.ksplit - 1) / p.ksplit;
  p.slabs = (nk + per - 1) / per;
  return p;
}

// The rows without a gradient (prompts, padding, clipped tokens) are left out
// of both products where these cost more than the two kernels and the copy that
// it takes, about 10 us: from 2^33 products on (26 us at the tensor cores' full
// rate), and with more rows than one CTA pair's tile.
bool gathers(int M, int H, int V) {
  return M > 256 && static_cast<double>(M) * H * V >= static_cast<double>(1LL << 33);
}

// Tile width of the products with the vocabulary: 256 columns, but up to 128
// rows (one CTA a tile) 128 while these take one round: 77 rows of 872 x 3032
// then take 12.0 to 12.8 us, else 15.6 (near the full round they are even: 16
// rows of 2048 x 18000 take 25.3 to 26.6 and 24.4).  With more rounds the wider
// tiles read E faster: 16 rows of 2048 x 22000 take 26 us and 36 in tiles of 128,
// of 2048 x 151936 110 in five rounds and 145 in nine.
int tile_width(int M, int N) { return M <= 128 && (N + 127) / 128 <= gemm_num_sms() ? 128 : 256; }

// rows for the TMA and for 16-byte loads
bool rows_ok(const __half* p, int ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0; }

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

struct PdlScope {  // the chain's kernels await one another (pdl_wait); the first is launched normally
  bool was = pdl_enabled();
  ~PdlScope() { set_pdl(was); }
};

}  // namespace

size_t lm_logprobs_workspace(int M, int H, int V, bool backward) {
  if (!backward) return up256(sizeof(float) * M) + up256(sizeof(float2) * static_cast<size_t>(M) * ((V + 127) / 128));
  const BwdPlan p = bwd_plan(M, H, V);
  const size_t gather = gathers(M, H, V) ? 4 * up256(sizeof(int) * M) + 256 +
                                              up256(sizeof(__half) * static_cast<size_t>(M) * ((H + 7) / 8 * 8))
                                        : 0;
  return gather + up256(sizeof(__half) * static_cast<size_t>(M) * p.vc) +
         up256(sizeof(float) * static_cast<size_t>(p.slabs) * p.slab_rows * p.ld_acc);
}

cudaError_t lm_logprobs(const __half* x, const __half* E, const int* targets, float* logp, float* lse, int M, int H,
                        int V, int ldx, int lde, void* ws, int* err, cudaStream_t st) {
  char* w = static_cast<char*>(ws);
  return lm_logprobs(x, E, targets, logp, lse, M, H, V, ldx, lde,
                     reinterpret_cast<float2*>(w + up256(sizeof(float) * M)), reinterpret_cast<float*>(w), err, st);
}

cudaError_t lm_logprobs(const __half* x, const __half* E, const int* targets, float* logp, float* lse, int M, int H,
                        int V, int ldx, int lde, float2* part, float* tgt_logit, int* err, cudaStream_t st) {
  int slots = (V + 127) / 128;
  EpiArgs ea;
  ea.targets = targets;
  ea.tgt_logit = tgt_logit;
  ea.part2 = part;
  PdlScope scope;
  set_pdl(false);
  cudaError_t e;
  if (!rows_ok(x, ldx) || !rows_ok(E, lde)) return cudaErrorInvalidValue;
  if (M == 1 && sizeof(float) * (static_cast<size_t>(H) + 255) <= kOneSmem) {
    slots = std::min(slots, kOneBlocks * gemm_num_sms());
    e = one_row(x, E, targets, H, V, lde, part, tgt_logit, slots, st);
  } else {
    e = gemm(Operand{x, M, H, ldx}, Operand{E, V, H, lde}, M, V, Epi::kLogProb, ea, err, st,
             tile_width(M, V));
  }
  if (e != cudaSuccess) return e;
  set_pdl(true);
  auto finish = [&](auto kern, int rb) {
    int warps = rb;
    while (warps < kWarps && warps * (32 / rb) < slots) warps *= 2;
    return launch_pdl(kern, (M + rb - 1) / rb, 32 * warps, 0, st, ea.part2, ea.tgt_logit, targets, x, E, M, H, V, ldx,
                      lde, slots, logp, lse);
  };
  return M <= 8 * gemm_num_sms() ? finish(logprob_finish_kernel<4>, 4) : finish(logprob_finish_kernel<32>, 32);
}

cudaError_t lm_logprobs_backward(const __half* x, const __half* E, const int* targets, const float* lse,
                                 const float* dlogp, __half* dx, int M, int H, int V, int ldx, int lde, int lddx,
                                 float scale, void* ws, int* err, cudaStream_t st) {
  if (!rows_ok(x, ldx) || !rows_ok(E, lde)) return cudaErrorInvalidValue;
  const BwdPlan p = bwd_plan(M, H, V);
  char* w = static_cast<char*>(ws);
  __half* pc = reinterpret_cast<__half*>(w);
  float* acc = reinterpret_cast<float*>(w + up256(sizeof(__half) * static_cast<size_t>(M) * p.vc));
  PdlScope scope;
  set_pdl(false);
  const int* in_targets = targets;
  const float* in_lse = lse;
  const __half* in_x = x;
  const int* m_rows = nullptr;
  const int* place = nullptr;
  int in_ldx = ldx;
  if (gathers(M, H, V)) {
    char* g = reinterpret_cast<char*>(acc) + up256(sizeof(float) * static_cast<size_t>(p.slabs) * p.slab_rows * p.ld_acc);
    const size_t ints = up256(sizeof(int) * M);
    int* list = reinterpret_cast<int*>(g);
    int* at = reinterpret_cast<int*>(g + ints);
    int* tc = reinterpret_cast<int*>(g + 2 * ints);
    float* lsec = reinterpret_cast<float*>(g + 3 * ints);
    int* count = reinterpret_cast<int*>(g + 4 * ints);
    __half* xc = reinterpret_cast<__half*>(g + 4 * ints + 256);
    in_ldx = (H + 7) / 8 * 8;
    cudaError_t e = launch_pdl(live_rows_kernel, 1, 1024, 0, st, targets, dlogp, M, V, list, at, count);
    if (e != cudaSuccess) return e;
    set_pdl(true);
    e = launch_pdl(gather_rows_kernel, (M + 7) / 8, 256, 0, st, x, ldx, lse, targets, list, count, H, xc, in_ldx, lsec,
                   tc);
    if (e != cudaSuccess) return e;
    in_targets = tc;
    in_lse = lsec;
    in_x = xc;
    m_rows = count;
    place = at;
  }
  for (int v0 = 0; v0 < V; v0 += p.vc) {
    const int n = std::min(p.vc, V - v0);
    const __half* Ec = E + static_cast<size_t>(v0) * lde;
    EpiArgs ea;
    ea.targets = in_targets;
    ea.lse = in_lse;
    ea.m_rows = m_rows;
    ea.vocab_off = v0;
    ea.out = pc;
    ea.ld_out = p.vc;
    cudaError_t e = gemm(Operand{in_x, M, H, in_ldx}, Operand{Ec, n, H, lde}, M, n, Epi::kProbs, ea, err, st,
                         tile_width(M, n));
    if (e != cudaSuccess) return e;
    set_pdl(true);
    EpiArgs eb;
    eb.out = acc;
    eb.ld_out = p.ld_acc;
    eb.accumulate = v0 > 0;
    eb.ksplit = p.slabs;
    eb.slab_rows = p.slab_rows;
    eb.m_rows = m_rows;
    // acc (+)= probabilities . E_c (E_c [n, H] read MN-major); one writer per element and chunk
    e = gemm(Operand{pc, M, n, p.vc}, Operand{Ec, H, n, lde, true}, M, H, Epi::kStoreF32, eb, err, st, 256);
    if (e != cudaSuccess) return e;
  }
  // columns a warp: 128, more while there are over 16 warps an SM
  int cols = 128;
  while (cols < H && static_cast<int64_t>(M) * ((H + cols - 1) / cols) > 16 * gemm_num_sms()) cols *= 2;
  const int parts = (H + cols - 1) / cols;
  const int64_t items = static_cast<int64_t>(M) * parts;
  return launch_pdl(logprob_dx_kernel, static_cast<unsigned>((items + 7) / 8), 256, 0, st, acc, p.slabs, p.slab_rows,
                    p.ld_acc, place, x, ldx, E, lde, lse, dlogp, targets, M, H, V, scale, dx, lddx, cols, parts);
}

cudaError_t ce_stream_logp(const float* part_ref, const float* part_sum, const float* tgt_logit, const int* targets,
                           const __half* xf, const __half* E, int M, int H, int V, int slots, float* logp,
                           cudaStream_t st) {
  return launch_pdl(stream_logp_kernel, (M + kStreamWarps - 1) / kStreamWarps, 32 * kStreamWarps, 0, st, part_ref,
                    part_sum, tgt_logit, targets, xf, E, M, H, V, slots, logp);
}

}  // namespace llmcu
