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

constexpr int kRows = 32;   // rows per CTA of the forward's finishing kernel: one per lane
constexpr int kWarps = 32;  // its warps share the slots

// Joins the slots' (max, sum) pairs of 32 rows: warp w takes slots w, w + 32,
// ...; lanes are rows, so every load is 256 contiguous bytes.  Before that,
// while the GEMM still runs, warp w forms row w's target logit (x, E and the
// targets are complete before the GEMM starts); it also replaces the GEMM's
// value in the sum.
__global__ void __launch_bounds__(kRows* kWarps)
    logprob_finish_kernel(const float2* __restrict__ part, const float* __restrict__ tgt_logit,
                          const int* __restrict__ targets, const __half* __restrict__ x, const __half* __restrict__ E,
                          int M, int H, int V, int ldx, int lde, int slots, float* __restrict__ logp,
                          float* __restrict__ lse) {
  pdl_trigger();
  __shared__ float2 red[kWarps][kRows];
  __shared__ float exact[kRows];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  {
    const int row = blockIdx.x * kRows + w;
    const int t = row < M ? targets[row] : -1;
    if (t >= 0 && t < V) {
      const float l = target_logit(x + static_cast<size_t>(row) * ldx, E + static_cast<size_t>(t) * lde, H, lane);
      if (lane == 0) exact[w] = l;
    }
  }
  pdl_wait();
  const int m = blockIdx.x * kRows + lane;
  float mx = -INFINITY, s = 0.f;
  auto join = [&](float2 o) {
    const float n = fmaxf(mx, o.x);
    if (n > -INFINITY) {
      s = s * exp2f((mx - n) * kLog2e) + o.y * exp2f((o.x - n) * kLog2e);
    } else {
      s += o.y;  // 0, or a NaN
    }
    mx = n;
  };
  if (m < M) {
#pragma unroll 8
    for (int i = w; i < slots; i += kWarps) join(__ldg(part + static_cast<size_t>(i) * M + m));
  }
  red[w][lane] = make_float2(mx, s);
  __syncthreads();
  if (w == 0 && m < M) {
    mx = -INFINITY;
    s = 0.f;
    for (int i = 0; i < kWarps; ++i) join(red[i][lane]);
    const int t = targets[m];
    const bool ok = t >= 0 && t < V;
    if (ok) {
      const float rough = tgt_logit[m], d = exact[lane] - rough;
      if (isfinite(d)) s = fmaf(exp2f((rough - mx) * kLog2e), expm1f(d), s);
    }
    const float l = mx + logf(s);
    lse[m] = l;
    logp[m] = ok ? exact[lane] - l : 0.f;
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
    const float rough = tgt_logit[m], d = exact - rough;
    if (isfinite(d)) s = fmaf(exp2f((rough - mx) * kLog2e), expm1f(d), s);
    logp[m] = exact - (mx + logf(s));
  }
}

// dx row m from the K slices' partial sums (slab k: rows [k * slab_rows, ...)
// of acc), in slice order, and the target's own term in fp32.
__global__ void __launch_bounds__(256)
    logprob_dx_kernel(const float* __restrict__ acc, int slabs, int slab_rows, int ld_acc,
                      const __half* __restrict__ x, int ldx, const __half* __restrict__ E, int lde,
                      const float* __restrict__ lse, const float* __restrict__ dlogp, const int* __restrict__ targets,
                      int H, int V, float scale, __half* __restrict__ dx, int lddx) {
  pdl_trigger();
  __shared__ float s_exact;
  const int m = blockIdx.x;
  const int t = targets[m];
  const bool ok = t >= 0 && t < V;
  if (ok && threadIdx.x < 32) {  // inputs alone: while the last GEMM still runs
    const float l = target_logit(x + static_cast<size_t>(m) * ldx, E + static_cast<size_t>(t) * lde, H, threadIdx.x);
    if (threadIdx.x == 0) s_exact = l;
  }
  __syncthreads();
  pdl_wait();
  // 1 - p_t without cancellation for a confident token
  const float g = ok ? scale * dlogp[m] : 0.f;
  const float one_minus = ok ? -expm1f(s_exact - lse[m]) : 0.f;
  const float unshift = exp2f(-kProbShift);
  const __half* et = E + static_cast<size_t>(ok ? t : 0) * lde;
  const float* a0 = acc + static_cast<size_t>(m) * ld_acc;
  __half* out = dx + static_cast<size_t>(m) * lddx;
  const bool vec = (reinterpret_cast<uintptr_t>(dx) & 7) == 0 && (lddx & 3) == 0;
  for (int c = threadIdx.x * 4; c < H; c += blockDim.x * 4) {
    float r[4] = {0.f, 0.f, 0.f, 0.f};
    if (ok) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int k = 0; k < slabs; ++k) {  // ld_acc is a multiple of 4; what lies past H is not used
        const float4 o = *reinterpret_cast<const float4*>(a0 + static_cast<size_t>(k) * slab_rows * ld_acc + c);
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

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

struct PdlScope {  // the chain's kernels await one another (pdl_wait); the first is launched normally
  bool was = pdl_enabled();
  ~PdlScope() { set_pdl(was); }
};

}  // namespace

size_t lm_logprobs_workspace(int M, int H, int V, bool backward) {
  if (!backward) return up256(sizeof(float) * M) + up256(sizeof(float2) * static_cast<size_t>(M) * ((V + 127) / 128));
  const BwdPlan p = bwd_plan(M, H, V);
  return up256(sizeof(__half) * static_cast<size_t>(M) * p.vc) +
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
  const int slots = (V + 127) / 128;
  EpiArgs ea;
  ea.targets = targets;
  ea.tgt_logit = tgt_logit;
  ea.part2 = part;
  PdlScope scope;
  set_pdl(false);
  cudaError_t e = gemm(Operand{x, M, H, ldx}, Operand{E, V, H, lde}, M, V, Epi::kLogProb, ea, err, st, 256);
  if (e != cudaSuccess) return e;
  set_pdl(true);
  return launch_pdl(logprob_finish_kernel, (M + kRows - 1) / kRows, kRows * kWarps, 0, st, ea.part2, ea.tgt_logit,
                    targets, x, E, M, H, V, ldx, lde, slots, logp, lse);
}

cudaError_t lm_logprobs_backward(const __half* x, const __half* E, const int* targets, const float* lse,
                                 const float* dlogp, __half* dx, int M, int H, int V, int ldx, int lde, int lddx,
                                 float scale, void* ws, int* err, cudaStream_t st) {
  const BwdPlan p = bwd_plan(M, H, V);
  char* w = static_cast<char*>(ws);
  __half* pc = reinterpret_cast<__half*>(w);
  float* acc = reinterpret_cast<float*>(w + up256(sizeof(__half) * static_cast<size_t>(M) * p.vc));
  PdlScope scope;
  set_pdl(false);
  for (int v0 = 0; v0 < V; v0 += p.vc) {
    const int n = std::min(p.vc, V - v0);
    const __half* Ec = E + static_cast<size_t>(v0) * lde;
    EpiArgs ea;
    ea.targets = targets;
    ea.lse = lse;
    ea.vocab_off = v0;
    ea.out = pc;
    ea.ld_out = p.vc;
    cudaError_t e = gemm(Operand{x, M, H, ldx}, Operand{Ec, n, H, lde}, M, n, Epi::kProbs, ea, err, st, 256);
    if (e != cudaSuccess) return e;
    set_pdl(true);
    EpiArgs eb;
    eb.out = acc;
    eb.ld_out = p.ld_acc;
    eb.accumulate = v0 > 0;
    eb.ksplit = p.slabs;
    eb.slab_rows = p.slab_rows;
    // acc (+)= probabilities . E_c (E_c [n, H] read MN-major); one writer per element and chunk
    e = gemm(Operand{pc, M, n, p.vc}, Operand{Ec, H, n, lde, true}, M, H, Epi::kStoreF32, eb, err, st, 256);
    if (e != cudaSuccess) return e;
  }
  return launch_pdl(logprob_dx_kernel, M, 256, 0, st, acc, p.slabs, p.slab_rows, p.ld_acc, x, ldx, E, lde, lse,
                    dlogp, targets, H, V, scale, dx, lddx);
}

cudaError_t ce_stream_logp(const float* part_ref, const float* part_sum, const float* tgt_logit, const int* targets,
                           const __half* xf, const __half* E, int M, int H, int V, int slots, float* logp,
                           cudaStream_t st) {
  return launch_pdl(stream_logp_kernel, (M + kStreamWarps - 1) / kStreamWarps, 32 * kStreamWarps, 0, st, part_ref,
                    part_sum, tgt_logit, targets, xf, E, M, H, V, slots, logp);
}

}  // namespace llmcu
