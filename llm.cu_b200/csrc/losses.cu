// losses.cu -- losses over token log-probabilities, with their gradients: the
// paired preference loss and the clipped policy loss with a KL term.
//
// Both read each log-probability once and write one gradient: 9-21 bytes a
// token against a few dozen instructions, so what bounds them is memory for
// long batches and launch latency for short ones.
//
// Tokens are taken four at a time by their place in memory: a "quad" is four
// elements whose first index in the [rows, ld] buffers is a multiple of 4,
// whatever row they start in, so that every buffer with a 16-byte aligned base
// (4 for the mask) is read by vectors at any ld.  Quads that reach over an end
// of their row, or buffers that are not aligned, are taken element by element.
#include <algorithm>
#include <cmath>

#include "common.cuh"

namespace llmcu {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over the CTA, in a fixed order, for every thread; `red` holds 32 values.
__device__ __forceinline__ double block_sum(double v, double* red) {
  v = warp_sum_f64(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  const int n = blockDim.x >> 5;
  return warp_sum_f64((threadIdx.x & 31) < n ? red[threadIdx.x & 31] : 0.0);
}

// One row of a [rows, ld] buffer in quads.
struct RowSpan {
  int64_t first, end;  // element indices of the row's tokens
  int64_t q0;          // first quad
  int nq;              // quads that touch the row
  __device__ RowSpan(int64_t row, int64_t ld, int seq) {
    first = row * ld;
    end = first + seq;
    q0 = first >> 2;
    nq = static_cast<int>(((end + 3) >> 2) - q0);
  }
};

// Four elements from index i on; the ones outside [first, end) keep `fill`.
__device__ __forceinline__ void load4(const float* __restrict__ p, int64_t i, int64_t first, int64_t end, bool vec,
                                      float fill, float (&v)[4]) {
  if (vec && i >= first && i + 4 <= end) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p + i));
    v[0] = a.x;
    v[1] = a.y;
    v[2] = a.z;
    v[3] = a.w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = i + j >= first && i + j < end ? __ldg(p + i + j) : fill;
  }
}
// Bit j: token i + j is scored (inside the row, and unmasked; no mask: all are).
__device__ __forceinline__ uint32_t load_mask(const uint8_t* __restrict__ p, int64_t i, int64_t first, int64_t end,
                                              bool vec) {
  uint32_t b = 0;
  if (vec && i >= first && i + 4 <= end) {
    if (!p) return 15u;
    const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(p + i));
#pragma unroll
    for (int j = 0; j < 4; ++j) b |= ((w >> (8 * j)) & 0xffu) ? 1u << j : 0u;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j >= first && i + j < end && (!p || __ldg(p + i + j))) b |= 1u << j;
  }
  return b;
}
__device__ __forceinline__ void store4(float* __restrict__ p, int64_t i, int64_t first, int64_t end, bool vec,
                                       const float (&v)[4]) {
  if (vec && i >= first && i + 4 <= end) {
    *reinterpret_cast<float4*>(p + i) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j >= first && i + j < end) p[i + j] = v[j];
  }
}

// --------------------------------------------------- preference loss
// Rows b = i (chosen) and P + i (rejected) of pair i:
//   R_b = sum over scored tokens of (logp - ref), or their mean
//   D = R_chosen - R_rejected,  h = beta D - margin
//   sigmoid  -(1 - e) log s(h) - e log s(-h)      dL/dD = beta (e - s(-h))
//   hinge    max(0, 1 - h)                        dL/dD = -beta where h < 1
//   squared  (D - 1 / (2 beta))^2                 dL/dD = 2 (D - 1 / (2 beta))
// and dlogp = +-dL/dD (times 1 / count for means) on the scored tokens, times
// the pair's upstream gradient.
//
// A cluster of CTAs takes a pair, each a share of the quads of both rows; the
// sums meet over distributed shared memory, in rank order.  The mask's bits
// of the first 8 x 2 quads of a thread stay in a register, so the second pass
// reads nothing for them and only writes.
//
// logp - ref is formed in fp32 (exact where the two are within a factor of
// two) and summed in 64 bits: R_chosen and R_rejected are sums of thousands
// of terms whose difference is of the order of one.
constexpr int kKept = 8;  // quads of each row whose mask bits a thread keeps

__global__ void __launch_bounds__(kThreads)
    preference_kernel(PreferenceArgs a) {
  __shared__ double red[32];
  __shared__ double part[4];
  const int C = a.cluster;
  const uint32_t rank = C > 1 ? cluster_ctarank() : 0u;
  const int pair = blockIdx.x / C;
  const int stride = C * kThreads;
  const int t0 = static_cast<int>(rank) * kThreads + threadIdx.x;
  double sum[2] = {0.0, 0.0};
  int cnt[2] = {0, 0};
  uint64_t kept = 0;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const RowSpan r(static_cast<int64_t>(side) * a.pairs + pair, a.ld, a.seq);
    int k = 0;
    for (int q = t0; q < r.nq; q += stride, ++k) {
      const int64_t i = (r.q0 + q) << 2;
      const uint32_t bits = load_mask(a.mask, i, r.first, r.end, a.vec);
      if (k < kKept) kept |= static_cast<uint64_t>(bits) << (4 * (k + kKept * side));
      if (!bits) continue;
      float lp[4], rf[4];
      load4(a.logp, i, r.first, r.end, a.vec, 0.f, lp);
      if (a.ref) {
        load4(a.ref, i, r.first, r.end, a.vec, 0.f, rf);
#pragma unroll
        for (int j = 0; j < 4; ++j) lp[j] -= rf[j];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if ((bits >> j) & 1) sum[side] += static_cast<double>(lp[j]);
      cnt[side] += __popc(bits);
    }
  }
  double v[4] = {sum[0], sum[1], static_cast<double>(cnt[0]), static_cast<double>(cnt[1])};
  const int nv = a.mean_tokens ? 4 : 2;
  for (int k = 0; k < nv; ++k) v[k] = block_sum(v[k], red);
  if (C > 1) {
    if (threadIdx.x == 0)
      for (int k = 0; k < nv; ++k) part[k] = v[k];
    cluster_sync_all();
    const uint32_t mine = smem_u32(part);
    for (int k = 0; k < nv; ++k) {
      v[k] = 0.0;
      for (int c = 0; c < C; ++c) v[k] += ld_cluster_f64(mapa_shared(mine + 8 * k, c));
    }
    cluster_sync_all();  // nobody leaves while its sums are read
  }
  const double share[2] = {a.mean_tokens ? 1.0 / fmax(v[2], 1.0) : 1.0, a.mean_tokens ? 1.0 / fmax(v[3], 1.0) : 1.0};
  const double R[2] = {v[0] * share[0], v[1] * share[1]};
  const double beta = a.beta, D = R[0] - R[1];
  float loss, dD;
  if (a.kind == kPrefSquared) {
    const double off = D - 0.5 / beta;
    loss = static_cast<float>(off * off);
    dD = static_cast<float>(2.0 * off);
  } else {
    const double hd = beta * D - static_cast<double>(a.margin);
    const float h = static_cast<float>(hd);
    if (a.kind == kPrefSigmoid) {
      const float e = a.smoothing, z = expf(-fabsf(h));
      const float l1 = log1pf(z);  // log(1 + e^x) = max(x, 0) + log1p(e^-|x|)
      loss = (1.f - e) * (fmaxf(-h, 0.f) + l1) + e * (fmaxf(h, 0.f) + l1);
      const float s_neg = h >= 0.f ? z / (1.f + z) : 1.f / (1.f + z);  // s(-h)
      dD = a.beta * (e - s_neg);
    } else {
      loss = hd < 1.0 ? static_cast<float>(1.0 - hd) : (hd >= 1.0 ? 0.f : h);  // NaN stays
      dD = hd < 1.0 ? -a.beta : (hd >= 1.0 ? 0.f : h);
    }
  }
  if (rank == 0 && threadIdx.x == 0) {
    if (a.loss) a.loss[pair] = loss;
    if (a.reward) {
      a.reward[pair] = static_cast<float>(beta * R[0]);
      a.reward[a.pairs + pair] = static_cast<float>(beta * R[1]);
    }
  }
  if (!a.dlogp) return;
  const float up = a.dloss ? __ldg(a.dloss + pair) : 1.0f / static_cast<float>(a.pairs);
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const RowSpan r(static_cast<int64_t>(side) * a.pairs + pair, a.ld, a.seq);
    const float g = (side ? -dD : dD) * up * static_cast<float>(share[side]);
    int k = 0;
    for (int q = t0; q < r.nq; q += stride, ++k) {
      const int64_t i = (r.q0 + q) << 2;
      const uint32_t bits = k < kKept ? static_cast<uint32_t>(kept >> (4 * (k + kKept * side))) & 15u
                                      : load_mask(a.mask, i, r.first, r.end, a.vec);
      float o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = (bits >> j) & 1 ? g : 0.f;
      store4(a.dlogp, i, r.first, r.end, a.vec, o);
    }
  }
}

// ------------------------------------------------------- policy loss
// Per scored token, with delta = logp - old, r = e^delta, advantage A and
// d = ref - logp:
//   obj = min(r A, clamp(r, 1 - low, 1 + high) A); with a dual clip c and A < 0: max(obj, c A)
//   l = -obj + beta (e^d - d - 1)
//   dl/dlogp = -r A where nothing clips, else 0;  - beta (e^d - 1)
// The loss is the sum of l times its row's weight: 1 / (scored tokens), 1 /
// (rows * the row's scored tokens), or 1 / norm.
//
// Whether a token clips is decided on delta in 64 bits against the logarithm
// of the border, so that a token next to it falls on the side that the inputs
// say.  e^d - d - 1 loses everything to cancellation for a small d; below 1/2
// its series d^2/2 (1 + d/3 (1 + d/4 (...))) is summed instead (ten terms: the
// next is under 2^-24 of the sum).
__device__ __forceinline__ float kl_of(float d, float em1) {
  if (fabsf(d) < 0.5f) {
    float s = 1.f;
#pragma unroll
    for (int k = 10; k >= 3; --k) s = fmaf(s, d * (1.0f / static_cast<float>(k)), 1.f);
    return 0.5f * d * d * s;
  }
  return em1 - d;
}

// Scored tokens: of each row (one CTA or warp a row) into counts[row], or of
// everything, a partial sum a CTA, into counts[0 .. gridDim.x).
__global__ void __launch_bounds__(kThreads) policy_count_kernel(PolicyArgs a, int* __restrict__ counts) {
  pdl_trigger();
  __shared__ int red[kThreads / 32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  if (a.agg == kPolicySequenceMean && a.seq <= 1024) {  // a warp a row
    const int row = blockIdx.x * (kThreads / 32) + w;
    if (row >= a.batch) return;
    const RowSpan r(row, a.ld, a.seq);
    int n = 0;
    for (int q = lane; q < r.nq; q += 32) n += __popc(load_mask(a.mask, (r.q0 + q) << 2, r.first, r.end, a.vec));
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) counts[row] = n;
    return;
  }
  int n = 0;
  if (a.agg == kPolicySequenceMean) {  // a CTA a row
    const RowSpan r(blockIdx.x, a.ld, a.seq);
    for (int q = threadIdx.x; q < r.nq; q += kThreads)
      n += __popc(load_mask(a.mask, (r.q0 + q) << 2, r.first, r.end, a.vec));
  } else {
    for (int64_t u = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; u < a.units;
         u += static_cast<int64_t>(gridDim.x) * kThreads) {
      const int row = static_cast<int>(__umulhi(static_cast<uint32_t>(u), a.div_m) >> a.div_s);
      const RowSpan r(row, a.ld, a.seq);
      const int q = static_cast<int>(u) - row * a.row_quads;
      if (q < r.nq) n += __popc(load_mask(a.mask, (r.q0 + q) << 2, r.first, r.end, a.vec));
    }
  }
  n = __reduce_add_sync(0xffffffffu, n);
  if (lane == 0) red[w] = n;
  __syncthreads();
  if (w == 0) {
    n = __reduce_add_sync(0xffffffffu, lane < kThreads / 32 ? red[lane] : 0);
    if (lane == 0) counts[blockIdx.x] = n;
  }
}

__global__ void __launch_bounds__(kThreads)
    policy_main_kernel(PolicyArgs a, const int* __restrict__ counts, int n_counts, double* __restrict__ partial) {
  pdl_trigger();
  pdl_wait();
  __shared__ double red[32];
  float weight = a.inv_norm;
  if (a.agg == kPolicyTokenMean) {
    double n = 0.0;
    for (int i = threadIdx.x; i < n_counts; i += kThreads) n += static_cast<double>(counts[i]);
    n = block_sum(n, red);
    weight = static_cast<float>(1.0 / fmax(n, 1.0));
  }
  double s_loss = 0.0, s_kl = 0.0;
  int64_t clips = 0, tokens = 0;
  for (int64_t u = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; u < a.units;
       u += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int row = static_cast<int>(__umulhi(static_cast<uint32_t>(u), a.div_m) >> a.div_s);
    const RowSpan r(row, a.ld, a.seq);
    const int q = static_cast<int>(u) - row * a.row_quads;
    if (q >= r.nq) continue;
    const int64_t i = (r.q0 + q) << 2;
    const uint32_t bits = load_mask(a.mask, i, r.first, r.end, a.vec);
    float g[4] = {0.f, 0.f, 0.f, 0.f};
    if (bits) {
      if (a.agg == kPolicySequenceMean) weight = 1.0f / (static_cast<float>(counts[row]) * static_cast<float>(a.batch));
      float lp[4], old[4], adv[4], ref[4];
      load4(a.logp, i, r.first, r.end, a.vec, 0.f, lp);
      load4(a.old, i, r.first, r.end, a.vec, 0.f, old);
      if (a.token_adv) {
        load4(a.adv, i, r.first, r.end, a.vec, 0.f, adv);
      } else {
        adv[0] = adv[1] = adv[2] = adv[3] = __ldg(a.adv + row);
      }
      if (a.ref) load4(a.ref, i, r.first, r.end, a.vec, 0.f, ref);
      float l = 0.f, kl = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!((bits >> j) & 1)) continue;
        const double delta = static_cast<double>(lp[j]) - static_cast<double>(old[j]);
        const float A = adv[j];
        const float rA = expf(static_cast<float>(delta)) * A;
        float obj = rA;
        bool clip = false;
        if (A > 0.f && delta > a.log_high) {
          obj = a.high * A;
          clip = true;
        } else if (A < 0.f && delta < a.log_low) {
          obj = a.low * A;
          clip = true;
        } else if (A < 0.f && delta > a.log_dual) {
          obj = a.dual * A;
          clip = true;
        }
        float gr = clip ? 0.f : -rA;
        float lj = -obj;
        if (a.ref) {
          const float d = ref[j] - lp[j];
          const float em1 = expm1f(d);
          const float k3 = kl_of(d, em1);
          gr = fmaf(-a.beta, em1, gr);
          lj = fmaf(a.beta, k3, lj);
          kl += k3;
        }
        l += lj;
        clips += clip;
        g[j] = gr * weight;
      }
      s_loss += static_cast<double>(l) * static_cast<double>(weight);
      s_kl += static_cast<double>(kl);
      tokens += __popc(bits);
    }
    if (a.dlogp) store4(a.dlogp, i, r.first, r.end, a.vec, g);
  }
  const double v[4] = {block_sum(s_loss, red), block_sum(s_kl, red), block_sum(static_cast<double>(clips), red),
                       block_sum(static_cast<double>(tokens), red)};
  if (threadIdx.x == 0) {
#pragma unroll
    for (int k = 0; k < 4; ++k) partial[blockIdx.x * 4 + k] = v[k];
  }
}

// The CTAs' partial sums, in order: loss, mean KL, share of clipped tokens, scored tokens.
__global__ void __launch_bounds__(kThreads) policy_stats_kernel(const double* __restrict__ partial, int n,
                                                               float* __restrict__ stats) {
  pdl_trigger();
  pdl_wait();
  __shared__ double red[32];
  double v[4] = {0.0, 0.0, 0.0, 0.0};
  for (int i = threadIdx.x; i < n; i += kThreads)
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] += partial[i * 4 + k];
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = block_sum(v[k], red);
  if (threadIdx.x == 0) {
    const double t = fmax(v[3], 1.0);
    stats[0] = static_cast<float>(v[0]);
    stats[1] = static_cast<float>(v[1] / t);
    stats[2] = static_cast<float>(v[2] / t);
    stats[3] = static_cast<float>(v[3]);
  }
}

bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

constexpr int kCountBlocks = 296;  // CTAs of the token count: two an SM

int policy_blocks(int64_t units) {
  const int64_t want = (units + kThreads - 1) / kThreads;
  return static_cast<int>(std::min<int64_t>(want, 8 * static_cast<int64_t>(gemm_num_sms())));
}

}  // namespace

cudaError_t preference_loss(PreferenceArgs a, cudaStream_t st) {
  a.vec = aligned(a.logp, 16) && aligned(a.ref, 16) && aligned(a.mask, 4) && aligned(a.dlogp, 16);
  // CTAs a pair: enough that a thread meets at most about two quads of each
  // row, but no more than keep the GPU's resident CTAs (8 an SM) busy
  int C = 1;
  const int quads = a.seq / 4 + 2;
  while (C < 8 && quads > 2 * C * kThreads && static_cast<int64_t>(a.pairs) * C < 8LL * gemm_num_sms()) C *= 2;
  a.cluster = C;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.pairs) * C);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = C > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, preference_kernel, a);
}

size_t policy_loss_workspace(int batch) {
  const size_t partial = sizeof(double) * 4 * 8 * static_cast<size_t>(gemm_num_sms());
  return partial + sizeof(int) * std::max<size_t>(kCountBlocks, static_cast<size_t>(batch));
}

cudaError_t policy_loss(PolicyArgs a, void* ws, cudaStream_t st) {
  a.vec = aligned(a.logp, 16) && aligned(a.old, 16) && aligned(a.ref, 16) && aligned(a.mask, 4) &&
          aligned(a.dlogp, 16) && (!a.token_adv || aligned(a.adv, 16));
  // unit u: quad u % row_quads of row u / row_quads (a row of seq tokens
  // touches at most row_quads quads), the division by a multiplication:
  // floor(u / d) = (u * m) >> (32 + s) for u < 2^31, m = ceil(2^(32 + s) / d), 2^s < d <= 2^(s + 1)
  a.row_quads = std::max(2, (a.seq + 6) / 4);
  a.units = static_cast<int64_t>(a.batch) * a.row_quads;
  if (a.units >= (1LL << 31)) return cudaErrorInvalidValue;
  const uint32_t d = static_cast<uint32_t>(a.row_quads);
  int s = 0;
  while ((2ull << s) < d) ++s;
  a.div_s = s;
  a.div_m = static_cast<uint32_t>(((1ull << (32 + s)) + d - 1) / d);
  double* partial = static_cast<double*>(ws);
  int* counts = reinterpret_cast<int*>(partial + 4 * 8 * static_cast<size_t>(gemm_num_sms()));
  const bool was = pdl_enabled();
  set_pdl(false);
  cudaError_t e = cudaSuccess;
  int n_counts = 0;
  if (a.agg == kPolicySequenceMean) {
    n_counts = a.seq <= 1024 ? (a.batch + kThreads / 32 - 1) / (kThreads / 32) : a.batch;
  } else if (a.agg == kPolicyTokenMean) {
    n_counts = static_cast<int>(std::min<int64_t>(kCountBlocks, (a.units + kThreads - 1) / kThreads));
  }
  if (n_counts) {
    e = launch_pdl(policy_count_kernel, n_counts, kThreads, 0, st, a, counts);
    set_pdl(true);
  }
  const int blocks = policy_blocks(a.units);
  if (e == cudaSuccess) e = launch_pdl(policy_main_kernel, blocks, kThreads, 0, st, a, counts, n_counts, partial);
  set_pdl(true);
  if (e == cudaSuccess) e = launch_pdl(policy_stats_kernel, 1, kThreads, 0, st, partial, blocks, a.stats);
  set_pdl(was);
  return e;
}

}  // namespace llmcu
