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
#include <initializer_list>

#include "common.cuh"

namespace llmcu {

namespace {

constexpr int kThreads = 256;
constexpr int kMainBlocks = 4;  // resident CTAs of the policy loss's main kernel on an SM

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sums of N values over the CTA, in a fixed order, for every thread; `red`
// holds N * 32 values.
template <int N>
__device__ __forceinline__ void block_sums(double (&v)[N], double* red) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = warp_sum_f64(v[k]);
  __syncthreads();
  if (lane == 0) {
#pragma unroll
    for (int k = 0; k < N; ++k) red[k * 32 + w] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) {
    v[k] = 0.0;
    for (int i = 0; i < nw; ++i) v[k] += red[k * 32 + i];
  }
}
// The CTAs' sums of a cluster, in rank order.  Each CTA stores its own into
// every other's shared memory (`slots`, 8 * N values), so that after one
// cluster barrier all reads are local and a CTA may leave at any time.  The
// kernel has arrived at the cluster barrier once before (cluster_begin), which
// this waits for: a CTA's shared memory exists once it runs.  `all` false:
// rank 0 alone gets the sums, and the others do not wait.
constexpr int kMaxCluster = 8;
__device__ __forceinline__ void cluster_begin(int C) {
  if (C > 1) cluster_arrive();
}
template <int N>
__device__ __forceinline__ void cluster_sums(double (&v)[N], double* slots, int C, int rank, bool first,
                                             bool all = true) {
  if (C == 1) return;
  if (first) cluster_wait();
  const int t = threadIdx.x;
  const int c = t / N, k = t - c * N;
  if (c < (all ? C : 1)) {
    double mine = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) mine = k == i ? v[i] : mine;
    st_cluster_f64(mapa_shared(smem_u32(slots + rank * N + k), c), mine);
  }
  cluster_arrive();
  if (!all && rank != 0) return;
  cluster_wait();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = 0.0;
    for (int r = 0; r < C; ++r) v[i] += slots[r * N + i];
  }
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
// The top bit of every byte of w that is not 0.
__device__ __forceinline__ uint32_t nonzero_bytes(uint32_t w) {
  return (((w & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w) & 0x80808080u;
}
// Bit j: byte j of an aligned four is not 0 (the bits, 8 apart, brought together
// by a product that carries none of them into another).
__device__ __forceinline__ uint32_t mask4(const uint8_t* p) {
  return ((nonzero_bytes(__ldg(reinterpret_cast<const uint32_t*>(p))) >> 7) * 0x01020408u) >> 24;
}
// Bit j: token i + j is scored (inside the row, and unmasked; no mask: all are).
__device__ __forceinline__ uint32_t load_mask(const uint8_t* __restrict__ p, int64_t i, int64_t first, int64_t end,
                                              bool vec) {
  uint32_t b = 0;
  if (vec && i >= first && i + 4 <= end) {
    if (!p) return 15u;
    b = mask4(p + i);
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
  __shared__ double red[4 * 32];
  __shared__ double slots[4 * kMaxCluster];
  const int C = a.cluster;
  const int rank = C > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  cluster_begin(C);
  const int pair = blockIdx.x / C;
  const int stride = C * kThreads;
  const int t0 = rank * kThreads + threadIdx.x;
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
  double share[2] = {1.0, 1.0};
  if (a.mean_tokens) {
    double v[4] = {sum[0], sum[1], static_cast<double>(cnt[0]), static_cast<double>(cnt[1])};
    block_sums(v, red);
    cluster_sums(v, slots, C, rank, true);
    sum[0] = v[0];
    sum[1] = v[1];
    share[0] = 1.0 / fmax(v[2], 1.0);
    share[1] = 1.0 / fmax(v[3], 1.0);
  } else {
    block_sums(sum, red);
    cluster_sums(sum, slots, C, rank, true);
  }
  const double R[2] = {sum[0] * share[0], sum[1] * share[1]};
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
      loss = (1.f - e) * (fmaxf(-h, 0.f) + l1);
      if (e > 0.f) loss += e * (fmaxf(h, 0.f) + l1);  // e = 0: h may be infinite
      if (e > 0.f) {
        // e - s(-h) would cancel near the h whose gradient is 0; from t = h less
        // that, e (1 - e) (e^t - 1) / (e + (1 - e) e^t), over e^t for t > 0
        const float t = static_cast<float>(hd - a.still), u = expm1f(-fabsf(t)), v = expf(-fabsf(t)), f = 1.f - e;
        dD = a.beta * f * (t > 0.f ? -e * u / fmaf(e, v, f) : e * u / fmaf(f, v, e));
      } else {
        dD = -a.beta * (h >= 0.f ? z / (1.f + z) : 1.f / (1.f + z));  // s(-h)
      }
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
  const float up = a.dloss ? __ldg(a.dloss + pair) : 1.0f / static_cast<float>(a.pairs);
#pragma unroll
  for (int side = 0; side < 2 && a.dlogp; ++side) {
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
// Whether a token clips is decided on delta against the logarithm of the
// border; next to it (which fp32 cannot tell) in 64 bits, so that the token
// falls on the side that the inputs say.
//
// Advantages are centred as a rule, so the sum of r A over a batch is a small
// difference of large terms: with e = r - 1 it is taken as the sum of A, in 64
// bits, and the sum of e A, whose terms are several times smaller.
//
// e^x - 1 and e^d - d - 1 lose everything to cancellation for a small argument;
// below 1 the series x^2 (1/2! + x/3! + ...) is summed, to x^12 / 12! (the next
// term is under 2^-25 of the sum).
//
// e^x leaves fp32 at 88.7, where the advantage (0 among others), beta or the
// weight may bring it back: a thread whose sums come to kHuge or more, or to NaN,
// takes its tokens again in 64 bits (far_terms), after its loop, so that the
// loop has neither tests nor registers for it (64-bit terms inside it cost 1024 x
// 8192 1.4 to 5 us of 36).
//
// Two tokens go through the series together (fma.rn.f32x2): the kernel is short
// of issue slots.
constexpr double kHuge = 1e16;
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ void unpack2(uint64_t v, float (&f)[2]) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f[0]), "=f"(f[1]) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
// rest = e^x - x - 1, em1 = e^x - 1, ex = e^x of two numbers.
__device__ __forceinline__ void exp_rest2(const float (&x)[2], float (&rest)[2], float (&em1)[2], float (&ex)[2]) {
  const uint64_t X = pack2(x[0], x[1]);
  auto both = [](float c) { return pack2(c, c); };
  uint64_t S = both(1.f / 479001600.f);
  S = fma2(S, X, both(1.f / 39916800.f));
  S = fma2(S, X, both(1.f / 3628800.f));
  S = fma2(S, X, both(1.f / 362880.f));
  S = fma2(S, X, both(1.f / 40320.f));
  S = fma2(S, X, both(1.f / 5040.f));
  S = fma2(S, X, both(1.f / 720.f));
  S = fma2(S, X, both(1.f / 120.f));
  S = fma2(S, X, both(1.f / 24.f));
  S = fma2(S, X, both(1.f / 6.f));
  S = fma2(S, X, both(0.5f));
  float s[2];
  unpack2(S, s);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    rest[j] = x[j] * x[j] * s[j];
    em1[j] = x[j] + rest[j];
    ex[j] = 1.f + em1[j];
    if (!(fabsf(x[j]) < 1.f)) {
      ex[j] = expf(x[j]);
      em1[j] = ex[j] - 1.f;
      rest[j] = ex[j] < INFINITY ? em1[j] - x[j] : ex[j];  // also where x itself is infinite
    }
  }
}

struct PolicyToken {
  float loss;  // the loss less -A
  float kl, grad;
  bool clip;
};
__device__ __forceinline__ void policy_tokens(const PolicyArgs& a, const float (&lp)[2], const float (&old)[2],
                                              const float (&adv)[2], const float (&ref)[2], PolicyToken (&t)[2]) {
  const float delta[2] = {lp[0] - old[0], lp[1] - old[1]};
  float rest[2], e[2], r[2];
  exp_rest2(delta, rest, e, r);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float A = adv[j];
    // clips above hi and below lo
    const bool pos = A > 0.f;
    const float hi = pos ? a.f_high : a.f_dual, lo = pos ? -INFINITY : a.f_low;
    bool above = delta[j] > hi, below = delta[j] < lo;
    if (fminf(fabsf(delta[j] - hi), fabsf(delta[j] - lo)) < a.near) {
      const double d64 = static_cast<double>(lp[j]) - static_cast<double>(old[j]);
      above = d64 > (pos ? a.log_high : a.log_dual);
      below = !pos && d64 < a.log_low;
    }
    t[j].clip = (above || below) && (pos || A < 0.f);
    const float bound = below ? a.low : pos ? a.high : a.dual;  // less 1, as e
    t[j].loss = t[j].clip ? -bound * A : -e[j] * A;
    t[j].grad = t[j].clip ? 0.f : -r[j] * A;
    t[j].kl = 0.f;
  }
  if (a.ref) {
    const float d[2] = {ref[0] - lp[0], ref[1] - lp[1]};
    float kl[2], em1[2], unused[2];
    exp_rest2(d, kl, em1, unused);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      t[j].kl = kl[j];
      if (a.beta > 0.f) {  // else a statistic alone: an infinite term times 0 would be NaN
        t[j].grad = fmaf(-a.beta, em1[j], t[j].grad);
        t[j].loss = fmaf(a.beta, kl[j], t[j].loss);
      }
    }
  }
}

// Unit u: four places of a row, of which the row's tokens are set in `in`
// (none: the unit lies past its row, or past the last).
struct PolicyUnit {
  int row;
  uint32_t in;
  int64_t i;
  __device__ __forceinline__ PolicyUnit(const PolicyArgs& a, int64_t u) {
    row = static_cast<int>(__umulhi(static_cast<uint32_t>(u), a.div_m) >> a.div_s);
    const int64_t first = static_cast<int64_t>(row) * a.ld;
    const int head = static_cast<int>(first) & 3;
    const int c = 4 * (static_cast<int>(u) - row * a.row_quads) - head;  // column of the first place
    i = first + c;
    const int left = a.seq - c;
    in = c < 0 ? 15u << -c : 15u;
    if (left < 4) in = left > 0 ? in & ((1u << left) - 1u) : 0u;
    in &= u < a.units ? 15u : 0u;
  }
  __device__ __forceinline__ bool whole(const PolicyArgs& a) const { return in == 15u && a.vec; }
  // which of them are scored
  __device__ __forceinline__ uint32_t mask(const PolicyArgs& a) const {
    if (!a.mask) return in;
    if (whole(a)) return mask4(a.mask + i);
    uint32_t b = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if ((in >> j) & 1) b |= __ldg(a.mask + i + j) ? 1u << j : 0u;
    return b;
  }
  __device__ __forceinline__ void store(const PolicyArgs& a, const float (&v)[4]) const {
    if (whole(a)) {
      *reinterpret_cast<float4*>(a.dlogp + i) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if ((in >> j) & 1) a.dlogp[i + j] = v[j];
    }
  }
};

// The four tokens of a quad: gradients (0 where nothing is scored), sums.
struct PolicyQuad {
  float lp[4], old[4], adv[4], ref[4];
  __device__ __forceinline__ void load(const PolicyArgs& a, const PolicyUnit& p) {
    if (!a.token_adv) adv[0] = adv[1] = adv[2] = adv[3] = __ldg(a.adv + p.row);
    if (p.whole(a)) {
      vec4(a.logp + p.i, lp);
      vec4(a.old + p.i, old);
      if (a.token_adv) vec4(a.adv + p.i, adv);
      if (a.ref) vec4(a.ref + p.i, ref);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if ((p.in >> j) & 1) {
          lp[j] = __ldg(a.logp + p.i + j);
          old[j] = __ldg(a.old + p.i + j);
          if (a.token_adv) adv[j] = __ldg(a.adv + p.i + j);
          if (a.ref) ref[j] = __ldg(a.ref + p.i + j);
        }
    }
  }
  static __device__ __forceinline__ void vec4(const float* p, float (&v)[4]) {
    const float4 x = __ldg(reinterpret_cast<const float4*>(p));
    v[0] = x.x;
    v[1] = x.y;
    v[2] = x.z;
    v[3] = x.w;
  }
  // gradients times `weight`; the quad's loss, KL terms and clipped tokens added up
  __device__ __forceinline__ void run(const PolicyArgs& a, uint32_t bits, float weight, float (&g)[4], double& loss,
                                      double& kl, int& clips) const {
    float l = 0.f, n = 0.f;
    double adv_sum = 0.0;
#pragma unroll
    for (int h = 0; h < 4; h += 2) {
      const float x[2] = {lp[h], lp[h + 1]}, o[2] = {old[h], old[h + 1]}, A[2] = {adv[h], adv[h + 1]},
                  rf[2] = {ref[h], ref[h + 1]};
      PolicyToken t[2];
      policy_tokens(a, x, o, A, rf, t);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const bool on = (bits >> (h + j)) & 1;
        g[h + j] = on ? t[j].grad * weight : 0.f;
        l += on ? t[j].loss : 0.f;
        n += on ? t[j].kl : 0.f;
        clips += on && t[j].clip;
        adv_sum += static_cast<double>(on ? A[j] : 0.f);
      }
    }
    loss += static_cast<double>(l) - adv_sum;
    kl += static_cast<double>(n);
  }
};

// A quad's loss, KL terms and gradients in 64 bits.
__device__ __forceinline__ void far_terms(const PolicyArgs& a, const PolicyUnit& p, uint32_t bits, double weight,
                                          float (&g)[4], double& loss, double& kl) {
#pragma unroll 1
  for (int j = 0; j < 4; ++j) {
    if (!((bits >> j) & 1)) continue;
    const double lp = static_cast<double>(__ldg(a.logp + p.i + j));
    const double A = static_cast<double>(__ldg(a.adv + (a.token_adv ? p.i + j : p.row)));
    const double delta = lp - static_cast<double>(__ldg(a.old + p.i + j));
    const bool above = delta > (A > 0.0 ? a.log_high : a.log_dual), below = delta < a.log_low;
    double grad = 0.0;
    if (A > 0.0 ? above : A < 0.0 && (above || below)) {
      loss -= (1.0 + static_cast<double>(A > 0.0 ? a.high : below ? a.low : a.dual)) * A;
    } else if (A != 0.0 || !(delta == delta)) {  // no advantage, no term, whatever the ratio (but NaN stays)
      grad = -exp(delta) * A;
      loss += grad;
    }
    if (a.ref) {
      const double d = static_cast<double>(__ldg(a.ref + p.i + j)) - lp, u = expm1(d);
      const double k = u < INFINITY ? u - d : u;  // u also where d itself is infinite
      kl += k;
      if (a.beta > 0.f) {
        loss += static_cast<double>(a.beta) * k;
        grad -= static_cast<double>(a.beta) * u;
      }
    }
    const float out = static_cast<float>(grad * weight);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i == j) g[i] = out;
  }
}

__device__ __forceinline__ void write_stats(const double (&v)[4], float* stats) {
  const double t = fmax(v[3], 1.0);
  stats[0] = static_cast<float>(v[0]);
  stats[1] = static_cast<float>(v[1] / t);
  stats[2] = static_cast<float>(v[2] / t);
  stats[3] = static_cast<float>(v[3]);
}

// Everything in one launch, for batches of at most kSmallUnits quads: each
// thread of one cluster holds one quad, the scored tokens are counted (of each
// row in shared memory, for means over rows), and the counts and then the sums
// meet over distributed shared memory.
constexpr int kSmallCluster = kMaxCluster;
constexpr int kSmallThreads = 1024;
constexpr int kSmallUnits = kSmallCluster * kSmallThreads;
constexpr int kSmallRows = 1024;

__global__ void __launch_bounds__(kSmallThreads) policy_small_kernel(PolicyArgs a, int C) {
  __shared__ double red[4 * 32];
  __shared__ double slots[2][4 * kMaxCluster];
  __shared__ int rows[kSmallRows];  // this CTA's scored tokens of each row
  extern __shared__ int all_rows[];  // [C][batch]: every CTA's
  const int rank = C > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  cluster_begin(C);
  const bool by_row = a.agg == kPolicySequenceMean;
  const int nt = blockDim.x;
  if (by_row) {
    for (int r = threadIdx.x; r < a.batch; r += nt) rows[r] = 0;
    __syncthreads();
  }
  const PolicyUnit p(a, rank * nt + threadIdx.x);
  const uint32_t bits = p.mask(a);
  PolicyQuad quad;
  if (bits) quad.load(a, p);
  if (by_row && bits) atomicAdd(&rows[p.row], __popc(bits));
  double weight = a.inv_norm;
  if (a.agg == kPolicyTokenMean) {
    double n[1] = {static_cast<double>(__popc(bits))};
    block_sums(n, red);
    cluster_sums(n, slots[0], C, rank, true);
    weight = 1.0 / fmax(n[0], 1.0);
  } else if (by_row) {
    if (C > 1) cluster_wait();
    __syncthreads();
    const uint32_t to = smem_u32(all_rows + rank * a.batch);
    for (int e = threadIdx.x; e < a.batch * C; e += nt) {
      const int c = e / a.batch, r = e - c * a.batch;
      st_cluster_s32(mapa_shared(to + 4 * r, c), rows[r]);
    }
    cluster_sync_all();
    if (bits) {
      int n = 0;
      for (int c = 0; c < C; ++c) n += all_rows[c * a.batch + p.row];
      weight = 1.0 / (static_cast<double>(n) * static_cast<double>(a.batch));
    }
  }
  float g[4] = {0.f, 0.f, 0.f, 0.f};
  double l = 0.0, kl = 0.0;
  int clips = 0;
  if (bits) quad.run(a, bits, static_cast<float>(weight), g, l, kl, clips);
  if (!(fabs(l) < kHuge && fabs(kl) < kHuge)) {
    float far_g[4] = {0.f, 0.f, 0.f, 0.f};
    double far_l = 0.0, far_kl = 0.0;
    far_terms(a, p, bits, weight, far_g, far_l, far_kl);
    kl = far_kl;
    if (!(fabs(l) < kHuge)) {  // else the KL terms alone are far, with kl_beta 0
      l = far_l;
#pragma unroll
      for (int j = 0; j < 4; ++j) g[j] = far_g[j];
    }
  }
  if (a.dlogp) p.store(a, g);
  double v[4] = {l * weight, kl, static_cast<double>(clips), static_cast<double>(__popc(bits))};
  block_sums(v, red);
  cluster_sums(v, slots[1], C, rank, a.agg == kPolicyConstant, false);
  if (rank == 0 && threadIdx.x == 0) write_stats(v, a.stats);
}

// Scored tokens among the 16 mask bytes from index i (a multiple of 16) on,
// inside [first, end).
__device__ __forceinline__ int count16(const PolicyArgs& a, int64_t i, int64_t first, int64_t end) {
  if (!a.mask) return static_cast<int>(min(i + 16, end) - max(i, first));
  int n = 0;
  if (a.vec16 && i >= first && i + 16 <= end) {
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(a.mask + i));
    n = __popc(nonzero_bytes(w.x)) + __popc(nonzero_bytes(w.y)) + __popc(nonzero_bytes(w.z)) +
        __popc(nonzero_bytes(w.w));
  } else {
    for (int64_t j = max(i, first); j < min(i + 16, end); ++j) n += __ldg(a.mask + j) != 0;
  }
  return n;
}

// Means over rows: the rows' weights, 1 / (batch * scored tokens), into
// weights[row] (one CTA or warp a row); else the scored tokens of everything, a
// partial sum a CTA, into counts[0 .. gridDim.x).  *ended = 0.
__global__ void __launch_bounds__(kThreads)
    policy_count_kernel(PolicyArgs a, int* __restrict__ counts, double* __restrict__ weights,
                        unsigned* __restrict__ ended) {
  pdl_trigger();
  if (blockIdx.x == 0 && threadIdx.x == 0) *ended = 0u;
  __shared__ int red[kThreads / 32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int n = 0;
  auto count_row = [&](int row, int at, int step) {
    const int64_t first = static_cast<int64_t>(row) * a.ld, end = first + a.seq;
    for (int64_t i = (first & ~int64_t{15}) + 16 * at; i < end; i += 16 * step) n += count16(a, i, first, end);
  };
  if (a.agg == kPolicySequenceMean && a.seq <= 1024) {  // a warp a row
    const int row = blockIdx.x * (kThreads / 32) + w;
    if (row < a.batch) count_row(row, lane, 32);
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0 && row < a.batch) weights[row] = 1.0 / (static_cast<double>(max(n, 1)) * static_cast<double>(a.batch));
    return;
  }
  if (a.agg == kPolicySequenceMean) {  // a CTA a row
    count_row(blockIdx.x, threadIdx.x, kThreads);
  } else if (a.seq <= 2048) {  // warps take rows in turn
    for (int row = blockIdx.x * (kThreads / 32) + w; row < a.batch; row += gridDim.x * (kThreads / 32))
      count_row(row, lane, 32);
  } else {  // the grid takes rows' pieces of 256 x 16 tokens in turn
    const int pieces = (a.seq + 15 + 16 * kThreads - 1) / (16 * kThreads);
    for (int64_t k = blockIdx.x; k < static_cast<int64_t>(a.batch) * pieces; k += gridDim.x) {
      const int row = static_cast<int>(k / pieces);
      const int64_t first = static_cast<int64_t>(row) * a.ld, end = first + a.seq;
      const int64_t i = (first & ~int64_t{15}) + 16 * ((k - static_cast<int64_t>(row) * pieces) * kThreads + threadIdx.x);
      if (i < end) n += count16(a, i, first, end);
    }
  }
  n = __reduce_add_sync(0xffffffffu, n);
  if (lane == 0) red[w] = n;
  __syncthreads();
  if (w == 0) {
    n = __reduce_add_sync(0xffffffffu, lane < kThreads / 32 ? red[lane] : 0);
    if (lane == 0) {
      if (a.agg == kPolicySequenceMean)
        weights[blockIdx.x] = 1.0 / (static_cast<double>(max(n, 1)) * static_cast<double>(a.batch));
      else
        counts[blockIdx.x] = n;
    }
  }
}

// The CTAs' partial sums, in order: loss, mean KL, share of clipped tokens, scored tokens.
__device__ __forceinline__ void sum_partials(const double* partial, int n, double* red, float* stats) {
  double v[4] = {0.0, 0.0, 0.0, 0.0};
  for (int i = threadIdx.x; i < n; i += kThreads)
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] += __ldcg(partial + i * 4 + k);
  block_sums(v, red);
  if (threadIdx.x == 0) write_stats(v, stats);
}
__global__ void __launch_bounds__(kThreads) policy_stats_kernel(const double* __restrict__ partial, int n,
                                                               float* __restrict__ stats) {
  pdl_trigger();
  pdl_wait();
  __shared__ double red[4 * 32];
  sum_partials(partial, n, red, stats);
}

__global__ void __launch_bounds__(kThreads, kMainBlocks)
    policy_main_kernel(PolicyArgs a, const int* __restrict__ counts, int n_counts, const double* __restrict__ weights,
                       double* partial, unsigned* ended) {
  pdl_trigger();
  pdl_wait();
  __shared__ double red[4 * 32];
  __shared__ bool last;
  double weight = a.inv_norm;  // of every token, but for means over rows: of the sums
  if (a.agg == kPolicyTokenMean) {
    double n[1] = {0.0};
    for (int i = threadIdx.x; i < n_counts; i += kThreads) n[0] += static_cast<double>(counts[i]);
    block_sums(n, red);
    weight = 1.0 / fmax(n[0], 1.0);
  }
  const bool by_row = a.agg == kPolicySequenceMean;
  if (by_row) weight = 1.0;
  float each = static_cast<float>(weight);
  double v[4] = {0.0, 0.0, 0.0, 0.0};
  int clips = 0;
  int64_t tokens = 0;
  // A CTA takes a run of units; the mask of the next one is fetched a turn
  // ahead, so that the loads it decides on wait for nothing
  const int64_t run = (a.units + gridDim.x - 1) / gridDim.x;
  const int64_t u_end = min(a.units, (blockIdx.x + 1) * run);
  int64_t u = blockIdx.x * run + threadIdx.x;
  PolicyUnit next(a, u < u_end ? u : a.units);
  uint32_t next_bits = next.mask(a);
  for (; u < u_end; u += kThreads) {
    const PolicyUnit p = next;
    const uint32_t bits = next_bits;
    float g[4] = {0.f, 0.f, 0.f, 0.f};
    PolicyQuad quad;
    if (bits) quad.load(a, p);
    if (u + kThreads < u_end) {
      next = PolicyUnit(a, u + kThreads);
      next_bits = next.mask(a);
    }
    if (bits) {
      if (by_row) {
        const double w = weights[p.row];
        each = static_cast<float>(w);
        double l = 0.0;
        quad.run(a, bits, each, g, l, v[1], clips);
        v[0] += l * w;
      } else {
        quad.run(a, bits, each, g, v[0], v[1], clips);
      }
      tokens += __popc(bits);
    }
    if (a.dlogp) p.store(a, g);
  }
  if (!(fabs(v[0]) < kHuge && fabs(v[1]) < kHuge)) {
    const bool all = !(fabs(v[0]) < kHuge);  // else the KL terms alone are far, with kl_beta 0
    if (all) v[0] = 0.0;
    v[1] = 0.0;
#pragma unroll 1
    for (u = blockIdx.x * run + threadIdx.x; u < u_end; u += kThreads) {
      const PolicyUnit p(a, u);
      const uint32_t bits = p.mask(a);
      if (!bits) continue;
      const double w = by_row ? weights[p.row] : weight;
      float g[4] = {0.f, 0.f, 0.f, 0.f};
      double l = 0.0;
      far_terms(a, p, bits, w, g, l, v[1]);
      if (!all) continue;
      v[0] += by_row ? l * w : l;
      if (a.dlogp) p.store(a, g);
    }
  }
  v[0] *= weight;
  v[2] = static_cast<double>(clips);
  v[3] = static_cast<double>(tokens);
  block_sums(v, red);
  if (threadIdx.x == 0) {
#pragma unroll
    for (int k = 0; k < 4; ++k) partial[blockIdx.x * 4 + k] = v[k];
    if (ended) {
      __threadfence();
      last = atomicAdd(ended, 1u) + 1u == gridDim.x;
    }
  }
  if (!ended) return;
  __syncthreads();
  if (last) {
    __threadfence();
    sum_partials(partial, gridDim.x, red, a.stats);
  }
}

bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

constexpr int kCountBlocks = 1184;  // CTAs of the token count: eight an SM

int policy_blocks(int64_t units) {
  const int64_t want = (units + kThreads - 1) / kThreads;
  return static_cast<int>(std::min<int64_t>(want, kMainBlocks * static_cast<int64_t>(gemm_num_sms())));
}

}  // namespace

cudaError_t preference_loss(PreferenceArgs a, cudaStream_t st) {
  a.vec = aligned(a.logp, 16) && aligned(a.ref, 16) && aligned(a.mask, 4) && aligned(a.dlogp, 16);
  // CTAs a pair: enough that a thread meets at most about four quads of each
  // row, but no more than keep the GPU's resident CTAs (8 an SM) busy
  int C = 1;
  const int quads = a.seq / 4 + 2;
  while (C < 8 && quads > 4 * C * kThreads && static_cast<int64_t>(a.pairs) * C < 8LL * gemm_num_sms()) C *= 2;
  a.cluster = C;
  const double e = a.smoothing;
  a.still = e > 0.0 ? std::log((1.0 - e) / e) : 0.0;
  return launch_cluster(preference_kernel, static_cast<unsigned>(a.pairs) * C, kThreads, C, 0, st, false, a);
}

constexpr size_t kEndedBytes = 16;  // CTAs of the main kernel that have ended

size_t policy_loss_workspace(int batch) {
  const size_t partial = sizeof(double) * 4 * kMainBlocks * static_cast<size_t>(gemm_num_sms());
  return partial + kEndedBytes + std::max(sizeof(int) * kCountBlocks, sizeof(double) * static_cast<size_t>(batch));
}

cudaError_t policy_loss(PolicyArgs a, void* ws, cudaStream_t st, int* launches) {
  a.vec16 = aligned(a.mask, 16);
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
  a.f_low = static_cast<float>(a.log_low);
  a.f_high = static_cast<float>(a.log_high);
  a.f_dual = static_cast<float>(a.log_dual);
  // how near to a border fp32 cannot be trusted: some steps of the largest
  double most = 1.0;
  for (double b : {a.log_low, a.log_high, a.log_dual})
    if (std::isfinite(b)) most = std::max(most, std::fabs(b));
  a.near = static_cast<float>(1e-6 * most);
  if (a.units <= kSmallUnits && (a.agg != kPolicySequenceMean || a.batch <= kSmallRows)) {
    // CTAs of 256 threads, of 1024 once a cluster of eight does not suffice
    const int nt = a.units <= kSmallCluster * kThreads ? kThreads : kSmallThreads;
    int C = 1;
    while (C * nt < a.units) C *= 2;
    const size_t smem = a.agg == kPolicySequenceMean ? sizeof(int) * C * a.batch : 0;
    if (launches) ++*launches;
    return launch_cluster(policy_small_kernel, C, nt, C, smem, st, false, a, C);
  }
  double* partial = static_cast<double*>(ws);
  char* behind = reinterpret_cast<char*>(partial + 4 * kMainBlocks * static_cast<size_t>(gemm_num_sms()));
  unsigned* ended = reinterpret_cast<unsigned*>(behind);
  int* counts = reinterpret_cast<int*>(behind + kEndedBytes);
  double* weights = reinterpret_cast<double*>(counts);  // the one or the other
  const bool was = pdl_enabled();
  set_pdl(false);
  cudaError_t e = cudaSuccess;
  int n_counts = 0;
  if (a.agg == kPolicySequenceMean) {
    n_counts = a.seq <= 1024 ? (a.batch + kThreads / 32 - 1) / (kThreads / 32) : a.batch;
  } else if (a.agg == kPolicyTokenMean) {
    n_counts = static_cast<int>(std::min<int64_t>(kCountBlocks, (a.units / 4 + kThreads - 1) / kThreads + 1));
  }
  if (n_counts) {
    e = launch_pdl(policy_count_kernel, n_counts, kThreads, 0, st, a, counts, weights, ended);
    set_pdl(true);
  }
  const int blocks = policy_blocks(a.units);
  if (launches) *launches += 2;  // the count and the main kernel, or the main kernel and the sums
  // The count has zeroed `ended`, by which the main kernel's last CTA knows itself and sums up: a launch less
  // (64 x 2047: 17.2 us a call against 18.7, where the host's launches take longer than the kernels; replayed
  // from a graph 8.5 against 8.2).  Without a count a kernel of its own sums up.
  if (e == cudaSuccess)
    e = launch_pdl(policy_main_kernel, blocks, kThreads, 0, st, a, counts, n_counts, weights, partial,
                   n_counts ? ended : nullptr);
  set_pdl(true);
  if (e == cudaSuccess && !n_counts) e = launch_pdl(policy_stats_kernel, 1, kThreads, 0, st, partial, blocks, a.stats);
  set_pdl(was);
  return e;
}

}  // namespace llmcu
