// Drafted decoding besides its attention (tree.hip), for gfx950: logits to the probabilities that are
// sampled from, the walk that accepts or refuses drafted tokens, and the accepted rows moved together
// in the caches.
#include <math.h>

#include "fx_device.h"
#include "fx_internal.h"

namespace fx {

// ---- probabilities -----------------------------------------------------------------------
//
// p_v = exp((l_v - m) / T) / sum over the kept u of exp((l_u - m) / T), m the row's maximum, kept: the
// top_k largest logits and the equals of the last of them (GPT.generate's rule).  HBM-bound: a row is
// read once and written once.  One workgroup a row.

constexpr int kProbThreads = 1024, kProbWaves = kProbThreads / 64;
constexpr float kDraftNegInf = -__builtin_huge_valf();

// a logit's bits in an order that unsigned comparison keeps, both zeros alike
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}

template <typename F>
__device__ __forceinline__ auto block_reduce(decltype(F::zero()) v, decltype(F::zero()) * sh) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = F::join(v, __shfl_xor(v, off, 64));
    __syncthreads();   // the last use of sh is over
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (int w = 1; w < kProbWaves; ++w) v = F::join(v, sh[w]);
    return v;
}
struct JoinMax {
    static __device__ __forceinline__ float zero() { return kDraftNegInf; }
    static __device__ __forceinline__ float join(float a, float b) { return fmaxf(a, b); }
};
struct JoinSum {
    static __device__ __forceinline__ float zero() { return 0.f; }
    static __device__ __forceinline__ float join(float a, float b) { return a + b; }
};
struct JoinSumD {
    static __device__ __forceinline__ double zero() { return 0.0; }
    static __device__ __forceinline__ double join(double a, double b) { return a + b; }
};
struct JoinCount {
    static __device__ __forceinline__ int zero() { return 0; }
    static __device__ __forceinline__ int join(int a, int b) { return a + b; }
};

// A row of V values from flat index i0 of a 16-byte aligned tensor, NP a 16-byte load: f(value, v) for
// every v of this thread's, the row's ragged ends by single loads
template <bool BF, typename Fn>
__device__ __forceinline__ void each_logit(const void* base, int64_t i0, int64_t V, Fn f) {
    constexpr int NP = BF ? 8 : 4;
    const int64_t head = min(V, (NP - i0 % NP) % NP), body = (V - head) / NP;
    auto one = [&](int64_t v) { return BF ? bf16_to_f32(static_cast<const uint16_t*>(base)[i0 + v]) : static_cast<const float*>(base)[i0 + v]; };
    for (int64_t i = threadIdx.x; i < body; i += kProbThreads) {
        const int64_t v = head + i * NP;
        float x[NP];
        const uint4 u = ld16(static_cast<const char*>(base) + (i0 + v) * (BF ? 2 : 4));
        if constexpr (BF) {
            unpack8(u, x);
        } else {
            x[0] = __uint_as_float(u.x), x[1] = __uint_as_float(u.y), x[2] = __uint_as_float(u.z), x[3] = __uint_as_float(u.w);
        }
#pragma unroll
        for (int e = 0; e < NP; ++e) f(x[e], v + e);
    }
    if ((int64_t)threadIdx.x < head) f(one(threadIdx.x), (int64_t)threadIdx.x);
    const int64_t v = head + body * NP + threadIdx.x;
    if (v < V) f(one(v), v);
}

template <bool BF>
__global__ void __launch_bounds__(kProbThreads) probs_kernel(const void* logits, float* probs, int64_t V, double temperature, int64_t top_k) {
    __shared__ float shf[kProbWaves];
    __shared__ int shi[kProbWaves];
    const int64_t i0 = (int64_t)blockIdx.x * V;
    float m = kDraftNegInf;
    bool nan = false;
    each_logit<BF>(logits, i0, V, [&](float x, int64_t) { m = fmaxf(m, x), nan |= x != x; });
    m = block_reduce<JoinMax>(m, shf);
    nan = __syncthreads_or(nan);
    float* out = probs + i0;
    if (nan || m == kDraftNegInf || m == __builtin_huge_valf()) {   // no probabilities
        const float v = !nan && m == kDraftNegInf ? 0.f : __builtin_nanf("");
        for (int64_t i = threadIdx.x; i < V; i += kProbThreads) out[i] = v;
        return;
    }
    uint32_t key = 0;   // logits from this key on are kept
    if (top_k > 0 && top_k < V) {
        // the largest key with top_k keys at or above it, a bit at a time
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t t = key | (1u << bit);
            int n = 0;
            each_logit<BF>(logits, i0, V, [&](float x, int64_t) { n += order_key(x) >= t; });
            if (block_reduce<JoinCount>(n, shi) >= top_k) key = t;
        }
    }
    // 2^((l - m) log2(e) / T): the difference is rounded once, the factor is held in two parts
    const double f = 1.4426950408889634 / temperature;
    const float hi = (float)f, lo = (float)(f - (double)hi);
    auto val = [&](float x) {
        const float d = x - m;
        const float y = d * hi;
        if (y < -200.f) return 0.f;   // -inf among them
        return exp2_fast(y) * (1.f + kLn2 * (fmaf(d, hi, -y) + d * lo));
    };
    float s = 0.f;
    each_logit<BF>(logits, i0, V, [&](float x, int64_t) { s += order_key(x) >= key ? val(x) : 0.f; });
    s = block_reduce<JoinSum>(s, shf);
    const float inv = 1.f / s;
    each_logit<BF>(logits, i0, V, [&](float x, int64_t v) { out[v] = order_key(x) >= key ? val(x) * inv : 0.f; });
}

int sampling_probs(const void* logits, bool bf16, float* probs, int64_t rows, int64_t V, double temperature, int64_t top_k, void* stream) {
    FX_REQUIRE(rows >= 0 && rows < 0x7fffffffLL && V >= 1 && V < 0x7fffffffLL, "sampling_probs: bad shape rows=%lld V=%lld", (long long)rows, (long long)V);
    FX_REQUIRE(temperature > 0.f && temperature < __builtin_huge_val(), "sampling_probs: temperature %g must be positive and finite", temperature);
    if (rows == 0) return 0;
    FX_REQUIRE(logits && probs && (((uintptr_t)logits | (uintptr_t)probs) & 15) == 0, "sampling_probs: logits and probs must be 16-byte aligned");
    if (bf16)
        hipLaunchKernelGGL((probs_kernel<true>), dim3((unsigned)rows), dim3(kProbThreads), 0, (hipStream_t)stream, logits, probs, V, temperature, top_k);
    else
        hipLaunchKernelGGL((probs_kernel<false>), dim3((unsigned)rows), dim3(kProbThreads), 0, (hipStream_t)stream, logits, probs, V, temperature, top_k);
    return check_launch("sampling_probs");
}

// ---- verification ------------------------------------------------------------------------
//
// The walk stands on a node (first the root) with target row p and draft row q, and asks its children
// in their order.  After a rejection the target is norm(max(p' - q, 0)), p' what it was; unnormalised
// that is max(p - c q, 0) with the sum S, where c <- c + S, S <- sum_v max(p_v - c q_v, 0) (from c = 0,
// S = 1: max(max(p - c q, 0) / S - q, 0) = max(p - (c + S) q, 0) / S), so no row is written and a
// rejection costs one pass over two rows.  Child i with token x is accepted where
// u_i S q(x) < max(p(x) - c q(x), 0).  Without draft rows a proposal is certain of its token: q(x) = 1
// there, and a rejection takes x out of p.  The last token is drawn from what is left of the last
// row by its running sum.  Sums and tests are in 64 bits: the tokens do not hang on a summation order.

constexpr int kVerNodes = 64;
constexpr int kVerSeg = 256;                      // values of a segment of the running sum
constexpr int64_t kVerMaxV = 1 << 20;
constexpr int kVerSegs = (int)(kVerMaxV / kVerSeg);

__global__ void __launch_bounds__(kProbThreads) verify_kernel(const float* probs, const float* draft, const int64_t* tokens, const int32_t* parents,
                                                              const float* uniform, int64_t* out, int32_t* path, int32_t* counts, int32_t N, int64_t V) {
    __shared__ int64_t tok[kVerNodes];
    __shared__ int par[kVerNodes], spath[kVerNodes];
    __shared__ float un[kVerNodes], pt[kVerNodes], qt[kVerNodes];
    __shared__ double seg[kVerSegs + 1], shd[kProbWaves];
    __shared__ int64_t last;
    const int64_t b = blockIdx.x;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const float* P = probs + b * N * V;
    const float* Q = draft ? draft + b * N * V : nullptr;
    if ((int)threadIdx.x < N) {
        const int i = threadIdx.x;
        const int64_t x = tokens[b * N + i];
        int p = parents[b * N + i];
        if (i == 0 || p < 0 || p >= i || x < 0 || x >= V) p = -1;   // the root; padding and what is no token are never asked
        tok[i] = x;
        par[i] = p;
        un[i] = uniform[b * N + i];
        pt[i] = p < 0 ? 0.f : fmaxf(P[p * V + x], 0.f);
        qt[i] = p < 0 || !Q ? 1.f : Q[p * V + x];
    }
    __syncthreads();

    int cur = 0, n = 0;
    uint64_t drop = 0;    // rejected children of cur (no draft rows)
    double c = 0.0, S = 1.0;
    bool stale = false;   // c has moved since S was formed
    auto weight = [&](int64_t v) {
        const float p = P[cur * V + v];
        if (Q) return fmax((double)p - c * (double)Q[cur * V + v], 0.0);
        for (uint64_t d = drop; d; d &= d - 1)
            if (tok[__ffsll((unsigned long long)d) - 1] == v) return 0.0;
        return (double)fmaxf(p, 0.f);
    };
    auto row_sum = [&] {
        double s = 0.0;
        for (int64_t v = threadIdx.x; v < V; v += kProbThreads) s += weight(v);
        return block_reduce<JoinSumD>(s, shd);
    };
    if (threadIdx.x == 0) spath[0] = 0;
    for (int i = 1; i < N; ++i) {
        if (par[i] != cur) continue;
        double left = (double)pt[i];
        if (Q) {
            if (stale) S = row_sum(), stale = false;
            left = fmax(left - c * (double)qt[i], 0.0);
        } else {
            for (uint64_t d = drop; d; d &= d - 1)
                if (tok[__ffsll((unsigned long long)d) - 1] == tok[i]) left = 0.0;
        }
        if ((double)un[i] * S * (double)qt[i] < left) {
            cur = i, c = 0.0, S = 1.0, drop = 0, stale = false;
            if (threadIdx.x == 0) spath[n + 1] = i;
            ++n;
        } else if (Q) {
            c += S;
            stale = true;
        } else {
            S -= left;
            drop |= 1ull << i;
        }
    }
    // segment sums of what is left, then of the row itself where nothing is
    const int64_t nseg = (V + kVerSeg - 1) / kVerSeg;
    double W = 0.0;
    for (int round = 0; round < 2; ++round) {
        for (int64_t s = w; s < nseg; s += kProbWaves) {
            double x = 0.0;
#pragma unroll
            for (int e = 0; e < kVerSeg / 64; ++e) {
                const int64_t v = s * kVerSeg + e * 64 + lane;
                if (v < V) x += weight(v);
            }
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
            if (lane == 0) seg[s] = x;
        }
        double x = 0.0;
        __syncthreads();
        for (int64_t s = threadIdx.x; s < nseg; s += kProbThreads) x += seg[s];
        W = block_reduce<JoinSumD>(x, shd);
        if (W > 0.0) break;
        c = 0.0, drop = 0;
        __syncthreads();
    }
    if (w == 0) {
        int64_t got = -1;
        if (W > 0.0 && W < __builtin_huge_val()) {
            const double at = (double)un[0] * W;
            // the first segment whose running sum passes `at`; by rounding none may: the last with weight
            double before = 0.0, base = 0.0;
            int64_t pick = -1, some = -1;
            double some_base = 0.0;
            for (int64_t s0 = 0; s0 < nseg && pick < 0; s0 += 64) {
                const double x = s0 + lane < nseg ? seg[s0 + lane] : 0.0;
                double up = x;
#pragma unroll
                for (int off = 1; off < 64; off <<= 1) {
                    const double o = __shfl_up(up, off, 64);
                    if (lane >= off) up += o;
                }
                const uint64_t past = __ballot(x > 0.0 && before + up > at), has = __ballot(x > 0.0);
                if (has) {
                    const int l = 63 - __clzll((long long)has);
                    some = s0 + l;
                    some_base = before + __shfl(up, l, 64) - __shfl(x, l, 64);
                }
                if (past) {
                    const int l = __ffsll((unsigned long long)past) - 1;
                    pick = s0 + l;
                    base = before + __shfl(up, l, 64) - __shfl(x, l, 64);
                }
                before += __shfl(up, 63, 64);
            }
            if (pick < 0) pick = some, base = some_base;
            // and the value within it, four of each lane's
            double x[kVerSeg / 64], sum = 0.0;
            const int64_t v0 = pick * kVerSeg + lane * (kVerSeg / 64);
#pragma unroll
            for (int e = 0; e < kVerSeg / 64; ++e) x[e] = v0 + e < V ? weight(v0 + e) : 0.0, sum += x[e];
            double up = sum;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const double o = __shfl_up(up, off, 64);
                if (lane >= off) up += o;
            }
            double run = base + (up - sum);
            int hit = -1, any = -1;
#pragma unroll
            for (int e = 0; e < kVerSeg / 64; ++e) {
                run += x[e];
                if (x[e] > 0.0) {
                    any = e;
                    if (hit < 0 && run > at) hit = e;
                }
            }
            const uint64_t hits = __ballot(hit >= 0), anys = __ballot(any >= 0);
            if (hits) {
                const int l = __ffsll((unsigned long long)hits) - 1;
                got = pick * kVerSeg + l * (kVerSeg / 64) + __shfl(hit, l, 64);
            } else if (anys) {
                const int l = 63 - __clzll((long long)anys);
                got = pick * kVerSeg + l * (kVerSeg / 64) + __shfl(any, l, 64);
            }
        }
        if (lane == 0) last = got;
    }
    __syncthreads();
    if ((int)threadIdx.x < N) {
        const int d = threadIdx.x;
        path[b * N + d] = d <= n ? spath[d] : -1;
        out[b * N + d] = d < n ? tok[spath[d + 1]] : d == n ? last : -1;
        if (d == 0) counts[b] = n + 1;
    }
}

int verify_draft(const float* probs, const float* draft, const int64_t* tokens, const int32_t* parents, const float* uniform,
                 int64_t* out, int32_t* path, int32_t* counts, int32_t B, int32_t N, int64_t V, void* stream) {
    FX_REQUIRE(B >= 0 && N >= 1 && N <= kVerNodes && V >= 1 && V <= kVerMaxV, "verify_draft: bad shape B=%d N=%d (up to %d) V=%lld (up to %lld)",
               B, N, kVerNodes, (long long)V, (long long)kVerMaxV);
    if (B == 0) return 0;
    FX_REQUIRE(probs && tokens && parents && uniform && out && path && counts, "verify_draft: null pointer");
    hipLaunchKernelGGL(verify_kernel, dim3((unsigned)B), dim3(kProbThreads), 0, (hipStream_t)stream, probs, draft, tokens, parents, uniform, out,
                       path, counts, N, V);
    return check_launch("verify_draft");
}

// ---- accepted rows together --------------------------------------------------------------
//
// Bound by the moved rows' bytes, read and written once.  A thread owns 16 bytes of a (tensor,
// sequence)'s row and moves them for every d: the path ascends, so a row that is written
// (ctx + d <= ctx + path[d]) is never one that is still to be read.

__global__ void __launch_bounds__(256) compact_kernel(CompactArgs a) {
    const int y = blockIdx.y, b = y % a.B, ten = y / a.B;
    const int ctx = a.ctx[b];
    int n = a.counts[b];
    n = n < 0 ? 0 : (n > a.N ? a.N : n);
    if (a.ctx_out && ten == 0 && blockIdx.x == 0 && threadIdx.x == 0) a.ctx_out[b] = ctx + n;
    const int i = blockIdx.x * 256 + threadIdx.x, cpr = a.D / 8;
    if (i >= a.H * cpr || ctx < 0) return;
    const int h = i / cpr, col = (i - h * cpr) * 8;
    uint16_t* p = a.at[ten] + b * a.sb[ten] + h * a.sh[ten] + col;
    const int64_t st = a.st[ten];
    for (int d = 0; d < n; ++d) {
        const int s = a.path[(int64_t)b * a.N + d];
        if (s <= d || s >= a.T - ctx) continue;   // in its place already, or no row of the cache
        st16(p + (int64_t)(ctx + d) * st, ld16(p + (int64_t)(ctx + s) * st));
    }
}

int compact_cache(const CompactArgs& a, void* stream) {
    FX_REQUIRE(a.count >= 1 && a.count <= kCompactTensors && a.B >= 1 && a.T >= 1 && a.H >= 1 && a.D >= 8 && a.D % 8 == 0 && a.N >= 1,
               "compact_cache: bad shape (%d tensors, B=%d T=%d H=%d D=%d N=%d)", a.count, a.B, a.T, a.H, a.D, a.N);
    FX_REQUIRE((int64_t)a.count * a.B <= 65535 && (int64_t)a.H * a.D <= 0x7fffffffLL, "compact_cache: grid too large");
    FX_REQUIRE(a.ctx && a.path && a.counts, "compact_cache: null pointer");
    for (int i = 0; i < a.count; ++i)
        FX_REQUIRE(a.at[i] && ((uintptr_t)a.at[i] & 15) == 0 && a.sb[i] % 8 == 0 && a.st[i] % 8 == 0 && a.sh[i] % 8 == 0,
                   "compact_cache: caches must be 16-byte aligned with strides of multiples of 8 elements");
    const unsigned chunks = (unsigned)((a.H * (a.D / 8) + 255) / 256);
    hipLaunchKernelGGL(compact_kernel, dim3(chunks, (unsigned)(a.count * a.B)), dim3(256), 0, (hipStream_t)stream, a);
    return check_launch("compact_cache");
}

}  // namespace fx
