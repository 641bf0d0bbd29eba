// The selection of a beam search's step, for gfx950: of all continuations of a sequence's K beams by one of
// V tokens, the best K.
//
//   s[k, v] = score[k] + l[k, v] - log sum_u exp(l[k, u]),   ranked by w[k] s[k, v];
//
// a beam that is done has one continuation, itself.  Equal ranks go to the lower beam, then to the
// larger logit, then to the lower token.  Within a beam the order is that of the logits, so each row is
// cut into chunks, a workgroup each, which keep their best K logits and the sum of their exponentials;
// a second kernel, a workgroup a sequence, joins them.  Sums beside the exponentials' own are in 64 bits: what
// order two beams' continuations have is decided there.
//
// HBM-bound: the logits are read once.  A chunk lies in registers.  64 groups of its logits have a
// maximum each; the K-th largest of these is at most the chunk's K-th logit, and few logits lie above
// it: they are listed and ranked by counting.
#include <math.h>

#include "fx_device.h"
#include "fx_internal.h"

namespace fx {

constexpr int kBeamThreads = 256, kBeamWaves = kBeamThreads / 64;
constexpr int kBeamList = 512;      // logits of the list
constexpr float kBeamNegInf = -__builtin_huge_valf();

// bits in an order that unsigned comparison keeps, both zeros alike
__device__ __forceinline__ uint32_t beam_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float beam_logit(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }
// the same of a rank; NaN above all
__device__ __forceinline__ uint64_t rank_key(double x) {
    if (x != x) return ~0ull;
    const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
    return b ^ ((b >> 63) ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ uint64_t shfl_xor64(uint64_t x, int off) {
    return (uint64_t)(uint32_t)__shfl_xor((int)(uint32_t)x, off, 64) | (uint64_t)(uint32_t)__shfl_xor((int)(uint32_t)(x >> 32), off, 64) << 32;
}
__device__ __forceinline__ uint64_t wave_max64(uint64_t x) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const uint64_t o = shfl_xor64(x, off);
        x = o > x ? o : x;
    }
    return x;
}

// chunks of a row, and logits of each (a whole number of vectors; the last is shorter)
struct BeamPlan {
    int32_t chunks, length;
};

// the workspace: of each row and chunk the best K (logit's key, complement of the token; 0: none), then the maximum and sum
__device__ __forceinline__ uint64_t* beam_lists(const BeamArgs& a) { return static_cast<uint64_t*>(a.work); }
__device__ __forceinline__ float2* beam_stats(const BeamArgs& a, const BeamPlan& p) {
    return reinterpret_cast<float2*>(beam_lists(a) + (int64_t)a.B * a.K * p.chunks * a.K);
}
// a beam with continuations by its logits
__device__ __forceinline__ bool beam_goes_on(const BeamArgs& a, int64_t row) {
    const float s = a.scores[row];
    return !(a.done && a.done[row]) && s == s && s != kBeamNegInf;
}

template <bool BF, int NR>
__global__ void __launch_bounds__(kBeamThreads) beam_chunk_kernel(BeamArgs a, BeamPlan plan) {
    constexpr int NP = BF ? 8 : 4;
    __shared__ float gmax[kBeamWaves][64], shm[kBeamWaves], shs[kBeamWaves];
    __shared__ uint32_t bound;
    __shared__ int listed;
    __shared__ uint64_t list[kBeamList];
    const int64_t row = blockIdx.x / plan.chunks;
    const int chunk = (int)(blockIdx.x - row * plan.chunks);
    if (!beam_goes_on(a, row)) return;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    // flat places: the chunk's first and last, and the first vector
    const int64_t i0 = row * a.V + (int64_t)chunk * plan.length;
    const int64_t i1 = min(i0 + plan.length, (row + 1) * a.V), f0 = i0 / NP * NP;

    float x[NR][NP];
    uint4 raw[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const int64_t f = f0 + (int64_t)(i * kBeamThreads + tid) * NP;
        const uint32_t ninf = BF ? 0xff80ff80u : 0xff800000u;
        raw[i] = make_uint4(ninf, ninf, ninf, ninf);
        if (f >= i0 && f + NP <= i1) raw[i] = ld16(static_cast<const char*>(a.logits) + f * (BF ? 2 : 4));
    }
    float own = kBeamNegInf;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const int64_t f = f0 + (int64_t)(i * kBeamThreads + tid) * NP;
        if constexpr (BF) unpack8(raw[i], x[i]);
        else x[i][0] = __uint_as_float(raw[i].x), x[i][1] = __uint_as_float(raw[i].y), x[i][2] = __uint_as_float(raw[i].z), x[i][3] = __uint_as_float(raw[i].w);
        if (f < i1 && f + NP > i0 && !(f >= i0 && f + NP <= i1)) {   // the chunk's ragged ends
#pragma unroll
            for (int e = 0; e < NP; ++e)
                if (f + e >= i0 && f + e < i1)
                    x[i][e] = BF ? bf16_to_f32(static_cast<const uint16_t*>(a.logits)[f + e]) : static_cast<const float*>(a.logits)[f + e];
        }
#pragma unroll
        for (int e = 0; e < NP; e += 2) {
            own = fmaxf(own, fmaxf(x[i][e], x[i][e + 1]));
            nan |= __builtin_isunordered(x[i][e], x[i][e + 1]);
        }
    }
    // the sum above the thread's own maximum, before the workgroup waits for the slowest of its loads
    const float mine = own == kBeamNegInf ? 0.f : own;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int e = 0; e < NP; ++e) s += exp2_fast((x[i][e] - mine) * kLog2e);

    if (tid == 0) listed = 0;
    gmax[w][lane] = own;
    nan = __syncthreads_or(nan);
    __syncthreads();
    float m = kBeamNegInf;
    if (w == 0) {
        float g = gmax[0][lane];
#pragma unroll
        for (int i = 1; i < kBeamWaves; ++i) g = fmaxf(g, gmax[i][lane]);
        const uint32_t k = beam_key(g);
        uint32_t lo = k, hi = k;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            lo = min(lo, (uint32_t)__shfl_xor((int)lo, off, 64));
            hi = max(hi, (uint32_t)__shfl_xor((int)hi, off, 64));
        }
        lo = __builtin_amdgcn_readfirstlane(lo);
        hi = __builtin_amdgcn_readfirstlane(hi);
        if (lane == 0) shm[0] = beam_logit(hi);
        // a bound with K or a few more group maxima at or above it
        int have = 64;
        while (lo < hi && have > a.K + a.K / 4) {
            const uint32_t mid = lo + (hi - lo) / 2 + 1;
            const int c = __popcll(__ballot(k >= mid));
            if (c >= a.K) lo = mid, have = c;
            else hi = mid - 1;
        }
        if (lane == 0) bound = lo;
    }
    __syncthreads();
    m = shm[0];
    const float least = beam_logit(bound);
    const int64_t place = row * plan.chunks + chunk;
    uint64_t* out = beam_lists(a) + place * a.K;
    float2* stat = beam_stats(a, plan) + place;
    if (nan || m == __builtin_huge_valf()) {   // no sum: the beam's score is NaN
        if (tid == 0) *stat = make_float2(__builtin_nanf(""), 0.f);
        for (int i = tid; i < a.K; i += kBeamThreads) out[i] = 0;
        return;
    }
    s *= exp2_fast((mine - m) * kLog2e);   // a thread without logits: mine is 0 and s 0
    if (own == kBeamNegInf) s = 0.f;
    s = group_sum<64>(s);
    if (lane == 0) shs[w] = s;

    auto key = [&](int i, int e) {
        const uint32_t tok = (uint32_t)(f0 + (int64_t)(i * kBeamThreads + tid) * NP + e - row * a.V);
        return (uint64_t)beam_key(x[i][e]) << 32 | (0xffffffffu - tok);
    };
    if (own >= least && own > kBeamNegInf) {
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int e = 0; e < NP; ++e)
                if (x[i][e] >= least && x[i][e] > kBeamNegInf) {
                    const int at = atomicAdd(&listed, 1);
                    if (at < kBeamList) list[at] = key(i, e);
                }
    }
    __syncthreads();
    if (tid == 0) {
        float z = shs[0];
#pragma unroll
        for (int i = 1; i < kBeamWaves; ++i) z += shs[i];
        *stat = make_float2(m, m == kBeamNegInf ? 0.f : z);
    }
    const int n = listed;
    if (n <= kBeamList) {
        for (int i = tid; i < n; i += kBeamThreads) {
            const uint64_t k = list[i];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += list[j] > k;
            if (rank < a.K) out[rank] = k;
        }
        for (int i = n + tid; i < a.K; i += kBeamThreads) out[i] = 0;
        return;
    }
    // many equals: the best one by one, each below the last
    uint64_t last = ~0ull;
    for (int j = 0; j < a.K; ++j) {
        uint64_t best = 0;
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int e = 0; e < NP; ++e) {
                const uint64_t k = x[i][e] > kBeamNegInf ? key(i, e) : 0;
                if (k < last && k > best) best = k;
            }
        best = wave_max64(best);
        __syncthreads();   // the last round's are read
        if (lane == 0) list[w] = best;
        __syncthreads();
        best = list[0];
#pragma unroll
        for (int i = 1; i < kBeamWaves; ++i) best = list[i] > best ? list[i] : best;
        if (tid == 0) out[j] = best;
        last = best;   // 0 where none is left: so is what follows
    }
}

// A workgroup a sequence.  A wave a row at a time: the sum of its chunks' exponentials, and its best K of the
// chunks' lists, which are sorted: a lane holds the head of a list.  Then one wave merges the rows' lists the same way.
__global__ void __launch_bounds__(1024) beam_join_kernel(BeamArgs a, BeamPlan plan) {
    __shared__ uint64_t best[kBeamMost][kBeamMost];
    __shared__ float top[kBeamMost];      // a row's largest logit, and the logarithm of its sum
    __shared__ double logs[kBeamMost];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int64_t row0 = (int64_t)blockIdx.x * a.K;
    for (int k = w; k < a.K; k += waves) {
        const int64_t row = row0 + k;
        if (!beam_goes_on(a, row)) continue;
        const float2* st = beam_stats(a, plan) + row * plan.chunks;
        float m = kBeamNegInf;
        bool nan = false;
        for (int c = lane; c < plan.chunks; c += 64) m = fmaxf(m, st[c].x), nan |= st[c].x != st[c].x;
        m = group_max<64>(m);
        double z = 0.0;
        for (int c = lane; c < plan.chunks; c += 64)
            if (st[c].x != kBeamNegInf) z += (double)st[c].y * exp((double)st[c].x - (double)m);
        z = group_sum_d<64>(z);
        const bool bad = __ballot(nan) != 0;
        if (lane == 0) top[k] = m, logs[k] = bad ? __builtin_nan("") : log(z);
        if (bad) continue;
        constexpr int LL = 2;   // lists of a lane: 128 chunks at most
        const uint64_t* at[LL];
        uint64_t head[LL], next[LL];
        int left[LL];
#pragma unroll
        for (int i = 0; i < LL; ++i) {
            const int c = lane + 64 * i;
            at[i] = beam_lists(a) + (row * plan.chunks + min(c, plan.chunks - 1)) * a.K;
            left[i] = c < plan.chunks ? a.K : 0;
            head[i] = left[i] > 0 ? at[i][0] : 0;
            next[i] = left[i] > 1 ? at[i][1] : 0;
        }
        for (int j = 0; j < a.K; ++j) {
            const uint64_t first = wave_max64(head[0] > head[1] ? head[0] : head[1]);
            if (lane == 0) best[k][j] = first;
#pragma unroll
            for (int i = 0; i < LL; ++i)
                if (first && head[i] == first) {   // keys hold their tokens: no two are alike
                    head[i] = next[i];
                    --left[i], ++at[i];
                    next[i] = left[i] > 1 ? at[i][1] : 0;
                }
        }
    }
    __syncthreads();
    if (w != 0) return;
    // lane k: the head of row k's list
    const int k = lane;
    const int64_t row = row0 + min(k, a.K - 1);
    const float score = a.scores[row];
    const bool goes = beam_goes_on(a, row), single = !goes && (a.done && a.done[row] ? score != kBeamNegInf : score != score);
    const double weight = a.weight ? (double)a.weight[row] : 1.0, most = top[min(k, a.K - 1)], less = logs[min(k, a.K - 1)];
    const bool bad = goes && less != less;
    int j = 0;
    double sum = 0.0;
    uint64_t rank = 0;
    auto take = [&] {   // the list's head: its score and rank; the least rank where there is none
        rank = 0;
        sum = (double)kBeamNegInf;
        if (k >= a.K) return;
        if (goes && !bad) {
            const uint64_t b = j < a.K ? best[k][j] : 0;
            if (b) sum = (double)score + (((double)beam_logit((uint32_t)(b >> 32)) - most) - less);
        } else if (j == 0 && (single || bad)) {
            sum = bad ? __builtin_nan("") : (double)score;
        }
        const double r = sum == (double)kBeamNegInf ? sum : weight * sum;
        rank = r == (double)kBeamNegInf ? 0 : rank_key(r);
    };
    take();
    for (int i = 0; i < a.K; ++i) {
        const uint64_t first = wave_max64(rank);
        const int64_t at = row0 + i;
        if (first == 0) {
            if (lane == 0) a.out[at] = kBeamNegInf, a.rows[at] = -1, a.tokens[at] = a.fill;
            continue;
        }
        const int win = __ffsll((unsigned long long)__ballot(rank == first)) - 1;   // equals: the lower beam
        if (lane == win) {
            a.out[at] = (float)sum;
            a.rows[at] = (int32_t)row;
            a.tokens[at] = goes && !bad ? (int64_t)(0xffffffffu - (uint32_t)best[k][j]) : a.fill;
            ++j;
            take();
        }
    }
}

static BeamPlan beam_plan(int32_t B, int32_t K, int64_t V, bool bf16) {
    BeamPlan p{};
    constexpr int64_t most = 8192;
    p.chunks = (int32_t)((V + most - 1) / most);
    p.length = (int32_t)(((V + p.chunks - 1) / p.chunks + 7) / 8 * 8);
    p.chunks = (int32_t)((V + p.length - 1) / p.length);
    return p;
}

int64_t beam_select_workspace(int32_t B, int32_t K, int64_t V, bool bf16) {
    if (B < 1 || K < 1 || K > kBeamMost || V < 1 || V > kBeamVocab) return 0;
    const BeamPlan p = beam_plan(B, K, V, bf16);
    return (int64_t)B * K * p.chunks * (K + 1) * (int64_t)sizeof(uint64_t);
}

int beam_select(const BeamArgs& a, void* stream) {
    FX_REQUIRE(a.B >= 1 && a.K >= 1 && a.K <= kBeamMost, "beam_select: %d beams (1 to %d) of %d sequences", a.K, kBeamMost, a.B);
    FX_REQUIRE(a.V >= 1 && a.V <= kBeamVocab, "beam_select: %lld logits a row (1 to %lld)", (long long)a.V, (long long)kBeamVocab);
    FX_REQUIRE(a.logits && a.scores && a.out && a.rows && a.tokens && a.work, "beam_select: null pointer");
    FX_REQUIRE((((uintptr_t)a.logits | (uintptr_t)a.work) & 15) == 0, "beam_select: logits and work must be 16-byte aligned");
    const BeamPlan p = beam_plan(a.B, a.K, a.V, a.bf16);
    const int64_t grid = (int64_t)a.B * a.K * p.chunks;
    FX_REQUIRE(grid < (1 << 23), "beam_select: too many rows");   // a launch has less than 2^32 work items
    // NR vectors a thread: one more vector than the chunk's, where its first logit is not a vector's first
    if (a.bf16)
        hipLaunchKernelGGL((beam_chunk_kernel<true, 5>), dim3((unsigned)grid), dim3(kBeamThreads), 0, (hipStream_t)stream, a, p);
    else
        hipLaunchKernelGGL((beam_chunk_kernel<false, 9>), dim3((unsigned)grid), dim3(kBeamThreads), 0, (hipStream_t)stream, a, p);
    if (int e = check_launch("beam_select")) return e;
    const int waves = a.K < 16 ? a.K : 16;
    hipLaunchKernelGGL(beam_join_kernel, dim3((unsigned)a.B), dim3(64 * waves), 0, (hipStream_t)stream, a, p);
    return check_launch("beam_select_join");
}

}  // namespace fx
