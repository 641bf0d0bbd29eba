// The selection of a beam search's step, for gfx950: of all continuations of a sequence's K beams by one of
// V tokens, the best K.
//
//   s[k, v] = score[k] + l[k, v] - log sum_u exp(l[k, u]),   ranked by w[k] s[k, v];
//
// a beam that is done has one continuation, itself.  Equal ranks go to the lower beam, then to the
// larger logit, then to the lower token.  Within a beam the order is that of the logits, so each row is
// cut into chunks, a workgroup each, which keep their best K logits and the sum of their exponentials;
// a second kernel, a workgroup a sequence, joins them.  Exponentials and a chunk's sum of them are in 32 bits, which
// leaves log sum exp off by at most 66 2^-23 and 3 2^-24 of the mean distance from the maximum, and all behind them in 64: rows of
// equal logits have equal sums, and ranks of unlike rows that are nearer than that may go either way.
//
// HBM-bound: the logits are read once.  A chunk lies in registers.  64 groups of its logits have a
// maximum each; the K-th largest of these is at most the chunk's K-th logit, and few logits lie above
// it: they are listed and ranked by counting.
//
// 32 sequences of 8 beams over 131,071 bf16 tokens, a quarter of the beams done (50 MB): 27 us, 19 of them the chunks (2.6 TB/s;
// with nothing but its loads that kernel takes 13.5, the exponentials and the lists are 2.5 each), 7.5 the join.  512 beams
// of 50,304 fp32 (103 MB) 32.  One sequence of 4 beams of 50,304 9.5: the two launches' chains of round trips.
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
// Reductions over a wave by lane shifts (row_shr 1, 2, 4, 8, then broadcasts of lanes 15 and 31): the last lane's, for all.
// A lane that nothing is shifted to takes `old`.
template <int CTRL>
__device__ __forceinline__ uint32_t shifted(uint32_t old, uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)old, (int)x, CTRL, 0xf, 0xf, false);
}
template <int CTRL>
__device__ __forceinline__ uint64_t shifted(uint64_t old, uint64_t x) {
    return (uint64_t)shifted<CTRL>((uint32_t)(old >> 32), (uint32_t)(x >> 32)) << 32 | shifted<CTRL>((uint32_t)old, (uint32_t)x);
}
__device__ __forceinline__ float last_lane(float x) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), 63)); }
__device__ __forceinline__ uint64_t last_lane(uint64_t x) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), 63) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, 63);
}
#define FX_WAVE_STEPS(step) step(0x111) step(0x112) step(0x114) step(0x118) step(0x142) step(0x143)
__device__ __forceinline__ float wave_max(float x) {
#define FX_STEP(c) x = fmaxf(x, __uint_as_float(shifted<c>(__float_as_uint(x), __float_as_uint(x))));
    FX_WAVE_STEPS(FX_STEP)
#undef FX_STEP
    return last_lane(x);
}
__device__ __forceinline__ float wave_sum(float x) {
#define FX_STEP(c) x += __uint_as_float(shifted<c>(0u, __float_as_uint(x)));
    FX_WAVE_STEPS(FX_STEP)
#undef FX_STEP
    return last_lane(x);
}
__device__ __forceinline__ double wave_sum(double x) {
#define FX_STEP(c) x += __longlong_as_double((long long)shifted<c>((uint64_t)0, (uint64_t)__double_as_longlong(x)));
    FX_WAVE_STEPS(FX_STEP)
#undef FX_STEP
    return __longlong_as_double((long long)last_lane((uint64_t)__double_as_longlong(x)));
}
__device__ __forceinline__ uint64_t wave_max64(uint64_t x) {
#define FX_STEP(c) { const uint64_t o = shifted<c>(x, x); x = o > x ? o : x; }
    FX_WAVE_STEPS(FX_STEP)
#undef FX_STEP
    return last_lane(x);
}
#undef FX_WAVE_STEPS

// chunks of a row, and logits of each (a whole number of vectors; the last is shorter)
struct BeamPlan {
    int32_t chunks, length;
    bool few;   // short chunks
};

// the workspace: of each row and chunk the best K (logit's key, complement of the token; 0: none), then the maximum and sum
__device__ __forceinline__ uint64_t* beam_lists(const BeamArgs& a) { return static_cast<uint64_t*>(a.work); }
__device__ __forceinline__ float2* beam_stats(const BeamArgs& a, const BeamPlan& p) {
    return reinterpret_cast<float2*>(beam_lists(a) + (int64_t)a.B * a.K * p.chunks * a.K);
}
// a beam with continuations by its logits
__device__ __forceinline__ bool beam_goes_on(const BeamArgs& a, int64_t row) {
    const float s = a.scores[row];
    const int d = a.done ? a.done[row] : 0;   // (both loads at once)
    return !d & (s == s) & (s != kBeamNegInf);
}

// A thread's part of a chunk: NR vectors of 16 bytes, as they lie in memory.  What a pass makes of a vector is not kept for the next.
// Vectors begin with the chunk, at whatever address that is: so what a thread sums, and in which order, is a matter of the row's
// places alone, and rows of equal logits have equal sums, bit for bit.
template <bool BF, int NR>
struct BeamChunk {
    static constexpr int NP = BF ? 8 : 4;
    uint4 raw[NR];
    float edge;           // one logit of the ragged end
    int tok0, edge_tok;   // the tokens of the first vector's first value and of the edge

    __device__ __forceinline__ static void unpack(const uint4& u, float* f) {
        if constexpr (BF) unpack8(u, f);
        else f[0] = __uint_as_float(u.x), f[1] = __uint_as_float(u.y), f[2] = __uint_as_float(u.z), f[3] = __uint_as_float(u.w);
    }
    // flat places [i0, i1) of the logits, from token `tok` of a row on; what is not theirs is -inf: neither listed nor summed
    __device__ __forceinline__ void load(const void* logits, int64_t i0, int64_t i1, int tok) {
        struct __attribute__((packed, aligned(BF ? 2 : 4))) Vector { uint4 x; };   // at a logit's address
        const char* base = static_cast<const char*>(logits) + i0 * (BF ? 2 : 4);
        const int n = (int)(i1 - i0), tid = threadIdx.x, whole = n / NP;
        const uint32_t ninf = BF ? 0xff80ff80u : 0xff800000u;
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const int v = tid + i * kBeamThreads;
            raw[i] = make_uint4(ninf, ninf, ninf, ninf);
            if (v < whole) raw[i] = reinterpret_cast<const Vector*>(base + (uint32_t)v * 16u)->x;
        }
        const int at = whole * NP + tid;
        edge = kBeamNegInf;
        if (at < n) edge = BF ? bf16_to_f32(reinterpret_cast<const uint16_t*>(base)[at]) : reinterpret_cast<const float*>(base)[at];
        tok0 = tok + tid * NP;
        edge_tok = tok + at;
    }
    // f(its number, its values, the first value's token) of every vector
    template <typename Fn>
    __device__ __forceinline__ void each(Fn f) {
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            asm volatile("" : "+v"(raw[i].x), "+v"(raw[i].y), "+v"(raw[i].z), "+v"(raw[i].w));
            float x[NP];
            unpack(raw[i], x);
            f(i, x, (uint32_t)(tok0 + i * kBeamThreads * NP));
            __builtin_amdgcn_sched_barrier(0);
        }
    }
};

__device__ __forceinline__ uint64_t beam_entry(float x, uint32_t tok) { return (uint64_t)beam_key(x) << 32 | (0xffffffffu - tok); }

template <bool BF, int NR>
__global__ void __launch_bounds__(kBeamThreads, 8) beam_chunk_kernel(BeamArgs a, BeamPlan plan) {
    constexpr int NP = BF ? 8 : 4;
    __shared__ float gmax[kBeamWaves][64], shs[kBeamWaves];
    __shared__ int listed;
    __shared__ uint64_t list[kBeamList];
    const int64_t row = blockIdx.x / plan.chunks;
    const int chunk = (int)(blockIdx.x - row * plan.chunks);
    if (!beam_goes_on(a, row)) return;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int64_t i0 = row * a.V + (int64_t)chunk * plan.length, i1 = min(i0 + plan.length, (row + 1) * a.V);
    BeamChunk<BF, NR> c;
    c.load(a.logits, i0, i1, chunk * plan.length);
    if (tid == 0) listed = 0;
    // One pass as the vectors come: the thread's largest and each vector's, and the sum of 2^(x log2 e - r) above a reference, the
    // first vector's largest, r rounded (what it is rounded by is taken from the sum).  A reference too far from the thread's
    // largest, a NaN or +inf: once more above the largest itself, which gives NaN for the last two.
    float own = kBeamNegInf, most[NR], about = 0.f, ref = 0.f, s = 0.f;
    c.each([&](int i, const float* x, uint32_t) {
        most[i] = fmaxf(x[0], x[1]);
#pragma unroll
        for (int e = 2; e < NP; e += 2) most[i] = fmaxf(most[i], fmaxf(x[e], x[e + 1]));
        own = fmaxf(own, most[i]);
        if (i == 0) {
            about = fabsf(own) < 1e38f ? own : 0.f;
            ref = about * kLog2e;
        }
        float t = 0.f;
#pragma unroll
        for (int e = 0; e < NP; e += 2) {
            s += exp2_fast(fmaf(x[e], kLog2e, -ref));
            t += exp2_fast(fmaf(x[e + 1], kLog2e, -ref));
        }
        s += t;
        asm volatile("" : "+v"(s), "+v"(own));
    });
    own = fmaxf(own, c.edge);   // (loaded last)
    s += exp2_fast(fmaf(c.edge, kLog2e, -ref));
    s *= exp2_fast(-fmaf(about, kLog2e, -ref));
    if (own == kBeamNegInf && s == 0.f) about = own;   // none of its own
    else if (!(fabsf(own - about) < 60.f)) {
        about = own == kBeamNegInf ? 0.f : own;
        s = exp2_fast((c.edge - about) * kLog2e);
        c.each([&](int, const float* x, uint32_t) {
#pragma unroll
            for (int e = 0; e < NP; ++e) s += exp2_fast((x[e] - about) * kLog2e);
            asm volatile("" : "+v"(s));
        });
    }
    gmax[w][lane] = s != s ? s : own;
    __syncthreads();
    // every wave by itself: the chunk's maximum, and a bound with K or a few more group maxima at or above it
    float g = gmax[0][lane];
    bool bad = g != g;
#pragma unroll
    for (int i = 1; i < kBeamWaves; ++i) bad |= gmax[i][lane] != gmax[i][lane], g = fmaxf(g, gmax[i][lane]);
    const float m = wave_max(g);
    const int64_t place = row * plan.chunks + chunk;
    uint64_t* out = beam_lists(a) + place * a.K;
    float2* stat = beam_stats(a, plan) + place;
    if (__ballot(bad)) {   // no sum: the beam's score is NaN
        if (tid == 0) *stat = make_float2(__builtin_nanf(""), 0.f);
        for (int i = tid; i < a.K; i += kBeamThreads) out[i] = 0;
        return;
    }
    const uint32_t k = beam_key(g), top = beam_key(m);
    // (logits of -inf continue nothing)
    uint32_t lo = beam_key(kBeamNegInf) + 1, hi = top;
    int have = __popcll(__ballot(k >= lo));
    if (have > a.K) {
        // the search begins above the least of the maxima
        lo = beam_key(-wave_max(k >= lo ? -g : kBeamNegInf));
        while (lo < hi && have > a.K + a.K / 4) {
            const uint32_t mid = lo + (hi - lo) / 2 + 1;
            const int n = __popcll(__ballot(k >= mid));
            if (n >= a.K) lo = mid, have = n;
            else hi = mid - 1;
        }
    }
    s = about == kBeamNegInf ? 0.f : s * exp2_fast((about - m) * kLog2e);
    s = wave_sum(s);
    if (lane == 0) shs[w] = s;
    const float least = beam_logit(lo);
    auto put = [&](float x, uint32_t tok) {
        const int at = atomicAdd(&listed, 1);
        if (at < kBeamList) list[at] = beam_entry(x, tok);
    };
    if (own >= least) {
        c.each([&](int i, const float* x, uint32_t tok) {
            if (most[i] >= least)
#pragma unroll
                for (int e = 0; e < NP; ++e)
                    if (x[e] >= least) put(x[e], tok + e);
        });
        if (c.edge >= least) put(c.edge, c.edge_tok);
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
            const uint64_t x = list[i];
            int rank = 0;
#pragma unroll 8
            for (int j = 0; j < n; ++j) rank += list[j] > x;
            if (rank < a.K) out[rank] = x;
        }
        for (int i = n + tid; i < a.K; i += kBeamThreads) out[i] = 0;
        return;
    }
    // many equals: the best one by one, each below the last, from memory
    uint64_t last = ~0ull;
    for (int j = 0; j < a.K; ++j) {
        uint64_t best = 0;
        for (int64_t f = i0 + tid; f < i1; f += kBeamThreads) {
            const float x = BF ? bf16_to_f32(static_cast<const uint16_t*>(a.logits)[f]) : static_cast<const float*>(a.logits)[f];
            const uint64_t y = x > kBeamNegInf ? beam_entry(x, (uint32_t)(f - row * a.V)) : 0;
            if (y < last && y > best) best = y;
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

// A continuation as it is ranked: its rank's key, then one of the beam, the logit and the token
struct BeamRank {
    uint64_t rank, rest;
    __device__ __forceinline__ bool above(const BeamRank& o) const { return rank > o.rank || (rank == o.rank && rest > o.rest); }
};

// A workgroup a sequence, bounded by its chain of round trips and waits.  Only what is not below the least of the rows' best
// continuations is looked at (where each row has one, K are not): of the chunks' lists, which are sorted, those with such a head;
// where these are many, only the K lists with the best heads, in which the best K continuations lie, and what is
// not below the last of their heads.  What remains is ranked by counting, of a few threads for each.  (Of 32 beams with a chunk a row
// that is most of K K, each compared with all: 4 sequences over 256 or 1,000 tokens 65 us, 9,000 45, 50,304 29; 16 beams 9 to 11.)
constexpr int kBeamJoin = 1024, kBeamChunks = 130;
constexpr int kBeamStage = kBeamMost * kBeamChunks;   // entries in LDS

struct BeamJoin {
    uint64_t stage[kBeamStage];                 // the lists' heads
    BeamRank head[kBeamStage];                  // the heads that are ranked
    int from[kBeamStage];                       // and their lists
    BeamRank cand[kBeamMost * kBeamMost];       // the last lists' continuations
    uint64_t entry[kBeamMost * kBeamMost];      // and their entries
    int row[kBeamMost * kBeamMost];             // and rows
    uint64_t best[kBeamMost], last;             // the rank of a row's best, of the last of the best heads
    double logs[kBeamMost], weight[kBeamMost];  // the logarithm of a row's sum, its weight
    float top[kBeamMost], score[kBeamMost];     // its largest logit, its score
    int chosen[kBeamMost], kind[kBeamMost], n, m;
};

__global__ void __launch_bounds__(kBeamJoin) beam_join_kernel(BeamArgs a, BeamPlan plan) {
    __shared__ BeamJoin j;
    enum { kNone, kLogits, kItself, kNaN };     // a row's continuations: none, those of its logits, itself, itself as NaN
    constexpr int kParts = (kBeamChunks + 63) / 64;
    constexpr uint64_t kSelf = 0xffffffffull;   // the entry of a row that goes on as it is (a logit's key and a token of 0)
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, threads = blockDim.x, S = plan.chunks, K = a.K;
    const int64_t row0 = (int64_t)blockIdx.x * K;
    const uint64_t* lists = beam_lists(a) + row0 * S * K;

    auto sum_of = [&](int k, uint64_t entry) {
        return j.kind[k] == kLogits ? (double)j.score[k] + (((double)beam_logit((uint32_t)(entry >> 32)) - (double)j.top[k]) - j.logs[k])
               : j.kind[k] == kItself ? (double)j.score[k] : __builtin_nan("");
    };
    auto ranked = [&](int k, uint64_t entry) -> BeamRank {   // {0, 0}: nothing
        const double s = sum_of(k, entry), r = j.weight[k] * s;
        if (s == (double)kBeamNegInf || r == (double)kBeamNegInf) return {0, 0};
        const uint64_t rest = (uint64_t)(kBeamMost - 1 - k) << 52 | (entry >> 32) << 20 | (uint32_t)(entry - (0xffffffffull - (kBeamVocab - 1)));
        return {rank_key(r), rest};
    };

    if (tid < K) j.chosen[tid] = -1;
    if (tid == 0) j.n = j.m = 0, j.last = 1;
    for (int k = w; k < K; k += threads / 64) {
        const int64_t row = row0 + k;
        const float sc = a.scores[row];
        const bool done = a.done ? a.done[row] : false;
        const float weight = a.weight ? a.weight[row] : 1.f;
        const float2* st = beam_stats(a, plan) + row * S;
        // (of a row without continuations by its logits, whatever lies there)
        float2 x[kParts];
        uint64_t h[kParts], best = 0;
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
            const int c = lane + 64 * i;
            x[i] = c < S ? st[c] : make_float2(kBeamNegInf, 0.f);
            h[i] = c < S ? lists[((int64_t)k * S + c) * K] : 0;
        }
        float m = kBeamNegInf;
        bool nan = false;
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
            if (lane + 64 * i < S) j.stage[k * S + lane + 64 * i] = h[i];
            best = h[i] > best ? h[i] : best;
            m = fmaxf(m, x[i].x), nan |= x[i].x != x[i].x;
        }
        m = wave_max(m);
        double z = 0.0;   // (an exponential in 32 bits is off by as much as those that the chunk's sum is of)
#pragma unroll
        for (int i = 0; i < kParts; ++i)
            if (x[i].x != kBeamNegInf) z += (double)(x[i].y * exp2_fast((x[i].x - m) * kLog2e));
        z = wave_sum(z);
        best = wave_max64(best);
        const bool fair = weight > 0.f && weight < __builtin_huge_valf();
        const int what = sc == kBeamNegInf ? kNone : sc != sc || !fair ? kNaN : done ? kItself : __ballot(nan) ? kNaN : kLogits;
        if (lane == 0) {
            j.kind[k] = what, j.top[k] = m, j.score[k] = sc, j.weight[k] = (double)weight, j.logs[k] = log(z);
            j.best[k] = what == kNone || (what == kLogits && best == 0) ? 0 : ranked(k, what == kLogits ? best : kSelf).rank;
        }
    }
    __syncthreads();

    uint64_t least = ~0ull;
#pragma unroll 4
    for (int k = 0; k < K; ++k) least = min(least, j.best[k]);
    for (int i = tid; i < K * S; i += threads) {
        const int k = i / S, what = j.kind[k];
        const uint64_t e = what == kLogits ? j.stage[i] : what != kNone && i == k * S ? kSelf : 0;
        if (e == 0) continue;
        const BeamRank x = ranked(k, e);
        if (x.rank == 0 || x.rank < least) continue;
        const int at = atomicAdd(&j.n, 1);
        j.head[at] = x;
        j.from[at] = i;
    }
    __syncthreads();
    // a power of two of threads counts, for each of n, how many lie above it
    auto group = [&](int n) {
        int G = 1;
        while (G < 64 && 2 * G * n <= threads) G *= 2;
        return G;
    };
    auto above = [&](const BeamRank* of, int n, const BeamRank& x, int G) {
        int c = 0;
#pragma unroll 4
        for (int o = tid % G; o < n; o += G) c += of[o].above(x);
        for (int off = 1; off < G; off *= 2) c += __shfl_xor(c, off, 64);
        return c;
    };
    // The lists of few heads are all looked at; of many, those of the best K.
    const bool few = j.n * K <= threads / 4;
    if (!few) {
        const int n = j.n, G = group(n);
        for (int i0 = 0; i0 < n; i0 += threads / G) {   // (all of a wave's threads take part in the exchange)
            const int i = i0 + tid / G;
            const BeamRank x = j.head[min(i, n - 1)];
            const int c = above(j.head, n, x, G);
            if (i < n && tid % G == 0 && c < K) {
                j.chosen[c] = j.from[i];
                if (c == K - 1) j.last = x.rank;
            }
        }
        __syncthreads();
    }
    const int* of = few ? j.from : j.chosen;
    const uint64_t bound = few ? max(least, (uint64_t)1) : j.last;
    for (int t = tid; t < (few ? j.n : K) * K; t += threads) {
        const int i = of[t / K], o = t % K;
        if (i < 0) continue;
        const int k = i / S;
        const uint64_t e = j.kind[k] == kLogits ? (o == 0 ? j.stage[i] : lists[(int64_t)i * K + o]) : o == 0 ? kSelf : 0;
        const BeamRank x = e ? ranked(k, e) : BeamRank{0, 0};
        if (x.rank < bound) continue;
        const int at = atomicAdd(&j.m, 1);
        j.cand[at] = x;
        j.entry[at] = e;
        j.row[at] = k;
    }
    __syncthreads();
    const int n = j.m, G = group(n);
    for (int i0 = 0; i0 < n; i0 += threads / G) {
        const int i = i0 + tid / G;
        const BeamRank x = j.cand[min(i, n - 1)];
        const int c = above(j.cand, n, x, G);
        if (i < n && tid % G == 0 && c < K) {
            const int k = j.row[i];
            a.out[row0 + c] = (float)sum_of(k, j.entry[i]);
            a.rows[row0 + c] = (int32_t)(row0 + k);
            a.tokens[row0 + c] = j.kind[k] == kLogits ? (int64_t)(0xffffffffu - (uint32_t)j.entry[i]) : a.fill;
        }
    }
    for (int i = n + tid; i < K; i += threads) a.out[row0 + i] = kBeamNegInf, a.rows[row0 + i] = -1, a.tokens[row0 + i] = a.fill;
}

// Chunks of as many places as 256 threads of eight vectors have, or of two (bf16: one) while that leaves CUs without one.  (Eight:
// rows of 131,072 logits are then whole rounds of workgroups, 256 rows of 131,071 fp32 39.5 us against 41.7 with nine, 32
// sequences of 8 bf16 beams 26.6 / 27.4, 512 beams of 50,304 fp32 32.1 / 32.8, none the slower.)
constexpr int kBeamVectors = 8;

static BeamPlan beam_plan(int32_t B, int32_t K, int64_t V, bool bf16) {
    BeamPlan p{};
    const int64_t vec = bf16 ? 8 : 4, rows = (int64_t)B * K, full = kBeamThreads * kBeamVectors * vec, brief = 2048;
    p.few = rows * ((V + full - 1) / full) <= device_cus() && V <= brief * kBeamChunks;
    const int64_t n = (V + (p.few ? brief : full) - 1) / (p.few ? brief : full);
    p.length = (int32_t)(((V + n - 1) / n + vec - 1) / vec * vec);
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
    const int64_t chunks = (int64_t)a.B * a.K * p.chunks;
    FX_REQUIRE(chunks < (1 << 24) && p.chunks <= kBeamChunks, "beam_select: too many rows");   // a launch has less than 2^32 work items
    const dim3 grid((unsigned)chunks), block(kBeamThreads);
    const hipStream_t st = (hipStream_t)stream;
    if (a.bf16 && p.few) hipLaunchKernelGGL((beam_chunk_kernel<true, 1>), grid, block, 0, st, a, p);
    else if (a.bf16) hipLaunchKernelGGL((beam_chunk_kernel<true, kBeamVectors>), grid, block, 0, st, a, p);
    else if (p.few) hipLaunchKernelGGL((beam_chunk_kernel<false, 2>), grid, block, 0, st, a, p);
    else hipLaunchKernelGGL((beam_chunk_kernel<false, kBeamVectors>), grid, block, 0, st, a, p);
    if (int e = check_launch("beam_select")) return e;
    // a wave a row, and a thread for each continuation of the last lists (K K <= 64 K up to 32 beams: two rows a wave past 16)
    const int threads = 64 * (a.K < 4 ? 4 : a.K < 16 ? a.K : 16);
    hipLaunchKernelGGL(beam_join_kernel, dim3((unsigned)a.B), dim3((unsigned)threads), 0, st, a, p);
    return check_launch("beam_select_join");
}

}  // namespace fx
