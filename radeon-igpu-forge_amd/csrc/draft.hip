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
// read once and written once.  One workgroup a row, which holds the row in registers (up to 65,536 fp32
// or 131,072 bf16 logits; what does not fit is read again, from the caches): the maximum, the selection,
// the sum and the output are passes over registers.  256 rows of 50,304 with top-k 50 take 23 us
// (4.5 TB/s), a single row 13; 768 rows of 131,071 bf16, all kept, 150 us (4.0 TB/s; half rows in
// registers and two workgroups a CU, or none and four, took 160 to 183).
//
// Rows of up to four vectors a thread leave room for two workgroups a CU (64 registers: 2,000 rows of 16,384
// fp32 with top-k 50 58 us against 90 with 66), and one's loads run beside the other's stores.  Longer rows
// are a workgroup's alone, so there it walks over several: a vector's registers take the next row's as
// soon as it is stored.  Rows of 9 to 13 vectors a thread (53,248 fp32) have a kernel of 13: what the one of 16 holds
// beyond the row's end is still walked over (256 rows, top-k 50, of 34,000 fp32 19.1 us / 20.2, of 53,000 25.3 / 25.9, one
// row of 34,000 13.1 / 14.4; kernels of 10, 12 and 14 instead are within 4 % of it on either side).  Against a
// workgroup for each row: 2,000 rows of 24,576 fp32 83 us / 92, 768 of
// 50,176 60 / 71, of 61,440 82 / 89, 768 bf16 rows of 131,071 150 / 160 (300 rows of 122,880 69 / 68);
// below eight vectors it would be the slower, by the registers it takes (2,000 of 16,384 56 / 48).
//
// The selection.  The top_k-th largest of the threads' own maxima is at most the top_k-th largest
// logit, and few logits lie above it (of random ones -1024 ln(1 - k / 1024) for the k-th of 1024 maxima): those
// are listed, and the exact bound found among them.  Both searches are one wave's, halving an interval of
// order-preserving integer keys until the keys at or above its lower end are few enough, or top_k.
// Where fewer threads than top_k hold logits that are not -inf, the list is of all such logits (a row with 40 of 50,304 left,
// top-k 50, 18 us; with 60 left 13).  Where it is too small for the logits above the first bound (a sorted row, a thousand equals) the
// bound is found a bit at a time over the registers.  A top_k above 3/8 of the threads, whose list
// would near its 1024 places, goes to another kernel that finds the bound eleven bits at a time, three
// passes over memory that count the keys of what is settled of it: 256 rows, top-k 384 30 us against 52,
// top-k 512 105 (most lists full) against 52.

constexpr int kProbThreads = 1024, kProbWaves = kProbThreads / 64;
constexpr int kProbList = kProbThreads;   // logits of the list
constexpr int kProbTop = kProbThreads * 3 / 8;   // the largest top_k of the list
constexpr int kProbBins = 2048;
constexpr int kProbStream = 8;   // vectors a thread from which on a workgroup walks over rows
constexpr float kDraftNegInf = -__builtin_huge_valf();

// a logit's bits in an order that unsigned comparison keeps, both zeros alike, and the logit of such a key
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }

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

// A wave's search among n keys in LDS (n <= 64 R): a bound with at least `want` keys at or above it, and at most
// `most`, or, where equals prevent that, the want-th largest key itself (the largest bound with `want`).
template <int R>
__device__ __forceinline__ uint32_t wave_bound(const uint32_t* keys, int n, int want, int most, int lane) {
    uint32_t k[R], lo = 0xffffffffu, hi = 0u;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int j = i * 64 + lane;
        k[i] = j < n ? keys[j] : 0u;
        if (j < n) lo = min(lo, k[i]), hi = max(hi, k[i]);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        lo = min(lo, (uint32_t)__shfl_xor((int)lo, off, 64));
        hi = max(hi, (uint32_t)__shfl_xor((int)hi, off, 64));
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    // all keys are at or above lo; keys above hi: none.  (A slot past n holds 0, the least key, below any mid.)
    int have = n;
    while (lo < hi && have > most) {
        const uint32_t mid = lo + (hi - lo) / 2 + 1;
        int c = 0;
#pragma unroll
        for (int i = 0; i < R; ++i) c += __popcll(__ballot(k[i] >= mid));
        if (c >= want) lo = mid, have = c;
        else hi = mid - 1;
    }
    return lo;
}

// f(logit, place) for this thread's of a row of V from flat index i0 of a 16-byte aligned tensor: 16-byte loads, the ragged
// ends by single ones
template <bool BF, typename Fn>
__device__ __forceinline__ void each_logit(const void* base, int64_t i0, int64_t V, Fn f) {
    constexpr int NP = BF ? 8 : 4;
    const int64_t head = min(V, (NP - i0 % NP) % NP), body = (V - head) / NP;
    auto one = [&](int64_t v) { return BF ? bf16_to_f32(static_cast<const uint16_t*>(base)[i0 + v]) : static_cast<const float*>(base)[i0 + v]; };
#pragma unroll 2
    for (int64_t i = threadIdx.x; i < body; i += kProbThreads) {
        const uint4 u = ld16(static_cast<const char*>(base) + (i0 + head + i * NP) * (BF ? 2 : 4));
        float x[NP];
        if constexpr (BF) unpack8(u, x);
        else x[0] = __uint_as_float(u.x), x[1] = __uint_as_float(u.y), x[2] = __uint_as_float(u.z), x[3] = __uint_as_float(u.w);
#pragma unroll
        for (int e = 0; e < NP; ++e) f(x[e], head + i * NP + e);
    }
    if ((int64_t)threadIdx.x < head) f(one(threadIdx.x), (int64_t)threadIdx.x);
    const int64_t v = head + body * NP + threadIdx.x;
    if (v < V) f(one(v), v);
}

// The want-th largest key of a row, 11, 11 and 10 bits at a time: the bins of the keys that share the bits above.
template <bool BF>
__device__ __forceinline__ uint32_t radix_bound(const void* logits, int64_t i0, int64_t V, int want, uint32_t* hist) {
    __shared__ uint32_t digit;
    __shared__ int above;
    const int lane = threadIdx.x & 63;
    uint32_t key = 0, settled = 0;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int bits = pass < 2 ? 11 : 10, shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        __syncthreads();
        for (int i = threadIdx.x; i < kProbBins; i += kProbThreads) hist[i] = 0;
        __syncthreads();
        each_logit<BF>(logits, i0, V, [&](float x, int64_t) {
            const uint32_t k = order_key(x);
            if ((k & settled) == key) atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1)], 1u);
        });
        __syncthreads();
        if (threadIdx.x < 64) {   // bins from the top: 32 a lane (half of them empty in the last pass)
            constexpr int PL = kProbBins / 64;
            const int top = kProbBins - 1 - lane * PL;
            int sum = 0;
            for (int i = 0; i < PL; ++i) sum += (int)hist[top - i];
            int up = sum;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const int o = __shfl_up(up, off, 64);
                if (lane >= off) up += o;
            }
            const uint64_t past = __ballot(up >= want);
            if (lane == __ffsll((unsigned long long)past) - 1) {   // the want-th lies in this lane's bins
                int run = up - sum, i = 0;
                for (; i < PL - 1 && run + (int)hist[top - i] < want; ++i) run += (int)hist[top - i];
                digit = (uint32_t)(top - i);
                above = run;
            }
        }
        __syncthreads();
        key |= digit << shift;
        settled |= ((1u << bits) - 1) << shift;
        want -= above;
    }
    return key;
}

// Where V logits from flat index i0 of a 16-byte aligned tensor lie: whole vectors, and the row's ragged ends (fewer than
// two vectors' values, one a thread)
template <bool BF>
struct LogitPlace {
    static constexpr int NP = BF ? 8 : 4;
    const char* base;  // the first whole vector
    int64_t head;
    int edge_at;       // -1: none
    int body;
    int tid;           // the thread's index

    __device__ __forceinline__ void place(const void* logits, int64_t i0, int64_t V, int t) {
        tid = t;
        head = min(V, (32 - i0 % 32) % 32);   // the output's 128-byte lines, each a wave's own
        body = (int)((V - head) / NP);
        base = static_cast<const char*>(logits) + (i0 + head) * (BF ? 2 : 4);
        const int tail = (int)head + body * NP;
        edge_at = t < head ? t : t - head < V - tail ? tail + t - (int)head : -1;
    }
    // this thread's i-th vector; what lies behind the row's end is -inf: neither kept nor summed
    __device__ __forceinline__ uint4 load(int i) const {
        const uint32_t ninf = BF ? 0xff80ff80u : 0xff800000u;
        return tid < body - i * kProbThreads ? ld16(base + (uint32_t)(tid * 16 + i * kProbThreads * 16))
                                                          : make_uint4(ninf, ninf, ninf, ninf);
    }
    __device__ __forceinline__ float load_edge(const void* logits, int64_t i0) const {
        if (edge_at < 0) return kDraftNegInf;
        return BF ? bf16_to_f32(static_cast<const uint16_t*>(logits)[i0 + edge_at]) : static_cast<const float*>(logits)[i0 + edge_at];
    }
};

// A row as the threads of a workgroup hold it: NR 16-byte vectors each; vectors past those are read again at every pass
template <bool BF, int NR>
struct LogitRow : LogitPlace<BF> {
    using LogitPlace<BF>::NP;
    using LogitPlace<BF>::base;
    using LogitPlace<BF>::head;
    using LogitPlace<BF>::edge_at;
    using LogitPlace<BF>::body;
    using LogitPlace<BF>::tid;
    uint4 x[NR];
    float edge;

    __device__ __forceinline__ static void unpack(const uint4& u, float* f) {
        if constexpr (BF) unpack8(u, f);
        else f[0] = __uint_as_float(u.x), f[1] = __uint_as_float(u.y), f[2] = __uint_as_float(u.z), f[3] = __uint_as_float(u.w);
    }
    __device__ __forceinline__ void start(const void* logits, int64_t i0, int64_t V) {
        this->place(logits, i0, V, threadIdx.x);
#pragma unroll
        for (int i = 0; i < NR; ++i) x[i] = this->load(i);
        edge = this->load_edge(logits, i0);
    }
    // f(four values) for every four of the row's vectors.  What a pass makes of
    // a vector must not be kept in registers for the next pass, nor made before its turn: the vectors go
    // through an empty statement that the compiler cannot see through (LOOP: a copy of them does, since a loop
    // would otherwise hold the vectors twice).
    template <bool LOOP, typename Fn>
    __device__ __forceinline__ void each(Fn f) {
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            uint4 u;
            if constexpr (LOOP) {
                asm volatile("v_mov_b32 %0, %4\n\tv_mov_b32 %1, %5\n\tv_mov_b32 %2, %6\n\tv_mov_b32 %3, %7"
                             : "=&v"(u.x), "=&v"(u.y), "=&v"(u.z), "=&v"(u.w)
                             : "v"(x[i].x), "v"(x[i].y), "v"(x[i].z), "v"(x[i].w));
            } else {
                asm volatile("" : "+v"(x[i].x), "+v"(x[i].y), "+v"(x[i].z), "+v"(x[i].w));
                u = x[i];
            }
            float y[NP];
            unpack(u, y);
#pragma unroll
            for (int e = 0; e < NP; e += 4) f(y + e);
            __builtin_amdgcn_sched_barrier(0);
        }
        for (int j = NR * kProbThreads + threadIdx.x; j < body; j += kProbThreads) {
            float y[NP];
            unpack(ld16(base + (int64_t)j * 16), y);
#pragma unroll
            for (int e = 0; e < NP; e += 4) f(y + e);
        }
    }

    // out[place] = f(value) over the row's vectors, four values a store that its neighbours' follow: a bf16 vector's
    // eight would be two stores with gaps between the lanes, so a pair of lanes exchanges halves first.
    // NEXT: a vector's registers take the one of the row at `next` as soon as it is stored, so that loads run behind the
    // stores, and this is that row then (`more`: there is one).
    template <bool NEXT, typename Fn>
    __device__ __forceinline__ void write(float* out, Fn f, bool more, const void* logits, int64_t next, int64_t V) {
        LogitPlace<BF> to = *this;
        if constexpr (NEXT) {
            int t = threadIdx.x;
            asm volatile("" : "+v"(t));   // anew: addresses made of it are not kept in registers from one row for the next
            to.place(logits, next, V, t);
            if (!more) to.body = 0, to.edge_at = -1;
        }
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            asm volatile("" : "+v"(x[i].x), "+v"(x[i].y), "+v"(x[i].z), "+v"(x[i].w));
            put(x[i], i * kProbThreads + tid, out, f);
            if constexpr (NEXT) x[i] = to.load(i);
            __builtin_amdgcn_sched_barrier(0);
        }
        for (int j = NR * kProbThreads + threadIdx.x; (j & ~1) < body; j += kProbThreads)   // pairs of lanes stay together
            put(ld16(base + (int64_t)min(j, body - 1) * 16), j, out, f);
        if (edge_at >= 0) {
            float y[4] = {edge, edge, edge, edge};
            f(y);
            out[edge_at] = y[0];
        }
        if constexpr (NEXT) {
            edge = to.load_edge(logits, next);
            static_cast<LogitPlace<BF>&>(*this) = to;
        }
    }
    template <typename Fn>
    __device__ __forceinline__ void put(const uint4& u, int j, float* out, Fn f) const {
        float y[NP];
        unpack(u, y);
#pragma unroll
        for (int e = 0; e < NP; e += 4) f(y + e);
        if constexpr (!BF) {
            if (j < body) *reinterpret_cast<float4*>(out + head + (int64_t)j * 4) = make_float4(y[0], y[1], y[2], y[3]);
        } else {
            const bool odd = tid & 1;
            const int first = j & ~1;   // the pair's
            auto other = [](float v) {   // lane ^ 1's
                return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), 0xb1, 0xf, 0xf, true));
            };
            float a[4], b[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float low = other(y[e]), high = other(y[4 + e]);
                a[e] = odd ? high : y[e];
                b[e] = odd ? y[4 + e] : low;
            }
            float* p = out + head + (int64_t)first * 8 + (odd ? 4 : 0);
            if (first < body) *reinterpret_cast<float4*>(p) = make_float4(a[0], a[1], a[2], a[3]);
            if (first + 1 < body) *reinterpret_cast<float4*>(p + 8) = make_float4(b[0], b[1], b[2], b[3]);
        }
    }
};

// exp((l - m) / T) as 2^((l - m) f), f = log2(e) / T in two parts: the difference and the product are rounded, once each.
// The first part is below f and the second no less than the least normal number (2^-26 of the least f), so that -inf times
// the second is -inf too, and its power 0.
struct ProbVal {
    float m, hi, lo;
    __device__ __forceinline__ ProbVal(float m, double temperature) : m(m) {
        const double f = 1.4426950408889634 / temperature;
        hi = (float)f;
        if ((double)hi >= f) hi = __uint_as_float(__float_as_uint(hi) - 1);
        lo = fmaxf((float)(f - (double)hi), __FLT_MIN__);
    }
    __device__ __forceinline__ float operator()(float x) const {
        const float d = x - m;
        return exp2_fast(fmaf(d, hi, d * lo));
    }
};

// zeros or NaN for a row that has no probabilities: of -inf alone, or with a NaN or +inf
__device__ __forceinline__ bool no_probs(float m, bool nan, float* out, int64_t V) {
    const bool empty = !nan && m == kDraftNegInf;
    if (!nan && !empty && m != __builtin_huge_valf()) return false;
    const float v = empty ? 0.f : __builtin_nanf("");
    for (int64_t i = threadIdx.x; i < V; i += kProbThreads) out[i] = v;
    return true;
}

// Any top_k: every step a pass over memory (the first from HBM, the others from the caches)
template <bool BF>
__global__ void __launch_bounds__(kProbThreads) probs_passes_kernel(const void* logits, float* probs, int64_t V, double temperature, int top_k) {
    __shared__ float shf[kProbWaves];
    __shared__ uint32_t hist[kProbBins];
    const int64_t i0 = (int64_t)blockIdx.x * V;
    float* out = probs + i0;
    float m = kDraftNegInf;
    bool nan = false;
    each_logit<BF>(logits, i0, V, [&](float x, int64_t) { m = fmaxf(m, x), nan |= x != x; });
    m = block_reduce<JoinMax>(m, shf);
    nan = __syncthreads_or(nan);
    if (no_probs(m, nan, out, V)) return;
    const float least = key_value(radix_bound<BF>(logits, i0, V, top_k, hist));   // logits from here on are kept
    const ProbVal val(m, temperature);
    float s = 0.f;
    each_logit<BF>(logits, i0, V, [&](float x, int64_t) { s += x >= least ? val(x) : 0.f; });
    s = block_reduce<JoinSum>(s, shf);
    const float inv = 1.f / s;
    each_logit<BF>(logits, i0, V, [&](float x, int64_t v) { out[v] = x >= least ? val(x) * inv : 0.f; });
}

// TOP: with top_k (up to kProbTop), else over the whole row
template <bool BF, int NR, bool TOP>
__global__ void __launch_bounds__(kProbThreads, NR < kProbStream ? 8 : 4) probs_kernel(const void* logits, float* probs, int64_t rows, int64_t V, double temperature, int top_k) {
    __shared__ float shf[kProbWaves];
    __shared__ int shi[kProbWaves], listed;
    __shared__ uint32_t keys[TOP ? kProbThreads : 1], bound;   // the threads' maxima, then the list
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    constexpr bool STREAM = NR >= kProbStream;
    LogitRow<BF, NR> row;
    const int64_t step = (int64_t)gridDim.x * V;
    int64_t i0 = (int64_t)blockIdx.x * V;
    row.start(logits, i0, V);
#pragma unroll 1
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x, i0 += step) {
        float* out = probs + i0;
        const bool more = r + gridDim.x < rows;
        float own = row.edge;   // this thread's maximum
        bool nan = row.edge != row.edge;
        row.template each<false>([&](const float* y) {
            own = fmaxf(fmaxf(fmaxf(own, y[0]), fmaxf(y[1], y[2])), y[3]);
            nan |= __builtin_isunordered(y[0], y[1]) || __builtin_isunordered(y[2], y[3]);
            asm volatile("" : "+v"(own));
        });
        if constexpr (TOP) {
            if (threadIdx.x == 0) listed = 0;
            keys[threadIdx.x] = order_key(own);
        }
        float s = 0.f;
        if constexpr (!TOP) {
            // the sum above the thread's own maximum, before the workgroup waits for the slowest of its loads
            const ProbVal val(own == kDraftNegInf ? 0.f : own, temperature);
            s = val(row.edge);
            row.template each<false>([&](const float* y) {
#pragma unroll
                for (int e = 0; e < 4; ++e) s += val(y[e]);
                asm volatile("" : "+v"(s));
            });
        }
        const float m = block_reduce<JoinMax>(own, shf);
        nan = __syncthreads_or(nan);
        // a row of -inf, with NaN or with +inf goes through the same stores (a second place that loads the next row would take
        // registers) and is filled behind them
        const bool none = nan || m == kDraftNegInf || m == __builtin_huge_valf();
        float least = kDraftNegInf;   // logits from here on are kept
        if (TOP && !none) {
            if (w == 0) {
                const uint32_t t = wave_bound<kProbWaves>(keys, kProbThreads, top_k, top_k + top_k / 4 + 8, lane);
                if (lane == 0) bound = t;
            }
            __syncthreads();
            const float t = fmaxf(key_value(bound), -__FLT_MAX__);   // masked logits and what lies behind the row are not listed
            auto list = [&](float x) {
                if (x >= t) {
                    const int at = atomicAdd(&listed, 1);   // in any order: the list is only searched
                    if (at < kProbList) keys[at] = order_key(x);
                }
            };
            row.template each<false>([&](const float* y) {
                if (fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])) >= t) list(y[0]), list(y[1]), list(y[2]), list(y[3]);
            });
            list(row.edge);
            __syncthreads();
            const int n = listed;
            if (n <= top_k) {   // every listed logit: all that are not masked, if they are fewer
                least = t;
            } else if (n <= kProbList) {
                if (w == 0) {
                    const uint32_t t2 = n <= 256 ? wave_bound<4>(keys, n, top_k, top_k, lane) : wave_bound<kProbWaves>(keys, n, top_k, top_k, lane);
                    if (lane == 0) bound = t2;
                }
                __syncthreads();
                least = key_value(bound);
            } else {
                uint32_t key = 0;
                for (int bit = 31; bit >= 0; --bit) {
                    const uint32_t t2 = key | (1u << bit);
                    int c = order_key(row.edge) >= t2;
                    row.template each<true>([&](const float* y) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) c += order_key(y[e]) >= t2;
                        asm volatile("" : "+v"(c));
                    });
                    if (block_reduce<JoinCount>(c, shi) >= top_k) key = t2;
                }
                least = key_value(key);
            }
        }
        const ProbVal val(m, temperature);
        if constexpr (TOP) {
            s = row.edge >= least ? val(row.edge) : 0.f;
            row.template each<false>([&](const float* y) {
                if (!(fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])) >= least)) return;
#pragma unroll
                for (int e = 0; e < 4; ++e) s += y[e] >= least ? val(y[e]) : 0.f;
                asm volatile("" : "+v"(s));
            });
        } else {
            s *= val(own);   // from the thread's maximum to the row's
        }
        s = block_reduce<JoinSum>(s, shf);
        const float inv = 1.f / s;
        row.template write<STREAM>(out, [&](float* y) {
            if (TOP && !(fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])) >= least)) {
                y[0] = y[1] = y[2] = y[3] = 0.f;
                return;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = !TOP || y[e] >= least ? val(y[e]) * inv : 0.f;
        }, more, logits, i0 + step, V);
        if (none) {
            __syncthreads();
            no_probs(m, nan, out, V);
        }
        if (!STREAM) break;
    }
}

template <bool BF>
static void probs_launch(const void* logits, float* probs, int64_t rows, int64_t V, double temperature, int64_t top_k, hipStream_t st) {
    constexpr int NP = BF ? 8 : 4;
    const int64_t vectors = (V / NP + kProbThreads - 1) / kProbThreads;   // a thread's, of a row
    const bool top = top_k > 0 && top_k < V;
    const int64_t cus = device_cus();
    const dim3 grid((unsigned)rows), block(kProbThreads), resident((unsigned)(rows < cus ? rows : cus));
    if (top && top_k > kProbTop) {
        hipLaunchKernelGGL((probs_passes_kernel<BF>), grid, block, 0, st, logits, probs, V, temperature, (int)top_k);
        return;
    }
#define FX_PROBS(NR)                                                                                               \
    const dim3 g = NR >= kProbStream ? resident : grid;                                                            \
    if (top) hipLaunchKernelGGL((probs_kernel<BF, NR, true>), g, block, 0, st, logits, probs, rows, V, temperature, (int)top_k); \
    else hipLaunchKernelGGL((probs_kernel<BF, NR, false>), g, block, 0, st, logits, probs, rows, V, temperature, 0)
    if (vectors <= 1) { FX_PROBS(1); }
    else if (vectors <= 4) { FX_PROBS(4); }
    else if (vectors <= 8) { FX_PROBS(8); }
    else if (vectors <= 13) { FX_PROBS(13); }
    else { FX_PROBS(16); }
#undef FX_PROBS
}

int sampling_probs(const void* logits, bool bf16, float* probs, int64_t rows, int64_t V, double temperature, int64_t top_k, void* stream) {
    FX_REQUIRE(rows >= 0 && rows < 0x7fffffffLL && V >= 1 && V < 0x7fffffffLL, "sampling_probs: bad shape rows=%lld V=%lld", (long long)rows, (long long)V);
    FX_REQUIRE(temperature >= 1e-30 && temperature <= 1e30, "sampling_probs: temperature %g must lie in [1e-30, 1e30]", temperature);
    if (rows == 0) return 0;
    FX_REQUIRE(logits && probs && (((uintptr_t)logits | (uintptr_t)probs) & 15) == 0, "sampling_probs: logits and probs must be 16-byte aligned");
    // a launch has less than 2^32 work items; a multiple of 8 rows keeps the alignment
    constexpr int64_t most = (1ll << 31) / kProbThreads;
    for (int64_t r = 0; r < rows; r += most) {
        const int64_t n = rows - r < most ? rows - r : most;
        const char* x = static_cast<const char*>(logits) + r * V * (bf16 ? 2 : 4);
        if (bf16) probs_launch<true>(x, probs + r * V, n, V, temperature, top_k, (hipStream_t)stream);
        else probs_launch<false>(x, probs + r * V, n, V, temperature, top_k, (hipStream_t)stream);
    }
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

//
// One workgroup a sequence, every step of the walk in it: bound by the longest walk's passes, one behind the other on one
// CU.  A pass is as much 64-bit arithmetic as memory: VALU issues in 55 % of the SIMDs' cycles while they have waves, and the
// waves wait 56 % of their time for loads and barriers (a CU takes about 80 GB/s).  Rows are read in 16-byte vectors,
// several in flight and the next ones behind them.  64 trees of 24 nodes over 131,072 ids take 59 to 74 us by the seed (two passes a sequence on
// average, five or so in the longest walk; with the draft's row read at a leaf too 74 to 78), a chain of
// five over 50,304 12.6.  Launches that share a pass over
// several workgroups a sequence, and walk again from the start, took longer (84 us for four such launches, 101
// for six, against 70 to 80 then).
// The draw: the row's sum is taken in 16 regions, a wave each, then the region that the running sum passes
// the drawn point in by itself, down to what one wave scans.

constexpr int kVerNodes = 64;
constexpr int64_t kVerMaxV = 1 << 20;
constexpr int kVerScan = 512;   // values that a wave scans
constexpr int kVerVecs = 4;     // 16-byte vectors of each row that a thread has in flight, twice

// what rejections leave of a row: p, or max(p - c q, 0), or p without the dropped tokens
struct Left {
    const float *p, *q;   // the rows; q null: no draft rows
    const int64_t* tok;   // the nodes' tokens (LDS)
    uint64_t drop;        // nodes whose tokens are out (no draft rows)
    double c;             // zero while nothing is refused: the draft row is not read then (a leaf's may hold anything)
    int V;
    int off;              // values of the row's first 16-byte vector that lie before the row: vector i has values 4 i - off ..

    __device__ __forceinline__ void row(const float* probs, const float* draft, int64_t at) {
        p = probs + at;
        q = draft ? draft + at : nullptr;
        drop = 0;
        c = 0.0;
        off = (int)(at & 3);
    }
    __device__ __forceinline__ int vectors() const { return (V + off + 3) / 4; }
    __device__ __forceinline__ double at(int v) const {
        if (v < 0 || v >= V) return 0.0;
        if (c != 0.0) return fmax(fma(-c, (double)q[v], (double)p[v]), 0.0);
        for (uint64_t d = drop; d; d &= d - 1)
            if (tok[__ffsll((unsigned long long)d) - 1] == v) return 0.0;
        return (double)fmaxf(p[v], 0.f);
    }
    template <bool Q>
    __device__ __forceinline__ double four(const float4& x, const float4& y, int i) const {
        if constexpr (Q) {
            return (fmax(fma(-c, (double)y.x, (double)x.x), 0.0) + fmax(fma(-c, (double)y.y, (double)x.y), 0.0)) +
                   (fmax(fma(-c, (double)y.z, (double)x.z), 0.0) + fmax(fma(-c, (double)y.w, (double)x.w), 0.0));
        } else {
            float z[4] = {fmaxf(x.x, 0.f), fmaxf(x.y, 0.f), fmaxf(x.z, 0.f), fmaxf(x.w, 0.f)};
            for (uint64_t d = drop; d; d &= d - 1) {
                const int64_t e = tok[__ffsll((unsigned long long)d) - 1] - (4 * (int64_t)i - off);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (e == k) z[k] = 0.f;
            }
            return ((double)z[0] + (double)z[1]) + ((double)z[2] + (double)z[3]);
        }
    }
    // thread `first` of `stride`'s share of the sum over vectors [lo, hi)
    template <bool Q>
    __device__ __forceinline__ double share(int lo, int hi, int first, int stride) const {
        const float4* p4 = reinterpret_cast<const float4*>(p - off);
        const float4* q4 = reinterpret_cast<const float4*>((Q ? q : p) - off);
        double s = 0.0;
        // the row's ragged vectors, value by value
        const int whole = (V + off) / 4;   // vectors from here on end behind the row
        if (first == 0) {
            if (lo == 0 && off && hi > 0)
                for (int e = 0; e < 4; ++e) s += at(e - off);
            if (hi > whole && whole >= lo && (whole > 0 || !off))
                for (int e = 0; e < 4; ++e) s += at(4 * whole - off + e);
        }
        if (lo == 0 && off) lo = 1;
        hi = min(hi, whole);
        float4 x[kVerVecs], y[kVerVecs];
        const int step = kVerVecs * stride, turns = hi > lo ? (hi - lo) / step : 0;   // of whole steps, the same for every thread
        int i = lo + first;
        if (turns > 0) {
#pragma unroll
            for (int u = 0; u < kVerVecs; ++u) {
                x[u] = p4[i + u * stride];
                if constexpr (Q) y[u] = q4[i + u * stride];
            }
            for (int t = 1; t < turns; ++t, i += step) {
                float4 nx[kVerVecs], ny[kVerVecs];
#pragma unroll
                for (int u = 0; u < kVerVecs; ++u) {
                    nx[u] = p4[i + step + u * stride];
                    if constexpr (Q) ny[u] = q4[i + step + u * stride];
                }
#pragma unroll
                for (int u = 0; u < kVerVecs; ++u) {
                    s += four<Q>(x[u], y[u], i + u * stride);
                    x[u] = nx[u];
                    if constexpr (Q) y[u] = ny[u];
                }
            }
#pragma unroll
            for (int u = 0; u < kVerVecs; ++u) s += four<Q>(x[u], y[u], i + u * stride);
            i += step;
        }
#pragma unroll
        for (int u = 0; u < kVerVecs; ++u) {
            if (i + u * stride >= hi) continue;
            x[u] = p4[i + u * stride];
            if constexpr (Q) y[u] = q4[i + u * stride];
        }
#pragma unroll
        for (int u = 0; u < kVerVecs; ++u)
            if (i + u * stride < hi) s += four<Q>(x[u], y[u], i + u * stride);
        return s;
    }
    __device__ __forceinline__ double sum(int lo, int hi, int first, int stride) const {
        return c != 0.0 ? share<true>(lo, hi, first, stride) : share<false>(lo, hi, first, stride);
    }
};

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

__global__ void __launch_bounds__(kProbThreads) verify_kernel(const float* probs, const float* draft, const int64_t* tokens, const int32_t* parents,
                                                              const float* uniform, int64_t* out, int32_t* path, int32_t* counts, int32_t N, int64_t V) {
    __shared__ int64_t tok[kVerNodes];
    __shared__ int par[kVerNodes], spath[kVerNodes];
    __shared__ float un[kVerNodes], pt[kVerNodes], qt[kVerNodes];
    __shared__ double shd[kProbWaves], reg[2][kProbWaves];
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

    Left left;
    left.tok = tok;
    left.V = (int)V;
    left.row(probs, draft, b * N * V);
    int cur = 0, n = 0;
    double S = 1.0;
    bool stale = false;   // c has moved since S was formed
    if (threadIdx.x == 0) spath[0] = 0;
    for (int i = 1; i < N; ++i) {
        if (par[i] != cur) continue;
        double x = (double)pt[i];
        if (Q) {
            if (stale) S = block_reduce<JoinSumD>(left.sum(0, left.vectors(), threadIdx.x, kProbThreads), shd), stale = false;
            x = fmax(x - left.c * (double)qt[i], 0.0);
        } else {
            for (uint64_t d = left.drop; d; d &= d - 1)
                if (tok[__ffsll((unsigned long long)d) - 1] == tok[i]) x = 0.0;
        }
        if ((double)un[i] * S * (double)qt[i] < x) {
            cur = i;
            left.row(probs, draft, (b * N + i) * V);
            S = 1.0, stale = false;
            if (threadIdx.x == 0) spath[n + 1] = i;
            ++n;
        } else if (Q) {
            left.c += S;
            stale = true;
        } else {
            S -= x;
            left.drop |= 1ull << i;
        }
    }

    // the last token, from what is left; from the row itself where nothing is
    int lo = 0, hi = left.vectors(), got = -1;
    double at = 0.0, base = 0.0;   // the sum before vector lo
    bool any = true;
    for (int level = 0, round = 0;;) {
        if (level > 0 && (hi - lo) * 4 <= kVerScan) break;
        const int part = (hi - lo + kProbWaves - 1) / kProbWaves, l = lo + part * w;
        const double s = wave_sum_d(left.sum(min(l, hi), min(l + part, hi), lane, 64));
        if (lane == 0) reg[level & 1][w] = s;   // two, in turn: one barrier a level
        __syncthreads();
        double run = base, from = base, some_from = base;
        int pick = -1, some = -1;
        if (level == 0) {
            double W = 0.0;
            for (int x = 0; x < kProbWaves; ++x) W += reg[0][x];
            if (!(W > 0.0) && round == 0) {
                left.c = 0.0, left.drop = 0, round = 1;
                __syncthreads();
                continue;
            }
            if (!(W > 0.0) || W == __builtin_huge_val()) {
                any = false;
                break;
            }
            at = (double)un[0] * W;
        }
        for (int x = 0; x < kProbWaves; ++x) {
            const double z = reg[level & 1][x];
            if (z > 0.0) {
                some = x, some_from = run;
                if (pick < 0 && run + z > at) pick = x, from = run;
            }
            run += z;
        }
        if (pick < 0) pick = some, from = some_from;   // by rounding none may pass: the last with weight
        if (pick < 0) {   // a region's sum that its parts do not have: not reached
            any = false;
            break;
        }
        const int l2 = lo + part * pick;
        hi = min(l2 + part, hi);
        lo = l2;
        base = from;
        ++level;
    }
    if (any && w == 0) {
        constexpr int E = kVerScan / 64;
        double x[E], sum = 0.0;
        const int v0 = 4 * lo - left.off + lane * E, v1 = min(left.V, 4 * hi - left.off);
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = v0 + e < v1 ? left.at(v0 + e) : 0.0, sum += x[e];
        double up = sum;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const double o = __shfl_up(up, off, 64);
            if (lane >= off) up += o;
        }
        double run = base + (up - sum);
        int hit = -1, has = -1;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            run += x[e];
            if (x[e] > 0.0) {
                has = e;
                if (hit < 0 && run > at) hit = e;
            }
        }
        const uint64_t hits = __ballot(hit >= 0), some = __ballot(has >= 0);
        if (hits) {
            const int l = __ffsll((unsigned long long)hits) - 1;
            got = 4 * lo - left.off + l * E + __shfl(hit, l, 64);
        } else if (some) {
            const int l = 63 - __clzll((long long)some);
            got = 4 * lo - left.off + l * E + __shfl(has, l, 64);
        }
    }
    if (threadIdx.x == 0) last = got;
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
    FX_REQUIRE(B <= 0xffffffffu / kProbThreads, "verify_draft: grid too large (B=%d)", B);
    if (B == 0) return 0;
    FX_REQUIRE(probs && tokens && parents && uniform && out && path && counts, "verify_draft: null pointer");
    FX_REQUIRE((((uintptr_t)probs | (uintptr_t)draft) & 15) == 0, "verify_draft: probs and draft_probs must be 16-byte aligned");
    hipLaunchKernelGGL(verify_kernel, dim3((unsigned)B), dim3(kProbThreads), 0, (hipStream_t)stream, probs, draft, tokens, parents, uniform, out,
                       path, counts, N, V);
    return check_launch("verify_draft");
}

// ---- accepted rows together --------------------------------------------------------------
//
// Bound by the moved rows' bytes, read and written once, from pages all over the caches: 60 tensors of 48
// sequences, 112 MB, take 30 us cold (3.7 TB/s; 16 rows in flight 39, two to eight the same), a 12-layer cache's
// 1.8 MB 4.  A thread owns 16 bytes of a (tensor, sequence)'s row and moves them for every d, eight rows in
// flight: the path ascends, so a row that is written (ctx + d <= ctx + path[d]) is never one that is still to be
// read.

constexpr int kCompactRows = 8;

__global__ void __launch_bounds__(256) compact_kernel(CompactArgs a) {
    const int y = blockIdx.y, b = y % a.B, ten = y / a.B;
    const int ctx = a.ctx[b];
    int n = a.counts[b];
    n = n < 0 ? 0 : (n > a.N ? a.N : n);
    if (a.ctx_out && ten == 0 && blockIdx.x == 0 && threadIdx.x == 0) a.ctx_out[b] = ctx + n;
    const int i = blockIdx.x * blockDim.x + threadIdx.x, cpr = a.D / 8;
    if (i >= a.H * cpr || ctx < 0) return;
    const int h = i / cpr, col = (i - h * cpr) * 8;
    const int64_t st = a.st[ten];
    uint16_t* p = a.at[ten] + b * a.sb[ten] + h * a.sh[ten] + ctx * st + col;
    const int32_t* path = a.path + (int64_t)b * a.N;
    const int room = a.T - ctx;   // rows of the cache behind the context
    for (int d0 = 0; d0 < n; d0 += kCompactRows) {
        uint4 x[kCompactRows];
        bool move[kCompactRows];
#pragma unroll
        for (int u = 0; u < kCompactRows; ++u) {
            const int s = path[min(d0 + u, n - 1)];
            move[u] = d0 + u < n && s > d0 + u && s < room;   // else in its place already, or no row of the cache
            if (move[u]) x[u] = ld16(p + s * st);
        }
#pragma unroll
        for (int u = 0; u < kCompactRows; ++u)
            if (move[u]) st16(p + (d0 + u) * st, x[u]);
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
    const unsigned chunks = (unsigned)(a.H * (a.D / 8)), threads = chunks < 256 ? (chunks + 63) / 64 * 64 : 256;
    hipLaunchKernelGGL(compact_kernel, dim3((chunks + threads - 1) / threads, (unsigned)(a.count * a.B)), dim3(threads), 0, (hipStream_t)stream, a);
    return check_launch("compact_cache");
}

}  // namespace fx
