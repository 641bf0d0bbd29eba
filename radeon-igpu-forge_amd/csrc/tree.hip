// Attention of a tree of drafted tokens over a KV cache, for gfx950.
//
// Sequence b has ctx[b] keys in its cache; its tree's node j (a drafted token; node 0 the last
// token that is not drafted) has cache row ctx[b] + j.  A query of node i sees every row below
// ctx[b] and the rows of the nodes in its bit set tree[b, i]:
//
//   o[b, i, h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q[b, i, h] . k_j),
//
// over those rows j, in one pass with a running maximum and sum.  A node whose own bit is clear
// is padding: its output is zero and its row is nobody's key.  Query heads share key heads
// (H a multiple of Hkv): the N H / Hkv queries of one key head are the rows of one product.
//
// HBM-bound: every cached key and value is read once (4 D bytes a row and key head).  So the
// rows of a key head stay in one workgroup, 32 to a wave's MFMA tile, and the keys are split:
// over the workgroup's waves, and over workgroups ("units") for as many as fill the CUs at once.
// A unit's length comes from the sequences' own lengths on the device, so a long sequence among
// short ones gets more units; a second kernel joins the units of a row by their maxima and sums.
// Whether keys are split at all goes by the cache's size, which the host knows (the launch shape
// below): short contexts in a large cache pay for the second launch.
//
// 32 nodes of 4 query heads a key head, 4 sequences of 16,001 to 32,768 keys, 8 key heads of 128: 403 MB in 98 us (95 of
// them this kernel, 4.3 TB/s); one token over up to 65,011 keys of 16 heads of 64: 430 MB in 95 us (89, 4.8 TB/s).  Two
// tiles a step, or a second one in flight behind it, change neither: memory bounds the second.  The first's waves also wait
// for one another: MFMA is busy in 32 % of the SIMDs' cycles, VALU in 37 %, LDS in 26 %, and half again as many MFMA would
// add 15 us.  Short contexts are bounded by their chain of round trips (context, keys, sums): 225 keys of 12 heads take 7 us.
#include <math.h>

#include "fx_internal.h"
#include "fx_mfma.h"

namespace fx {

constexpr int kTreeWaves = 8;
constexpr int kTreeThreads = 64 * kTreeWaves;
constexpr int kTreeTile = 32;    // keys of a wave's step, rows of its queries
constexpr float kTreeNegInf = -__builtin_huge_valf();
constexpr float kTreeLazy = 8.f;   // the running maximum moves only past this (log2 units): p stays <= 2^8

// what a kernel needs besides the arguments: units a launch aims at (0: keys are not split), the
// fewest tiles of a unit, query row groups of a key head
struct TreePlan {
    int32_t units, least, groups, wq, grid;
};

// keys of a sequence with its context `c` (as the caller gave it): its tree's rows included
__device__ __forceinline__ int tree_len(const TreeArgs& a, int c) {
    const int64_t e = (int64_t)(c < 0 ? 0 : c) + a.first + a.N;
    return (int)(e < a.Tmax ? e : a.Tmax);
}
__device__ __forceinline__ uint32_t tree_tiles(const TreeArgs& a, int c) { return (uint32_t)((tree_len(a, c) + kTreeTile - 1) / kTreeTile); }

// The units of a launch, found by every wave by itself, 64 sequences at a time: `tiles` of a unit (as many as let
// all sequences' fit the launch's units, in whole steps of the workgroup's `wk` streams).  `mine`: the
// context of sequence `lane`, loaded once.
struct TreeUnits {
    uint32_t tiles;
    int mine;
    __device__ __forceinline__ void init(const TreeArgs& a, const TreePlan& p, uint32_t wk, int lane) {
        mine = lane < a.B ? a.ctx[lane] : 0;
        uint32_t sum = lane < a.B ? tree_tiles(a, mine) : 0u;
        for (int b = lane + 64; b < a.B; b += 64) sum += tree_tiles(a, a.ctx[b]);
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
        sum *= (uint32_t)(p.groups * a.Hkv);
        const uint32_t t = max((sum + p.units - 1) / (uint32_t)p.units, (uint32_t)p.least);
        tiles = (t + wk - 1) / wk * wk;
    }
    __device__ __forceinline__ uint32_t count(const TreeArgs& a, int c) const { return max(1u, (tree_tiles(a, c) + tiles - 1) / tiles); }
    // The sequence with unit u (counted a sequence at a time, in units of one key head and row group), its first
    // unit, their number and its context; false past the last sequence.
    __device__ __forceinline__ bool find(const TreeArgs& a, uint32_t u, int lane, int& b, uint32_t& first, uint32_t& n, int& c) const {
        uint32_t before = 0;
        for (int b0 = 0; b0 < a.B; b0 += 64) {
            const bool in = b0 + lane < a.B;
            const int x = b0 == 0 ? mine : in ? a.ctx[b0 + lane] : 0;
            const uint32_t k = in ? count(a, x) : 0u;
            uint32_t up = k;   // inclusive scan
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const uint32_t o = __shfl_up(up, off, 64);
                if (lane >= off) up += o;
            }
            const uint64_t past = __ballot(before + up > u);
            if (past) {
                const int l = __ffsll((unsigned long long)past) - 1;
                b = __builtin_amdgcn_readfirstlane(b0 + l);
                n = (uint32_t)__builtin_amdgcn_readlane((int)k, l);
                first = before + (uint32_t)__builtin_amdgcn_readlane((int)up, l) - n;
                c = __builtin_amdgcn_readlane(x, l);
                return true;
            }
            before += (uint32_t)__builtin_amdgcn_readlane((int)up, 63);
        }
        return false;
    }
};

// where the join finds a sequence's units: (first, count), behind the units' partials
__device__ __forceinline__ uint2* tree_places(const TreeArgs& a, const TreePlan& p) {
    return reinterpret_cast<uint2*>(a.work + (int64_t)p.grid * 32 * p.wq * (a.D + 2));
}

// bits of the tree's nodes that are keys: drafted before this call (below `first`), or queries of it
// that are no padding, and inside the cache
// (`word`: the bit set of query `lane`)
__device__ __forceinline__ uint64_t tree_live(const TreeArgs& a, uint64_t word, int ctx, int lane) {
    uint64_t live = (uint64_t)__ballot(lane < a.N && ((word >> ((a.first + lane) & 63)) & 1));
    live = a.first ? (live << a.first) | ((1ull << a.first) - 1) : live;
    const int room = a.Tmax - ctx;
    return room >= 64 ? live : live & ((1ull << (room > 0 ? room : 0)) - 1);
}

__device__ __forceinline__ bool bf16_not_finite(uint32_t h) { return (h & 0x7f80u) == 0x7f80u; }

// A wave's LDS operations are done in the order of its instructions; this keeps the compiler from moving
// them past each other where lanes read what other lanes wrote.
__device__ __forceinline__ void tree_wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A kernel argument's value in registers: a select between two arguments is otherwise one between their
// addresses, with a load behind it in the loop
__device__ __forceinline__ int64_t pinned(int64_t x) {
    asm volatile("" : "+s"(x));
    return x;
}

// Rows of one kind (keys or values) of a key head, as this lane loads them: cached ones, and the queries' own
struct TreeRows {
    const uint16_t *cached, *fresh;
    int64_t st, stn;
    // row j, clamped to the sequence's last
    __device__ __forceinline__ const uint16_t* at(int j, int end, int newrow) const {
        j = min(j, end - 1);
        const bool nw = j >= newrow;
        return (nw ? fresh : cached) + (j - (nw ? newrow : 0)) * (nw ? stn : st);
    }
};

// Workgroup: WQ groups of 32 query rows x WK = 8 / WQ streams of keys; wave (wq, wk) takes the unit's
// tiles wk, wk + WK, ... of 32 keys.  Per tile S^T = K Q^T (a lane holds 16 of the 32 keys of one
// query), the softmax, and O^T += V^T P^T with V read transposed (fx_mfma.h has the layouts).  Keys and
// values go through LDS in whole rows (16 lanes a 256-byte row: an operand's own pattern, 32 bytes of
// 32 rows, took the address unit 4 times as long and bound the kernel); the next tile is in flight
// in registers meanwhile.  One row group: each wave has a tile of its own and no barrier.  More: the WQ waves
// of a stream load a tile together (each loading it for itself kept the address unit 90% busy),
// into one of two buffers, with a barrier a tile.  The WK streams of a row join through LDS.
template <int D, int WQ>
__global__ void __launch_bounds__(kTreeThreads) tree_attn_kernel(TreeArgs a, TreePlan plan) {
    constexpr int WK = kTreeWaves / WQ;
    constexpr int LPR = D / 8;        // lanes of a row in 16-byte loads
    constexpr int RPI = 64 / LPR;     // rows of a wave-wide load
    constexpr int NV = kTreeTile / RPI;
    constexpr int PW = 2 * NV / WQ;   // loads of a wave: of one row group keys, then values; else of one kind
    constexpr int KS = D / 16;        // steps of the score product
    constexpr int DT = D / 32;
    constexpr int KLD = D + 8;        // LDS row of K: 16 rows of an operand read cover all banks
    constexpr int VLD = D + 32;       // and of V: 4 rows of a transposed read fall in distinct banks
    constexpr int OLD = D + 4;        // LDS row of a wave's fp32 output
    constexpr int kTile = kTreeTile * (KLD + VLD);   // elements
    constexpr int kBufs = WQ == 1 ? 1 : 2;
    constexpr int kTBytes = kBufs * WK * kTile * 2;
    constexpr int kOBytes = kTreeWaves * kTreeTile * OLD * 4;
    static_assert(PW >= 1 && (WQ == 1 || PW * (WQ / 2) == NV), "a tile's loads over its waves");
    __shared__ __attribute__((aligned(16))) unsigned char lds[kTBytes > kOBytes ? kTBytes : kOBytes];
    __shared__ float2 ml[kTreeWaves][kTreeTile];
    __shared__ int odd[kBufs][kTreeWaves];   // the wave loaded an infinity or a NaN

    const int lane = threadIdx.x & 63, ln = lane & 31, g = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wq = w % WQ, wk = w / WQ;
    const int G = a.H / a.Hkv, heads = plan.groups * a.Hkv;

    // the unit: sequence, key head, row group, tiles [t0, t1)
    int b, hr, ctx;
    uint32_t count = 1, t0 = 0, t1 = 0xffffffffu;
    if (plan.units == 0) {
        b = blockIdx.x / heads;
        hr = blockIdx.x - b * heads;
        ctx = a.ctx[b];
    } else {
        TreeUnits units;
        units.init(a, plan, WK, lane);
        const uint32_t u = blockIdx.x / heads;
        hr = blockIdx.x - u * heads;
        uint32_t first;
        if (!units.find(a, u, lane, b, first, count, ctx)) return;
        if (u == first && hr == 0 && threadIdx.x == 0) tree_places(a, plan)[b] = make_uint2(first, count);
        t0 = __builtin_amdgcn_readfirstlane((u - first) * units.tiles);
        t1 = __builtin_amdgcn_readfirstlane(t0 + units.tiles);
    }
    const int h = hr % a.Hkv, rg = hr / a.Hkv;

    // this lane's query row: node and head; and the tree's word of query `lane`
    const int rows = a.N * G;
    const int r = (rg * WQ + wq) * kTreeTile + ln;
    const int node = r < rows ? r / G : 0;
    uint64_t bits = (uint64_t)a.tree[b * a.treeb + node * a.treen];
    const uint64_t word = (uint64_t)a.tree[b * a.treeb + min(lane, a.N - 1) * a.treen];
    bf16x8 qf[KS];
    {
        const uint16_t* qp = a.q + b * a.qb + node * a.qn + (int64_t)(h * G + (r < rows ? r - node * G : 0)) * a.qh + 8 * g;
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[s] = __builtin_bit_cast(bf16x8, ld16(qp + 16 * s));
    }
    const int end = __builtin_amdgcn_readfirstlane(tree_len(a, ctx));
    ctx = __builtin_amdgcn_readfirstlane(ctx < 0 ? 0 : (ctx > a.Tmax ? a.Tmax : ctx));
    t1 = min(t1, (uint32_t)((end + kTreeTile - 1) / kTreeTile));
    const int newrow = a.knew ? ctx + a.first : a.Tmax;   // rows from here on come from knew / vnew

    uint16_t* const tile0 = reinterpret_cast<uint16_t*>(lds) + wk * kTile;   // of buffer 0
    const int lr = lane / LPR, lc = (lane % LPR) * 8;   // this lane's row of a load and its column
    const TreeRows ck = {a.k + b * a.kb + h * a.kh + lc, a.knew + b * a.knb + h * a.knh + lc, pinned(a.kt), pinned(a.knn)};
    const TreeRows cv = {a.v + b * a.vb + h * a.vh + lc, a.vnew + b * a.vnb + h * a.vnh + lc, pinned(a.vt), pinned(a.vnn)};
    const bool values = WQ > 1 && wq >= WQ / 2;         // this wave loads values, of a stream's several
    const TreeRows mine = values ? cv : ck;
    const int part = WQ > 1 ? (wq % (WQ > 1 ? WQ / 2 : 1)) * PW : 0;   // its first load of the tile's NV of that kind

    uint64_t live = 0;   // set once the first loads are under way
    uint4 st[PW];
    // Tiles of the context alone take their rows as they lie; the tree's (at most three a sequence) clamp
    // the row to the last one.
    auto load_rows = [&](const TreeRows& c, int j0, int first, int n, uint4* to) {
        if (j0 + kTreeTile <= ctx) {
            const uint16_t* p = c.cached + (j0 + first * RPI + lr) * c.st;
#pragma unroll
            for (int i = 0; i < n; ++i) to[i] = ld16(p + i * RPI * c.st);
        } else {
#pragma unroll
            for (int i = 0; i < n; ++i) to[i] = ld16(c.at(j0 + (first + i) * RPI + lr, end, newrow));
        }
    };
    auto load = [&](int j0) {
        if constexpr (WQ == 1) {
            load_rows(ck, j0, 0, NV, st);
            load_rows(cv, j0, 0, NV, st + NV);
        } else {
            load_rows(mine, j0, part, PW, st);
        }
    };
    // New rows into the cache, out of the registers of the wave that loaded them (for the first row group)
    auto keep_rows = [&](const TreeRows& c, int j0, int first, int n, const uint4* from) {
        if (rg != 0 || j0 + kTreeTile <= newrow) return;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const int j = j0 + (first + i) * RPI + lr;
            if (j >= newrow && j < end && ((live >> (j - ctx)) & 1)) st16(const_cast<uint16_t*>(c.cached) + j * c.st, from[i]);
        }
    };
    // Loaded values into LDS.  In the tree's tiles, values of rows that are nobody's key are zeros, whatever
    // they hold, and so are infinities and NaN: the queries that see them add them by themselves.
    auto put_values = [&](uint16_t* vt, int j0, int first, int n, uint4* from, int* flag) {
        if (j0 + kTreeTile > ctx) {
            bool bad = false;
#pragma unroll
            for (int i = 0; i < n; ++i) {
                const int j = j0 + (first + i) * RPI + lr;
                const bool key = j < ctx || (j < end && ((live >> (j - ctx)) & 1));
                const uint32_t keep = key ? 0xffffffffu : 0u;
                uint32_t x[4] = {from[i].x & keep, from[i].y & keep, from[i].z & keep, from[i].w & keep};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool lo = bf16_not_finite(x[e]), hi = bf16_not_finite(x[e] >> 16);
                    bad |= lo || hi;
                    x[e] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
                }
                from[i] = make_uint4(x[0], x[1], x[2], x[3]);
            }
            const uint64_t any = __ballot(bad);
            if (lane == 0) *flag = any != 0;
        }
#pragma unroll
        for (int i = 0; i < n; ++i) st16(vt + ((first + i) * RPI + lr) * VLD + lc, from[i]);
    };
    auto put = [&](int j0, int buf) {
        uint16_t* ks = tile0 + buf * WK * kTile;
        uint16_t* vt = ks + kTreeTile * KLD;
        if (WQ == 1 || !values) {
            keep_rows(ck, j0, part, WQ == 1 ? NV : PW, st);
#pragma unroll
            for (int i = 0; i < (WQ == 1 ? NV : PW); ++i) st16(ks + ((part + i) * RPI + lr) * KLD + lc, st[i]);
        }
        if (WQ == 1 || values) {
            uint4* v = st + (WQ == 1 ? NV : 0);
            keep_rows(cv, j0, part, WQ == 1 ? NV : PW, v);
            put_values(vt, j0, part, WQ == 1 ? NV : PW, v, &odd[buf][w]);
        }
    };

    const float sc = a.scale * kLog2e;
    float m = kTreeNegInf, l = 0.f;
    f32x16 acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;

    auto compute = [&](int j0, int buf) {
        const uint16_t* ks = tile0 + buf * WK * kTile;
        const uint16_t* vt = ks + kTreeTile * KLD;
        const bool tail = j0 + kTreeTile > ctx;
        f32x16 s;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
        for (int c = 0; c < KS; ++c) s = mfma32(lds_op_row(ks, KLD, 0, 16 * c, lane), qf[c], s);
        if (tail) {   // the tree's rows: one bit a key
            const uint32_t see = j0 < ctx ? (uint32_t)(bits << (ctx - j0)) | ((1u << (ctx - j0)) - 1u)
                                          : (j0 - ctx < 64 ? (uint32_t)(bits >> (j0 - ctx)) : 0u);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (!((see >> (8 * (i >> 2) + (i & 3) + 4 * g)) & 1u)) s[i] = kTreeNegInf;
        }
        float mc = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mc = fmaxf(mc, s[i]);
        mc = fmaxf(mc, __shfl_xor(mc, 32, 64));
        if (__ballot(mc * sc > m * sc + kTreeLazy)) {
            const float mn = fmaxf(m, mc);
            const float mu = mn == kTreeNegInf ? 0.f : mn;
            const float f = exp2_fast((m - mu) * sc);
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[d][i] *= f;
            m = mn;
        }
        const float ms = m == kTreeNegInf ? 0.f : m * sc;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[i] = exp2_fast(fmaf(s[i], sc, -ms));
            l += s[i];
        }
        if (tail) {
            int any = 0;
            if (WQ == 1) any = odd[0][w];
            else
#pragma unroll
                for (int x = WQ / 2; x < WQ; ++x) any |= odd[buf][wk * WQ + x];
            if (__ballot(any)) {
                // An infinity or a NaN among the tree's values belongs to the queries that see its row alone (a
                // product with the others' zeros would give them a NaN): added here, row by row.
                for (int j = 0; j < kTreeTile && j0 + j < end; ++j) {
                    if (j0 + j >= ctx && !((live >> (j0 + j - ctx)) & 1)) continue;
                    float p = 0.f;
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (8 * (i >> 2) + (i & 3) == (j & ~4)) p = s[i];
                    p = __shfl(p, ln + 32 * ((j >> 2) & 1), 64);
                    const uint16_t* row = cv.at(j0 + j, end, newrow) - lc + 4 * g;
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const uint32_t x = row[32 * d + 8 * (e >> 2) + (e & 3)];
                            if (bf16_not_finite(x) && p > 0.f) acc[d][e] += p * bf16_to_f32((uint16_t)x);
                        }
                        asm volatile("" ::: "memory");   // 32 columns' loads at a time: registers
                    }
                }
            }
        }
        bf16x8 vo[DT];
#pragma unroll
        for (int d = 0; d < DT; ++d) vo[d] = lds_op_t(vt, VLD, 0, 32 * d, lane);
        // p <= 2^8 in bf16, 2^-8 of it off at most; the sums take it unrounded.  One row group (a single token's heads among
        // them, whose decode attention keeps p in fp32) takes what that rounding drops as a second operand, p to 2^-16: 225 keys
        // of 12 heads 7.0 -> 7.1 us, 1,000 keys 9.8 -> 10.7 (a chain that nothing hides), 1,000 keys of 192 heads 11.4 -> 12.1,
        // one token over 65,011 95.1 both.  More row groups keep the one rounding: 128 rows of 8 heads of 128 over 32,768 keys
        // would go 98 -> 113 us, 305 rows 32.0 -> 35.5.
        constexpr int PARTS = WQ == 1 ? 2 : 1;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            f32x8 x = c == 0 ? __builtin_shufflevector(s, s, 0, 1, 2, 3, 4, 5, 6, 7)
                             : __builtin_shufflevector(s, s, 8, 9, 10, 11, 12, 13, 14, 15);
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
                const bf16x8 pf = __builtin_convertvector(x, bf16x8);
                if (part + 1 < PARTS) x -= __builtin_convertvector(pf, f32x8);
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    acc[d] = mfma32(vo[d], pf, acc[d]);
                    if (c == 0 && part + 1 == PARTS) vo[d] = lds_op_t(vt, VLD, 16, 32 * d, lane);
                }
            }
        }
    };

    // The loop has all of a step's loads in every turn (the last step is its own): the waits for older loads
    // count the younger.  The queries have to be here before it: a wait for them inside would be
    // one for the tile's loads behind them, every time.
    uint32_t t = t0 + wk;
    auto queries_here = [&] {
#pragma unroll
        for (int c = 0; c < KS; ++c) asm volatile("" : "+v"(qf[c]));
        live = tree_live(a, word, ctx, lane);
        bits = r < rows && ((bits >> (a.first + node)) & 1) ? bits & live : 0ull;
    };
    if constexpr (WQ == 1) {
        if (t < t1) {
            load((int)t * kTreeTile);
            queries_here();
            for (;; t += WK) {
                const int j0 = (int)t * kTreeTile;
                put(j0, 0);
                tree_wave_order();
                if (t + WK >= t1) break;
                load(j0 + WK * kTreeTile);
                compute(j0, 0);
                tree_wave_order();   // before the next tile is written over this one
            }
            compute((int)t * kTreeTile, 0);
        }
    } else {
        // every stream takes the steps of the first, for the barriers; a tile past the last one is the last
        // one's rows again, not counted
        const int steps = (int)((t1 - t0 + WK - 1) / WK);
        if (steps > 0) {
            load((int)t * kTreeTile);
            queries_here();
            int s = 0;
            for (; s < steps - 1; ++s, t += WK) {
                const int j0 = (int)t * kTreeTile;
                put(j0, s & 1);
                load(j0 + WK * kTreeTile);
                __syncthreads();
                compute(j0, s & 1);
            }
            put((int)t * kTreeTile, s & 1);
            __syncthreads();
            if (t < t1) compute((int)t * kTreeTile, s & 1);
        }
    }

    // join the WK streams of a row
    l += __shfl_xor(l, 32, 64);
    const float ms = m * sc;   // -inf where the stream had no key
    __syncthreads();           // V tiles are done with
    {
        float* op = reinterpret_cast<float*>(lds) + (w * kTreeTile + ln) * OLD;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<float4*>(op + 32 * d + 8 * q + 4 * g) =
                    make_float4(acc[d][4 * q], acc[d][4 * q + 1], acc[d][4 * q + 2], acc[d][4 * q + 3]);
        if (g == 0) ml[w][ln] = make_float2(ms, l);
    }
    __syncthreads();
    const int64_t per = (int64_t)32 * WQ * (D + 2);   // floats of a unit's partial
    float* unit = a.work + (int64_t)blockIdx.x * per;
    for (int i = threadIdx.x; i < 32 * WQ * LPR; i += kTreeThreads) {
        const int rr = i / LPR, c = (i % LPR) * 8;      // row of the unit, columns c..c+7
        const int row = rg * WQ * kTreeTile + rr;
        if (row >= rows) continue;
        const int wr = rr >> 5, rl = rr & 31;
        float M = kTreeNegInf;
#pragma unroll
        for (int x = 0; x < WK; ++x) M = fmaxf(M, ml[x * WQ + wr][rl].x);
        const float mu = M == kTreeNegInf ? 0.f : M;
        float L = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < WK; ++x) {
            const float2 z = ml[x * WQ + wr][rl];
            const float f = exp2_fast(z.x - mu);
            L += z.y * f;
            const float* op = reinterpret_cast<const float*>(lds) + ((x * WQ + wr) * kTreeTile + rl) * OLD + c;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] += op[e] * f;
        }
        if (count == 1) {
            const int n = row / G;
            const bool pad = !((a.tree[b * a.treeb + n * a.treen] >> (a.first + n)) & 1);
            const float inv = pad || L == 0.f ? 0.f : 1.f / L;
            const int64_t at = ((int64_t)b * a.N + n) * a.H + h * G + row - n * G;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = pad || L == 0.f ? 0.f : o[e] * inv;
            st16(a.o + at * D + c, pack8(o));
            if (a.lse && c == 0) a.lse[at] = pad || L == 0.f ? kTreeNegInf : (M + log2_fast(L)) * kLn2;
        } else {
#pragma unroll
            for (int e = 0; e < 8; e += 4)
                *reinterpret_cast<float4*>(unit + rr * D + c + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            if (c == 0) *reinterpret_cast<float2*>(unit + 32 * WQ * D + 2 * rr) = make_float2(M, L);
        }
    }
}

// Join the units of query rows: WPR waves a row (1, or 4 where a row has many units), D / 4 lanes of them for a
// unit's row of D floats.
template <int D, int WPR>
__global__ void __launch_bounds__(256) tree_join_kernel(TreeArgs a, TreePlan plan) {
    constexpr int LPR = D / 4, NS = WPR * 64 / LPR;   // units read side by side
    __shared__ float2 sml[WPR];
    __shared__ __attribute__((aligned(16))) float so[WPR][D];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int G = a.H / a.Hkv, heads = plan.groups * a.Hkv;
    const int row = WPR == 1 ? blockIdx.x * 4 + w : blockIdx.x;
    if (row >= a.B * a.N * a.H) return;
    const int hq = row % a.H, bn = row / a.H, n = bn % a.N, b = bn / a.N;
    const uint2 place = tree_places(a, plan)[b];
    const uint64_t bits = (uint64_t)a.tree[b * a.treeb + n * a.treen];
    const uint32_t first = place.x, count = place.y;
    if (count == 1) return;   // written by its unit
    const int h = hq / G, rq = n * G + hq - h * G, rg = rq / (32 * plan.wq), rr = rq - rg * 32 * plan.wq;
    const int64_t per = (int64_t)32 * plan.wq * (D + 2), step = heads * per;
    const float* base = a.work + ((int64_t)first * heads + rg * a.Hkv + h) * per;
    const int st = (WPR == 1 ? lane : (int)threadIdx.x) / LPR, c = (lane % LPR) * 4;
    float M = kTreeNegInf, L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    auto join = [&](float m, float l, const float4& x) {
        const float mn = fmaxf(M, m), mu = mn == kTreeNegInf ? 0.f : mn;
        const float f = exp2_fast(M - mu), fx = exp2_fast(m - mu);
        L = L * f + l * fx;
        o.x = o.x * f + x.x * fx;
        o.y = o.y * f + x.y * fx;
        o.z = o.z * f + x.z * fx;
        o.w = o.w * f + x.w * fx;
        M = mn;
    };
    constexpr int U = 4;   // units of a lane in flight
    for (uint32_t u = st; u < count; u += NS * U) {
        float2 z[U];
        float4 x[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const float* p = base + (int64_t)min(u + i * NS, count - 1) * step;
            z[i] = *reinterpret_cast<const float2*>(p + 32 * plan.wq * D + 2 * rr);
            x[i] = *reinterpret_cast<const float4*>(p + rr * D + c);
        }
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (u + i * NS < count) join(z[i].x, z[i].y, x[i]);
    }
#pragma unroll
    for (int off = LPR; off < 64; off <<= 1)
        join(__shfl_xor(M, off, 64), __shfl_xor(L, off, 64),
             make_float4(__shfl_xor(o.x, off, 64), __shfl_xor(o.y, off, 64), __shfl_xor(o.z, off, 64), __shfl_xor(o.w, off, 64)));
    if (WPR > 1) {
        if (lane < LPR) *reinterpret_cast<float4*>(&so[w % WPR][c]) = o;
        if (lane == 0) sml[w % WPR] = make_float2(M, L);
        __syncthreads();
        if (w != 0) return;
#pragma unroll
        for (int x = 1; x < WPR; ++x) join(sml[x].x, sml[x].y, *reinterpret_cast<const float4*>(&so[x][c]));
    }
    if (lane >= LPR) return;
    const bool none = L == 0.f || !((bits >> (a.first + n)) & 1);
    const float inv = none ? 0.f : 1.f / L;
    uint2 out;
    out.x = none ? 0u : pack_bf16x2(o.x * inv, o.y * inv);
    out.y = none ? 0u : pack_bf16x2(o.z * inv, o.w * inv);
    *reinterpret_cast<uint2*>(a.o + (int64_t)row * D + c) = out;
    if (a.lse && lane == 0) a.lse[row] = none ? kTreeNegInf : (M + log2_fast(L)) * kLn2;
}

// Launch shape.  One workgroup a CU is resident (its registers), so R = CUs of them run at once.
// Caches of up to six steps of a workgroup are not split: 12 key heads over 1,000 keys 10.7 us against 12.7 for two
// launches, over 1,500 13.1 / 12.9, over 2,000 15.6 / 12.7; 32 over 350 keys in four row groups 15.8 / 16.1.  Key
// heads (with row groups) below half of R are split into units that R leaves over, so that all of them run at once.
// More of them are split for unlike sequences alone, at twice the mean length, where a cache may hold 64 steps of a
// workgroup or more: one sequence of 19,000 keys among 63 of 500 (8 key heads) 32 us against 93, of 60,000
// 43 / 276, at the cost of a join that finds nothing: 192 of 18,000 keys each 162 / 159, 64 sequences
// of 500 24.6 / 19.9; in caches of 8,192 rows such splits lost 3 to 11 % on mixed lengths and are not made.
// Equal long sequences pay for a last round that is not full: 18,000 keys a head of 128 take 4.7 to 4.9 TB/s for 112 to
// 136 key heads (no step at half of R), 6.0 for 256, 4.2 for 264 and 6.0 for 512.
static TreePlan tree_plan(int32_t B, int32_t N, int32_t H, int32_t Hkv, int32_t Tmax) {
    TreePlan p{};
    const int rows = N * (H / Hkv);
    // row groups: one workgroup's while the keys' bytes bound it (8 tiles of 32 rows at most), else of whichever
    // size pads fewer rows (305 rows as three groups of four tiles 33 us, as two of eight 39)
    const int tiles32 = (rows + 31) / 32;
    p.wq = tiles32 == 1 ? 1 : tiles32 == 2 ? 2 : tiles32 <= 4 ? 4 : tiles32 <= 8 || (tiles32 + 3) / 4 % 2 == 0 ? 8 : 4;
    p.groups = (rows + 32 * p.wq - 1) / (32 * p.wq);
    const int64_t pairs = (int64_t)B * Hkv * p.groups, cus = device_cus();
    const int wk = kTreeWaves / p.wq;
    p.least = 2 * wk;
    const int64_t tiles = (Tmax + kTreeTile - 1) / kTreeTile;
    p.grid = (int32_t)pairs;
    if (tiles <= 6 * wk) return p;
    if (pairs < cus / 2) p.units = (int32_t)(cus - pairs);
    else if (pairs <= 8 * cus && tiles >= 64 * wk) p.units = (int32_t)(pairs / 2);
    else return p;
    // sum over sequences of ceil(tiles / unit) heads <= units + B heads, in whole multiples of heads
    const int32_t heads = p.groups * Hkv;
    p.grid = (int32_t)((p.units + pairs) / heads * heads);
    return p;
}

int64_t tree_attention_workspace(int32_t B, int32_t N, int32_t H, int32_t Hkv, int32_t Tmax, int32_t D) {
    if (B < 1 || N < 1 || Hkv < 1 || H < Hkv || H % Hkv || Tmax < 1 || (D != 64 && D != 128)) return 0;
    const TreePlan p = tree_plan(B, N, H, Hkv, Tmax);
    return p.units == 0 ? 0 : (int64_t)p.grid * 32 * p.wq * (D + 2) * (int64_t)sizeof(float) + B * (int64_t)sizeof(uint2);
}

template <int D>
static int tree_launch(const TreeArgs& a, const TreePlan& p, hipStream_t st) {
    const dim3 grid((unsigned)p.grid), block(kTreeThreads);
    switch (p.wq) {
        case 1: hipLaunchKernelGGL((tree_attn_kernel<D, 1>), grid, block, 0, st, a, p); break;
        case 2: hipLaunchKernelGGL((tree_attn_kernel<D, 2>), grid, block, 0, st, a, p); break;
        case 4: hipLaunchKernelGGL((tree_attn_kernel<D, 4>), grid, block, 0, st, a, p); break;
        default: hipLaunchKernelGGL((tree_attn_kernel<D, 8>), grid, block, 0, st, a, p); break;
    }
    if (int e = check_launch("tree_attention")) return e;
    if (p.units == 0) return 0;
    const int64_t rows = (int64_t)a.B * a.N * a.H;
    // Over 16 units a row, four waves of them: with 255 units 26 us against 46, with 31 27.0 / 27.6; with 7 a wave a row
    // is the better, 18 us against 25.
    if (p.units > 16 * a.B * p.groups * a.Hkv)
        hipLaunchKernelGGL((tree_join_kernel<D, 4>), dim3((unsigned)rows), dim3(256), 0, st, a, p);
    else
        hipLaunchKernelGGL((tree_join_kernel<D, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a, p);
    return check_launch("tree_attention_join");
}

int tree_attention(const TreeArgs& a, void* stream) {
    FX_REQUIRE(a.D == 64 || a.D == 128, "tree_attention: head_dim %d not supported (64 or 128)", a.D);
    FX_REQUIRE(a.B >= 1 && a.N >= 1 && a.Tmax >= 1 && a.Hkv >= 1 && a.H >= a.Hkv && a.H % a.Hkv == 0,
               "tree_attention: bad shape B=%d N=%d H=%d Hkv=%d Tmax=%d", a.B, a.N, a.H, a.Hkv, a.Tmax);
    FX_REQUIRE(a.first >= 0 && a.first <= 63 && a.first + a.N <= 64, "tree_attention: %d nodes behind %d: a tree has 64 at most", a.N, a.first);
    FX_REQUIRE(a.Tmax <= 0x7fffffff - 128, "tree_attention: Tmax=%d too large", a.Tmax);
    FX_REQUIRE(a.q && a.k && a.v && a.ctx && a.tree && a.o, "tree_attention: null pointer");
    FX_REQUIRE((a.knew == nullptr) == (a.vnew == nullptr), "tree_attention: knew and vnew go together");
    FX_REQUIRE(a.scale > 0.f && a.scale < __builtin_huge_valf(), "tree_attention: scale %g must be positive and finite", (double)a.scale);
    const int64_t s[] = {a.qb, a.qn, a.qh, a.kb, a.kt, a.kh, a.vb, a.vt, a.vh, a.knb, a.knn, a.knh, a.vnb, a.vnn, a.vnh};
    for (int64_t x : s) FX_REQUIRE(x % 8 == 0, "tree_attention: strides must be multiples of 8 elements");
    FX_REQUIRE((((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.o | (uintptr_t)a.work | (uintptr_t)a.knew |
                 (uintptr_t)a.vnew) & 15) == 0,
               "tree_attention: q, k, v, o, work, knew and vnew must be 16-byte aligned");
    const TreePlan p = tree_plan(a.B, a.N, a.H, a.Hkv, a.Tmax);
    const int64_t pairs = (int64_t)a.B * p.groups * a.Hkv, tiles = pairs * ((a.Tmax + kTreeTile - 1) / kTreeTile);
    FX_REQUIRE(tiles < 0x7fffffffLL && (int64_t)a.B * a.N * a.H < 0x7fffffffLL && pairs <= 0xffffffffu / kTreeThreads,
               "tree_attention: grid too large");   // a launch has less than 2^32 work items (units are made of few pairs alone)
    FX_REQUIRE(p.units == 0 || a.work, "tree_attention: null workspace");
    return a.D == 64 ? tree_launch<64>(a, p, (hipStream_t)stream) : tree_launch<128>(a, p, (hipStream_t)stream);
}

}  // namespace fx
