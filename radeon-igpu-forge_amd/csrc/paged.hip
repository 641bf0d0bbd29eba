// Attention of one new token a row over a paged key-value cache, for gfx950.
//
// Row r has lens[r] keys; key j lies in page table[r, j / P], row j % P of it:
//
//   o[r, h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q[r, h] . k_j),   j < lens[r],
//
// in one pass with a running maximum and sum.  Query heads share key heads: the G = H / Hkv heads of a
// key head are columns of one product, 16 to a wave's MFMA tile.  A row without keys gives zeros.  The
// new token's key and value (knew, vnew), where given, are key lens[r] - 1 and are written to its page.
//
// HBM-bound: a row's keys and values are read once for up to 32 query heads of a key head (4 D bytes a token and key head;
// once more for every further 32, and a page that rows share once for each of them).  So the keys are split
// evenly, whatever the rows' lengths: all rows' and heads' steps of 32 keys lie in one line, and each
// workgroup of one full round of CUs takes an equal piece of it, over the border of a row or a head if
// that falls in it.  A second kernel joins the rows that were cut.  Four waves a workgroup, each with a
// key head of its own where there are as many: no wave waits for another.  64 rows of up to 6,000 tokens, 8 key heads of 128:
// 788 MB in 129 us (6.1 TB/s; 124 of them this kernel, which streams at 7.1 behind its first round trips); 3 rows of up to
// 65,001 tokens, 16 heads of 64: 584 MB in 95 (89).  Tables of up to 1,536 keys are not split: a
// workgroup of eight waves a row and key head, one launch (one row of 12 heads over 217 keys 5.9 us against 9.3 split,
// 1,500 keys 11.7 / 11.5, 3,000 18.5 / 15.6; 64 rows of up to 1,500 40.3 / 41.3).
//
#include <math.h>

#include "fx_internal.h"
#include "fx_mfma.h"

namespace fx {

constexpr int kPagedTile = 32;       // keys of a wave's step
constexpr int kPagedCols = 16;       // query heads of an MFMA tile
constexpr float kPagedNegInf = -__builtin_huge_valf();
constexpr float kPagedLazy = 8.f;    // the running maximum moves only past this (log2 units): p stays <= 2^8

// what a kernel needs besides the arguments: groups of query heads of a key head, query heads of a group,
// workgroups of a split launch (0: not split), key heads and parts of the keys of a workgroup, whether loads go past the caches
struct PagedPlan {
    int32_t groups, gt, split, hw, kw;
    bool once;
};

__device__ __forceinline__ f32x4 mfma16(const bf16x8& a, const bf16x8& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// keys of a row whose length is given as `n`
__device__ __forceinline__ int paged_len(const PagedArgs& a, int n) {
    const int64_t most = (int64_t)a.M << a.shift;
    return n < 0 ? 0 : n < most ? n : (int)most;
}
// its steps, one at least: a row without keys has its zeros written
template <int KW>
__device__ __forceinline__ uint32_t paged_steps(const PagedArgs& a, int n) {
    const uint32_t l = (uint32_t)paged_len(a, n);
    return l ? (l + kPagedTile * KW - 1) / (kPagedTile * KW) : 1u;
}

// two tiles of query heads of 128 take more than the registers of two waves a SIMD: then four waves a workgroup
constexpr bool paged_wide(int D, int NT) { return D == 128 && NT == 2; }

// floats of a piece: its rows' outputs, their maxima and sums; whole 16-byte vectors
__host__ __device__ __forceinline__ int64_t paged_piece(const PagedPlan& p, int D) { return ((int64_t)p.gt * (D + 2) + 3) & ~3ll; }

// where the join finds the pieces of a row and head group: (first workgroup, count), behind the partials
__device__ __forceinline__ uint2* paged_places(const PagedArgs& a, const PagedPlan& p) {
    return reinterpret_cast<uint2*>(a.work + (int64_t)2 * p.split * p.hw * paged_piece(p, a.D));
}

// Workgroup: HW key heads x KW parts of a row's keys, a wave each.  Per tile of 32 keys S^T = K Q^T (a lane
// holds 8 of the 32 keys of one query head), the softmax, and O^T += V^T P^T.  Keys and values go through the wave's own
// LDS in whole rows (keys straight from memory in the operand's layout, 64 bytes of 16 rows a load: rows of 64 in
// pools of 16 heads 103 us against 98); values are read transposed (fx_mfma.h), keys in the order that the scores
// lie in.  The next tile is in flight in registers meanwhile.  P >= 16, so half a tile lies in one page: addresses
// are a base in scalar registers and an offset that does not change.  The wave holds 64 entries of the row's table
// in a register, and the 64 behind them.
// ONCE: pools that are too large to stay in the caches from one call to the next are loaded past them (64 rows of up to 6,000
// tokens 162 -> 152 us then; a batch whose 38 MB stay there would go from 10.5 to 13.9).  Else rows may share pages, and an eighth
// of the line goes to each XCD, whose L2 then has what a prompt's beams have in common (35 beams 38.9 -> 31.5 us).
template <int D, int NT, int HW, int KW, bool ONCE>
__global__ void __launch_bounds__(64 * HW * KW, paged_wide(D, NT) ? 1 : 2) paged_attn_kernel(PagedArgs a, PagedPlan plan) {
    constexpr int NW = HW * KW;
    constexpr int LPR = D / 8;         // lanes of a row in 16-byte loads
    constexpr int RPI = 64 / LPR;      // rows of a wave-wide load
    constexpr int NV = kPagedTile / RPI;
    constexpr int KS = D / 32;         // steps of the score product
    constexpr int DT = D / 16;
    constexpr int VLD = D + 16;        // LDS row of V: 8 rows of a transposed read fall in distinct banks
    constexpr int OLD = D + 4;         // LDS row of a wave's fp32 output
    constexpr int KLD = D + 8;         // LDS row of K: 16 rows of an operand read fall in distinct banks
    constexpr int kV = kPagedTile * (VLD + KLD) * 2, kO = kPagedCols * OLD * 4;
    constexpr int kWave = kV > kO ? kV : kO;
    __shared__ __attribute__((aligned(16))) unsigned char lds[NW * kWave];
    __shared__ float2 ml[NW][kPagedCols];

    const int lane = threadIdx.x & 63, lc = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hw = w % HW, kw = w / HW;
    const int G = a.H / a.Hkv, heads = plan.groups * (a.Hkv / HW), rowmask = (1 << a.shift) - 1;
    uint16_t* const vt = reinterpret_cast<uint16_t*>(lds + w * kWave);
    uint16_t* const kt = vt + kPagedTile * VLD;
    float* const ot = reinterpret_cast<float*>(lds + w * kWave);
    const float sc = a.scale * kLog2e;
    const int vr = lane / LPR, vc = (lane % LPR) * 8;   // this lane's row of a value load and its column

    // this workgroup's piece of the line, and where it begins: row, head group, step
    int r = 0, hr = 0;
    uint32_t s0 = 0, parts = 1, piece = blockIdx.x;
    uint64_t pos = 0, stop = 0, total = 0;
    if (plan.split == 0) {
        r = blockIdx.x / heads;
        hr = blockIdx.x - r * heads;
        stop = 1;
    } else {
        uint32_t sum = 0;
        for (int x = lane; x < a.R; x += 64) sum += paged_steps<KW>(a, a.lens[x]);
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
        total = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane(sum) * heads;
        parts = (uint32_t)(total < (uint32_t)plan.split ? total : plan.split);   // one step each at least
        if (blockIdx.x >= parts) return;
        if constexpr (!ONCE) {   // an eighth of the line for each XCD
            const uint32_t x = blockIdx.x % 8, each = parts / 8, more = parts % 8;
            piece = x * each + min(x, more) + blockIdx.x / 8;
        }
        pos = total * piece / parts;
        stop = total * (piece + 1) / parts;
        uint32_t at = (uint32_t)(pos / heads), before = 0;   // in steps of one head group
        for (int x0 = 0; x0 < a.R; x0 += 64) {
            const uint32_t k = x0 + lane < a.R ? paged_steps<KW>(a, a.lens[x0 + lane]) : 0u;
            uint32_t up = k;   // inclusive scan
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const uint32_t o = __shfl_up(up, off, 64);
                if (lane >= off) up += o;
            }
            const uint64_t past = __ballot(before + up > at);
            if (past) {
                const int l = __ffsll((unsigned long long)past) - 1;
                r = x0 + l;
                const uint32_t steps = (uint32_t)__builtin_amdgcn_readlane((int)k, l);
                before += (uint32_t)__builtin_amdgcn_readlane((int)up, l) - steps;
                const uint32_t in = (uint32_t)(pos - (uint64_t)before * heads);
                hr = in / steps;
                s0 = in - hr * steps;
                break;
            }
            before += (uint32_t)__builtin_amdgcn_readlane((int)up, 63);
        }
    }
    r = __builtin_amdgcn_readfirstlane(r);
    hr = __builtin_amdgcn_readfirstlane(hr);
    s0 = __builtin_amdgcn_readfirstlane(s0);

    while (pos < stop && r < a.R) {
        const int len = __builtin_amdgcn_readfirstlane(paged_len(a, a.lens[r]));
        const uint32_t steps = paged_steps<KW>(a, len);
        const uint32_t n = plan.split ? (uint32_t)(stop - pos < steps - s0 ? stop - pos : steps - s0) : steps;
        const int grp = hr / (a.Hkv / HW), h = (hr - grp * (a.Hkv / HW)) * HW + hw;
        const int q0 = grp * plan.gt, rows = min(plan.gt, G - q0);   // this group's first query head and their number

        bf16x8 qf[NT][KS];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const uint16_t* qp = a.q + (int64_t)r * a.qr + (int64_t)(h * G + q0 + min(t * kPagedCols + lc, rows - 1)) * a.qh + 8 * g;
#pragma unroll
            for (int s = 0; s < KS; ++s) qf[t][s] = __builtin_bit_cast(bf16x8, ld16(qp + 32 * s));
        }

        // this wave's tiles
        const int tiles = (len + kPagedTile - 1) / kPagedTile;
        const int ta = min((int)(s0 * KW), tiles), cnt = min((int)((s0 + n) * KW), tiles) - ta;
        int t = ta + cnt * kw / KW;
        const int t1 = ta + cnt * (kw + 1) / KW;

        const int32_t* tab = a.table + (int64_t)r * a.tab;
        auto window = [&](int e0) { return tab[min(e0 + lane, a.M - 1)]; };   // 64 entries from e0 on

        f32x4 acc[NT][DT];
        float m[NT], l[NT];
#pragma unroll
        for (int x = 0; x < NT; ++x) {
            m[x] = kPagedNegInf, l[x] = 0.f;
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[x][d] = f32x4{0.f, 0.f, 0.f, 0.f};
        }

        if (t < t1) {
            int base = ((t * kPagedTile) >> a.shift) & ~63;
            int win = window(base), nxt = window(base + 64);
            uint4 kk[NV], vv[NV];
            int have[2];   // keys of the loaded tile's halves
            const char* const kh = reinterpret_cast<const char*>(a.k + (int64_t)h * a.kh);
            const char* const vh = reinterpret_cast<const char*>(a.v + (int64_t)h * a.vh);
            const uint32_t kt2 = (uint32_t)a.kt * 2u, vt2 = (uint32_t)a.vt * 2u;
            auto get = [](const char* p) { return ONCE ? ld16_nt(p) : ld16(p); };
            auto load = [&](int j0) {
                const int b0 = (j0 >> a.shift) & ~63;
                if (b0 != base) {
                    base = b0;
                    win = nxt;
                    nxt = window(base + 64);
                }
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int js = j0 + 16 * half, jh = min(js, (len - 1) & ~15);   // a half without keys: the last one's rows again
                    const int id = __builtin_amdgcn_readlane(win, (jh >> a.shift) & 63);
                    const bool is = (uint32_t)id < (uint32_t)a.N;   // keys of an entry that is no page are nobody's
                    const int64_t page = is ? id : 0;
                    have[half] = is ? max(0, min(16, len - js)) : 0;
                    const char* kp = kh + (page * a.kp + (int64_t)(jh & rowmask) * a.kt) * 2;
                    const char* vp = vh + (page * a.vp + (int64_t)(jh & rowmask) * a.vt) * 2;
                    // rows behind the last key are its own again
                    const uint32_t lim = (uint32_t)(len - 1 - jh);
#pragma unroll
                    for (int i = 0; i < NV / 2; ++i) {
                        const uint32_t row = min((uint32_t)(i * RPI + vr), lim);
                        kk[half * NV / 2 + i] = get(kp + (__umul24(row, kt2) + 2u * vc));
                        vv[half * NV / 2 + i] = get(vp + (__umul24(row, vt2) + 2u * vc));
                    }
                    if (a.knew && js < len && lim < 16) {   // the new key and value: used from here, and kept
                        const bool keep = grp == 0 && is;
#pragma unroll
                        for (int i = 0; i < NV / 2; ++i)
                            if ((uint32_t)(i * RPI + vr) == lim) {
                                kk[half * NV / 2 + i] = ld16(a.knew + (int64_t)r * a.knr + (int64_t)h * a.knh + vc);
                                vv[half * NV / 2 + i] = ld16(a.vnew + (int64_t)r * a.vnr + (int64_t)h * a.vnh + vc);
                                if (keep) {
                                    st16(const_cast<char*>(kp) + (__umul24(lim, kt2) + 2u * vc), kk[half * NV / 2 + i]);
                                    st16(const_cast<char*>(vp) + (__umul24(lim, vt2) + 2u * vc), vv[half * NV / 2 + i]);
                                }
                            }
                    }
                }
            };

            load(t * kPagedTile);
            for (;;) {
                const int n0 = have[0], n1 = have[1];
                const bool part = n0 < 16 || n1 < 16;
                if (part) {   // values of rows that are no keys are zeros, whatever they hold
#pragma unroll
                    for (int i = 0; i < NV; ++i) {
                        const int row = (i % (NV / 2)) * RPI + vr;
                        if (row >= (i < NV / 2 ? n0 : n1)) vv[i] = make_uint4(0, 0, 0, 0);
                    }
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the last tile's reads come first
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int i = 0; i < NV; ++i) st16(kt + (i * RPI + vr) * KLD + vc, kk[i]), st16(vt + (i * RPI + vr) * VLD + vc, vv[i]);
                if (t + 1 < t1) load((t + 1) * kPagedTile);
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
                f32x4 s[NT][2];
#pragma unroll
                for (int x = 0; x < NT; ++x)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        s[x][half] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int c = 0; c < KS; ++c) s[x][half] = mfma16(*reinterpret_cast<const bf16x8*>(kt + (16 * half + lc) * KLD + 32 * c + 8 * g), qf[x][c], s[x][half]);
                    }
                bf16x8 hi[NT], lo[NT];
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    if (part) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (4 * g + i >= n0) s[x][0][i] = kPagedNegInf;
                            if (4 * g + i >= n1) s[x][1][i] = kPagedNegInf;
                        }
                    }
                    float mc = s[x][0][0];
#pragma unroll
                    for (int i = 1; i < 8; ++i) mc = fmaxf(mc, s[x][i >> 2][i & 3]);
                    mc = fmaxf(mc, __shfl_xor(mc, 16, 64));
                    mc = fmaxf(mc, __shfl_xor(mc, 32, 64));
                    if (__ballot(mc * sc > m[x] * sc + kPagedLazy)) {
                        const float mn = fmaxf(m[x], mc), mu = mn == kPagedNegInf ? 0.f : mn;
                        const float f = exp2_fast((m[x] - mu) * sc);
                        l[x] *= f;
#pragma unroll
                        for (int d = 0; d < DT; ++d) acc[x][d] *= f;
                        m[x] = mn;
                    }
                    const float ms = m[x] == kPagedNegInf ? 0.f : m[x] * sc;
                    f32x8 p;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        p[i] = exp2_fast(fmaf(s[x][i >> 2][i & 3], sc, -ms));
                        l[x] += p[i];
                    }
                    // p in two bf16 parts, to 2^-16: the output's rounding is the only one
                    hi[x] = __builtin_convertvector(p, bf16x8);
                    lo[x] = __builtin_convertvector(p - __builtin_convertvector(hi[x], f32x8), bf16x8);
                }
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const uint16_t* vp = vt + (4 * g + (lc >> 2)) * VLD + 16 * d + 4 * (lc & 3);
                    const bf16x8 vo = cat8(lds_tr16(vp), lds_tr16(vp + 16 * VLD));
#pragma unroll
                    for (int x = 0; x < NT; ++x) {
                        acc[x][d] = mfma16(vo, hi[x], acc[x][d]);
                        acc[x][d] = mfma16(vo, lo[x], acc[x][d]);
                    }
                }
                if (++t >= t1) break;
            }
        }

        const bool whole = n == steps;
        const int64_t per = paged_piece(plan, D);
        float* pieces = a.work + (2 * (int64_t)piece + (s0 == 0)) * HW * per;
        if (plan.split && s0 == 0 && threadIdx.x == 0) {   // the workgroup with the row's last step: the last one that begins at or before it
            const uint32_t last = whole ? piece : (uint32_t)(((pos + steps) * parts - 1) / total);
            paged_places(a, plan)[(int64_t)r * heads + hr] = make_uint2(piece, last - piece + 1);
        }
#pragma unroll
        for (int x = 0; x < NT; ++x) {
            float lx = l[x];
            lx += __shfl_xor(lx, 16, 64);
            lx += __shfl_xor(lx, 32, 64);
            const int some = min(kPagedCols, rows - x * kPagedCols);
            const float mx = m[x] * sc;
            if constexpr (KW == 1) {   // a wave has all of its head's keys of the segment
                if (lc < some) {
                    const int q = x * kPagedCols + lc;
                    if (whole) {
                        const float inv = lx == 0.f ? 0.f : 1.f / lx;
                        const int64_t at = (int64_t)r * a.H + h * G + q0 + q;
#pragma unroll
                        for (int d = 0; d < DT; ++d) {
                            f32x4 y = acc[x][d] * inv;
                            if (lx == 0.f) y = f32x4{0.f, 0.f, 0.f, 0.f};
                            *reinterpret_cast<uint2*>(a.o + at * D + 16 * d + 4 * g) = make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
                        }
                        if (a.lse && g == 0) a.lse[at] = lx == 0.f ? kPagedNegInf : (mx + log2_fast(lx)) * kLn2;
                    } else {
                        float* u = pieces + hw * per;
#pragma unroll
                        for (int d = 0; d < DT; ++d)
                            *reinterpret_cast<float4*>(u + q * D + 16 * d + 4 * g) = make_float4(acc[x][d][0], acc[x][d][1], acc[x][d][2], acc[x][d][3]);
                        if (g == 0) *reinterpret_cast<float2*>(u + (int64_t)plan.gt * D + 2 * q) = make_float2(mx, lx);
                    }
                }
            } else {   // join the waves of a head, 16 query heads at a time
                if (x > 0) __syncthreads();   // the last round's sums are read
                // the wave's own values are read: its LDS operations are done in order
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int d = 0; d < DT; ++d)
                    *reinterpret_cast<float4*>(ot + lc * OLD + 16 * d + 4 * g) = make_float4(acc[x][d][0], acc[x][d][1], acc[x][d][2], acc[x][d][3]);
                if (g == 0) ml[w][lc] = make_float2(mx, lx);
                __syncthreads();
                for (int i = threadIdx.x; i < HW * some * LPR; i += 64 * NW) {
                    const int b = i / (some * LPR), in = i - b * some * LPR, q = in / LPR, c = (in % LPR) * 8;   // the head among the workgroup's
                    float M = kPagedNegInf;
#pragma unroll
                    for (int y = 0; y < KW; ++y) M = fmaxf(M, ml[y * HW + b][q].x);
                    const float mu = M == kPagedNegInf ? 0.f : M;
                    float L = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
                    for (int y = 0; y < KW; ++y) {
                        const float2 z = ml[y * HW + b][q];
                        const float f = exp2_fast(z.x - mu);
                        L += z.y * f;
                        const float* op = reinterpret_cast<const float*>(lds + (y * HW + b) * kWave) + q * OLD + c;
#pragma unroll
                        for (int e = 0; e < 8; ++e) o[e] += op[e] * f;
                    }
                    if (whole) {
                        const float inv = L == 0.f ? 0.f : 1.f / L;
                        const int64_t at = (int64_t)r * a.H + (h - hw + b) * G + q0 + x * kPagedCols + q;
#pragma unroll
                        for (int e = 0; e < 8; ++e) o[e] = L == 0.f ? 0.f : o[e] * inv;
                        st16(a.o + at * D + c, pack8(o));
                        if (a.lse && c == 0) a.lse[at] = L == 0.f ? kPagedNegInf : (M + log2_fast(L)) * kLn2;
                    } else {
                        float* u = pieces + b * per;
                        *reinterpret_cast<float4*>(u + (x * kPagedCols + q) * D + c) = make_float4(o[0], o[1], o[2], o[3]);
                        *reinterpret_cast<float4*>(u + (x * kPagedCols + q) * D + c + 4) = make_float4(o[4], o[5], o[6], o[7]);
                        if (c == 0) *reinterpret_cast<float2*>(u + (int64_t)plan.gt * D + 2 * (x * kPagedCols + q)) = make_float2(M, L);
                    }
                }
            }
        }
        if (plan.split == 0) return;
        if (KW > 1) __syncthreads();   // before the next segment's values are written
        pos += n;
        s0 = 0;
        if (++hr == heads) hr = 0, ++r;
    }
}

// Join the pieces of a row and query head: a wave each, D / 4 lanes of it for a piece.
template <int D>
__global__ void __launch_bounds__(256) paged_join_kernel(PagedArgs a, PagedPlan plan) {
    constexpr int LPR = D / 4, NS = 64 / LPR;   // pieces read side by side
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int G = a.H / a.Hkv, sets = a.Hkv / plan.hw, heads = plan.groups * sets;
    const int64_t at = (int64_t)blockIdx.x * 4 + w;
    if (at >= (int64_t)a.R * a.H) return;
    const int r = (int)(at / a.H), hq = (int)(at - (int64_t)r * a.H), h = hq / G, q = hq - h * G, grp = q / plan.gt, rr = q - grp * plan.gt;
    const uint2 place = paged_places(a, plan)[(int64_t)r * heads + grp * sets + h / plan.hw];
    const uint32_t count = place.y;
    if (count == 1) return;   // written by its workgroup
    const int64_t per = paged_piece(plan, D);
    const int st = lane / LPR, c = (lane % LPR) * 4;
    float M = kPagedNegInf, L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    auto join = [&](float m, float l, const float4& x) {
        const float mn = fmaxf(M, m), mu = mn == kPagedNegInf ? 0.f : mn;
        const float f = exp2_fast(M - mu), fx = exp2_fast(m - mu);
        L = L * f + l * fx;
        o.x = o.x * f + x.x * fx;
        o.y = o.y * f + x.y * fx;
        o.z = o.z * f + x.z * fx;
        o.w = o.w * f + x.w * fx;
        M = mn;
    };
    constexpr int U = 4;   // pieces of a lane in flight
    for (uint32_t u = st; u < count; u += NS * U) {
        float2 z[U];
        float4 x[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const uint32_t k = min(u + i * NS, count - 1);
            const float* p = a.work + ((2 * (int64_t)(place.x + k) + (k == 0)) * plan.hw + h % plan.hw) * per;
            z[i] = *reinterpret_cast<const float2*>(p + (int64_t)plan.gt * D + 2 * rr);
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
    if (lane >= LPR) return;
    const float inv = L == 0.f ? 0.f : 1.f / L;
    uint2 out;
    out.x = L == 0.f ? 0u : pack_bf16x2(o.x * inv, o.y * inv);
    out.y = L == 0.f ? 0u : pack_bf16x2(o.z * inv, o.w * inv);
    *reinterpret_cast<uint2*>(a.o + at * D + c) = out;
    if (a.lse && lane == 0) a.lse[at] = L == 0.f ? kPagedNegInf : (M + log2_fast(L)) * kLn2;
}

// Launch shape.  One round of CUs: with two workgroups a CU 134 us for 130 (64 rows of up to 6,000 tokens), 102 for 98
// (long rows).
static PagedPlan paged_plan(int32_t R, int32_t H, int32_t Hkv, int32_t N, int32_t M, int32_t shift, int32_t D) {
    PagedPlan p{};
    const int G = H / Hkv;
    const int tiles = G <= kPagedCols ? 1 : 2;
    p.gt = G < kPagedCols * tiles ? G : kPagedCols * tiles;
    p.groups = (G + p.gt - 1) / p.gt;
    const int64_t keys = (int64_t)M << shift;
    p.hw = 1, p.kw = paged_wide(D, tiles) ? 4 : 8;
    const int64_t pages = (int64_t)R * M < N ? (int64_t)R * M : N;
    p.once = (pages << shift) * Hkv * D * 4 >= (int64_t)256 << 20;
    if (keys <= 6 * 8 * kPagedTile) return p;
    p.hw = Hkv % 4 == 0 ? 4 : Hkv % 2 == 0 ? 2 : 1;
    p.kw = 4 / p.hw;
    const int64_t steps = (keys + kPagedTile * p.kw - 1) / (kPagedTile * p.kw), all = steps * R * (Hkv / p.hw) * p.groups, most = device_cus();
    p.split = (int32_t)(all < most ? all : most);
    return p;
}

int64_t paged_attention_workspace(int32_t R, int32_t H, int32_t Hkv, int32_t N, int32_t M, int32_t shift, int32_t D) {
    if (R < 1 || Hkv < 1 || H < Hkv || H % Hkv || N < 1 || M < 1 || shift < 4 || shift > 20 || (D != 64 && D != 128)) return 0;
    const PagedPlan p = paged_plan(R, H, Hkv, N, M, shift, D);
    return p.split == 0 ? 0 : 2 * (int64_t)p.split * p.hw * paged_piece(p, D) * (int64_t)sizeof(float) + (int64_t)R * (Hkv / p.hw) * p.groups * (int64_t)sizeof(uint2);
}

template <int D, int NT, bool ONCE>
static void paged_launch(const PagedArgs& a, const PagedPlan& p, hipStream_t st) {
    const dim3 grid((unsigned)(p.split ? p.split : a.R * a.Hkv * p.groups)), block(64 * p.hw * p.kw);
    if constexpr (!paged_wide(D, NT))
        if (p.kw == 8) {
            hipLaunchKernelGGL((paged_attn_kernel<D, NT, 1, 8, ONCE>), grid, block, 0, st, a, p);
            return;
        }
    if (p.hw == 4) hipLaunchKernelGGL((paged_attn_kernel<D, NT, 4, 1, ONCE>), grid, block, 0, st, a, p);
    else if (p.hw == 2) hipLaunchKernelGGL((paged_attn_kernel<D, NT, 2, 2, ONCE>), grid, block, 0, st, a, p);
    else hipLaunchKernelGGL((paged_attn_kernel<D, NT, 1, 4, ONCE>), grid, block, 0, st, a, p);
}

template <int D>
static int paged_launch(const PagedArgs& a, const PagedPlan& p, hipStream_t st) {
    if (p.gt <= kPagedCols) p.once ? paged_launch<D, 1, true>(a, p, st) : paged_launch<D, 1, false>(a, p, st);
    else p.once ? paged_launch<D, 2, true>(a, p, st) : paged_launch<D, 2, false>(a, p, st);
    if (int e = check_launch("paged_attention")) return e;
    if (p.split == 0) return 0;
    hipLaunchKernelGGL((paged_join_kernel<D>), dim3((unsigned)(((int64_t)a.R * a.H + 3) / 4)), dim3(256), 0, st, a, p);
    return check_launch("paged_attention_join");
}

int paged_attention(const PagedArgs& a, void* stream) {
    FX_REQUIRE(a.D == 64 || a.D == 128, "paged_attention: head_dim %d not supported (64 or 128)", a.D);
    FX_REQUIRE(a.R >= 1 && a.M >= 1 && a.N >= 1 && a.Hkv >= 1 && a.H >= a.Hkv && a.H % a.Hkv == 0,
               "paged_attention: bad shape R=%d H=%d Hkv=%d M=%d N=%d", a.R, a.H, a.Hkv, a.M, a.N);
    FX_REQUIRE(a.shift >= 4 && a.shift <= 20, "paged_attention: pages of 2^%d rows (16 to 2^20)", a.shift);
    FX_REQUIRE(((int64_t)a.M << a.shift) <= 0x7fffffff - 128, "paged_attention: a table of %d pages of 2^%d rows is too wide", a.M, a.shift);
    FX_REQUIRE(a.q && a.k && a.v && a.table && a.lens && a.o, "paged_attention: null pointer");
    FX_REQUIRE((a.knew == nullptr) == (a.vnew == nullptr), "paged_attention: knew and vnew go together");
    FX_REQUIRE(a.scale > 0.f && a.scale < __builtin_huge_valf(), "paged_attention: scale %g must be positive and finite", (double)a.scale);
    const int64_t s[] = {a.qr, a.qh, a.kp, a.kt, a.kh, a.vp, a.vt, a.vh, a.knr, a.knh, a.vnr, a.vnh};
    for (int64_t x : s) FX_REQUIRE(x % 8 == 0, "paged_attention: strides must be multiples of 8 elements");
    for (int64_t x : {a.kt, a.vt})
        FX_REQUIRE(x >= 0 && x < (int64_t)1 << 23, "paged_attention: rows of a page %lld elements apart", (long long)x);
    FX_REQUIRE((((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.o | (uintptr_t)a.work | (uintptr_t)a.knew |
                 (uintptr_t)a.vnew) & 15) == 0,
               "paged_attention: q, k, v, o, work, knew and vnew must be 16-byte aligned");
    const PagedPlan p = paged_plan(a.R, a.H, a.Hkv, a.N, a.M, a.shift, a.D);
    const int64_t pairs = (int64_t)a.R * a.Hkv * p.groups;
    const int64_t steps = (((int64_t)a.M << a.shift) + kPagedTile * p.kw - 1) / (kPagedTile * p.kw);
    // a launch has less than 2^32 work items; all rows' steps are counted in 32 bits, and so is a row's place among those of its heads
    FX_REQUIRE(pairs < (1 << 23) && (int64_t)a.R * a.H < (1 << 25) && a.R * steps < 0x7fffffffLL && steps * p.groups * (a.Hkv / p.hw) <= 0xffffffffLL,
               "paged_attention: too many rows and heads");
    FX_REQUIRE(p.split == 0 || a.work, "paged_attention: null workspace");
    return a.D == 64 ? paged_launch<64>(a, p, (hipStream_t)stream) : paged_launch<128>(a, p, (hipStream_t)stream);
}

}  // namespace fx
