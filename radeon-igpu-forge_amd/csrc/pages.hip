// The tables of a paged key-value cache, for gfx950: pages for tokens that rows are about to add and
// the slots of those tokens, rows that go on from other rows, and prompts' keys and values into their slots.
//
// A page's uses count the rows that hold it; a page without uses is free.  Everything is a function of
// the tables alone: the free pages are taken from the lowest on, in the rows' order, and what a page's
// holders do to its uses are sums of whole numbers, so no result hangs on the order of workgroups.
#include "fx_device.h"
#include "fx_internal.h"

namespace fx {

constexpr int kPagesThreads = 1024, kPagesWaves = kPagesThreads / 64;
constexpr int kPagesScan = 16;   // pages a thread looks through at a time

__device__ __forceinline__ int pages_len(int n, int M, int shift) {
    const int64_t most = (int64_t)M << shift;
    return n < 0 ? 0 : n < most ? n : (int)most;
}
__device__ __forceinline__ int pages_of(int64_t n, int shift) { return (int)((n + (1 << shift) - 1) >> shift); }

// a value of every thread summed over the threads before it, and the workgroup's sum
__device__ __forceinline__ int block_before(int v, int* sh, int& sum) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int up = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int o = __shfl_up(up, off, 64);
        if (lane >= off) up += o;
    }
    __syncthreads();   // the last use of sh is over
    if (lane == 63) sh[w] = up;
    __syncthreads();
    int before = 0;
    sum = 0;
#pragma unroll
    for (int i = 0; i < kPagesWaves; ++i) {
        const int x = sh[i];
        if (i < w) before += x;
        sum += x;
    }
    return before + up - v;
}

// ---- extend ------------------------------------------------------------------------------
//
// Row r wants ceil((len + add) / P) - ceil(len / P) pages, and one more in place of its open page (the
// last one, where len is no multiple of P) if it may not write there: if more rows hold the page than
// are about to write into it, none may; else the one with the most tokens there may, the lowest of equals:
// it writes behind all of the others' tokens, so that one which is refused a page, and still holds this one, loses none.
// A row that wants some gets them if all rows' wants up to and with its own do not exceed the free pages; else it gets nothing.
//
// One workgroup, bounded by its chain of round trips: lengths, open pages, their uses, tables.  A thread has up to eight
// rows in registers.  The first pages' uses are under way meanwhile; free ones are looked for only as far as they are wanted.
// 40 rows of beams 6.2 us and 4.5 for the copies in 24 pools; 48 prompts, about 3,100 pages among 65,536, 8.0 and 2.8 for the slots.

// the workspace: a copy for each row, the page each wanted one is, and, of many rows that may have copies, for each page (the writer
// that may keep it, writers)
__device__ __forceinline__ int32_t* extend_list(const ExtendArgs& a) { return a.work + 4 * (int64_t)a.R; }

// the slot of row r's j-th new token, once its pages are in the table and its copy's entry says that it was served: then
// its tokens lie in the table with all of the new ones (a refused row's length may be anything)
__device__ __forceinline__ int64_t slot_of(const ExtendArgs& a, int r, int j) {
    if (j >= a.add[r] || !reinterpret_cast<const int4*>(a.work)[r].w) return -1;
    const int pos = max(a.lens[r], 0) + j;
    return ((int64_t)a.table[(int64_t)r * a.tab + (pos >> a.shift)] << a.shift) + (pos & ((1 << a.shift) - 1));
}

constexpr int kPagesFew = 256;                           // rows that are compared with one another in LDS

// Large pools (from kPagesCounted on) have their free pages counted first, a turn's kPagesThreads kPagesScan pages a workgroup, so that
// turns without any are passed over: of 1,000,000 pages with free ones at the end alone 92 us by one workgroup, 11 so.
constexpr int kPagesTurn = kPagesThreads * kPagesScan, kPagesCounted = 1 << 18;

__global__ void __launch_bounds__(kPagesThreads) count_kernel(const int32_t* uses, int N, int32_t* counts) {
    __shared__ int sh[kPagesWaves];
    const int off = (int)((reinterpret_cast<uintptr_t>(uses) >> 2) & 3), p = blockIdx.x * kPagesTurn + (int)threadIdx.x * kPagesScan - off;
    int n = 0;
    if (p >= 0 && p + kPagesScan <= N) {
#pragma unroll
        for (int i = 0; i < kPagesScan / 4; ++i) {
            const int4 u = *reinterpret_cast<const int4*>(uses + p + 4 * i);
            n += (u.x == 0) + (u.y == 0) + (u.z == 0) + (u.w == 0);
        }
    } else {
        for (int i = max(0, -p); i < min(kPagesScan, N - p); ++i) n += uses[p + i] == 0;
    }
    int sum;
    block_before(n, sh, sum);
    if (threadIdx.x == 0) counts[blockIdx.x] = sum;
}

template <int kPagesEach, bool COUNTED>   // rows of a thread, whether `counts` are given
__global__ void __launch_bounds__(kPagesThreads) extend_kernel(ExtendArgs a, int64_t list, const int32_t* counts, bool slots_too) {
    __shared__ __attribute__((aligned(8))) int32_t pre[kPagesRows + 1], col0[kPagesRows];   // pages wanted before a row, and the column of its first
    __shared__ int sh[kPagesWaves];
    int4* copies = reinterpret_cast<int4*>(a.work);
    int32_t *pages = extend_list(a), *writers = pages + list;
    const int tid = threadIdx.x, mask = (1 << a.shift) - 1;
    const int off = (int)((reinterpret_cast<uintptr_t>(a.uses) >> 2) & 3);   // 16-byte loads at their addresses

    // This thread's pages of a turn, kPagesScan from place(turn) on, and the turns that have free pages (all, where these were
    // not counted), 64 looked up at a time by every wave.
    const int turns = (a.N + off + kPagesTurn - 1) / kPagesTurn;
    auto place = [&](int turn) { return turn * kPagesTurn - off + tid * kPagesScan; };
    auto whole = [&](int p) { return p >= 0 && p + kPagesScan <= a.N; };
    int window = -64;
    uint64_t live = 0;
    int turn = -1;
    auto next = [&] {
        if (!COUNTED) return turn + 1 < turns ? turn + 1 : -1;
        while (live == 0) {
            window += 64;
            if (window >= turns) return -1;
            const int t = window + (tid & 63);
            live = __ballot(t < turns && counts[t] > 0);
        }
        const int t = window + __ffsll((unsigned long long)live) - 1;
        live &= live - 1;
        return t;
    };
    constexpr bool kAhead = kPagesEach == 1;   // the first turn's uses before all else (eight rows take the registers)
    int4 ahead[kPagesScan / 4];
    auto look = [&](int turn) {
        const int p = place(turn);
        if (turn >= 0 && whole(p))
#pragma unroll
            for (int i = 0; i < kPagesScan / 4; ++i) ahead[i] = *reinterpret_cast<const int4*>(a.uses + p + 4 * i);
    };
    if (kAhead) turn = next(), look(turn);

    int len[kPagesEach], add[kPagesEach], open[kPagesEach];   // a row's tokens, the new ones it may have, its open page (-1: none)
    bool copy[kPagesEach], any = false;
#pragma unroll
    for (int e = 0; e < kPagesEach; ++e) {
        const int r = e * kPagesThreads + tid;
        len[e] = add[e] = 0;
        open[e] = -1;
        copy[e] = false;
        if (r < a.R) len[e] = pages_len(a.lens[r], a.M, a.shift), add[e] = min(max(a.add[r], 0), a.most);
        if ((int64_t)len[e] + add[e] > (int64_t)a.M << a.shift) add[e] = 0;
    }
#pragma unroll
    for (int e = 0; e < kPagesEach; ++e)
        if (add[e] > 0 && (len[e] & mask)) {
            open[e] = a.table[(int64_t)(e * kPagesThreads + tid) * a.tab + (len[e] >> a.shift)];
            if ((uint32_t)open[e] >= (uint32_t)a.N) add[e] = 0;
        }
    int users[kPagesEach];
#pragma unroll
    for (int e = 0; e < kPagesEach; ++e) {
        users[e] = add[e] > 0 && (len[e] & mask) ? a.uses[open[e]] : 0;
        if (users[e] > 1 && !a.copies) add[e] = 0;
        any |= users[e] > 1 && add[e] > 0;
    }
    auto shares = [&](int e) { return users[e] > 1 && add[e] > 0; };
    if (__syncthreads_or(any)) {
        // who else writes into a row's open page: those that would rather keep it (a lower number: more tokens there, then a lower row), and all
        auto order = [&](int e) { return (mask - (len[e] & mask)) * kPagesRows + e * kPagesThreads + tid; };
        if (kPagesEach == 1 && a.R <= kPagesFew) {
            int before = 0, writes = 0;
            int2* const writer = reinterpret_cast<int2*>(pre);   // (page, order)
            const int mine = order(0);
            if (tid < a.R) writer[tid] = make_int2(shares(0) ? open[0] : -1, mine);
            __syncthreads();
            if (shares(0))
#pragma unroll 8
                for (int r = 0; r < a.R; ++r) {
                    const int2 o = writer[r];
                    writes += o.x == open[0];
                    before += (o.x == open[0]) & (o.y < mine);
                }
            copy[0] = shares(0) && (writes < users[0] || before > 0);
            __syncthreads();   // pre is used again
        } else {
#pragma unroll
            for (int e = 0; e < kPagesEach; ++e)
                if (shares(e)) writers[2 * (int64_t)open[e]] = 0x7fffffff, writers[2 * (int64_t)open[e] + 1] = 0;
            __syncthreads();
#pragma unroll
            for (int e = 0; e < kPagesEach; ++e)
                if (shares(e)) {
                    atomicMin(&writers[2 * (int64_t)open[e]], order(e));
                    atomicAdd(&writers[2 * (int64_t)open[e] + 1], 1);
                }
            __syncthreads();
#pragma unroll
            for (int e = 0; e < kPagesEach; ++e)
                if (shares(e)) {
                    const int first = __hip_atomic_load(&writers[2 * (int64_t)open[e]], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    const int count = __hip_atomic_load(&writers[2 * (int64_t)open[e] + 1], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    copy[e] = count < users[e] || order(e) != first;
                }
        }
    }

    int want = 0;   // of all rows so far
    int need[kPagesEach];
#pragma unroll
    for (int e = 0; e < kPagesEach; ++e) {
        need[e] = 0;
        if (e * kPagesThreads >= a.R) continue;
        const int r = e * kPagesThreads + tid, had = pages_of(len[e], a.shift);
        if (add[e] > 0) need[e] = pages_of((int64_t)len[e] + add[e], a.shift) - had + copy[e];
        int sum;
        const int begin = want + block_before(need[e], sh, sum);
        if (r < a.R) pre[r] = begin, col0[r] = had - copy[e];
        want += sum;
    }
    if (tid == 0) pre[a.R] = want;

    int have = 0;   // free pages found, up to `want`
    if (!kAhead) turn = next(), look(turn);
    while (turn >= 0 && have < want) {
        const int p = place(turn);
        uint32_t free = 0;
        if (whole(p)) {
#pragma unroll
            for (int i = 0; i < kPagesScan / 4; ++i) {
                const int4 u = ahead[i];
                free |= (uint32_t)((u.x == 0) | (u.y == 0) << 1 | (u.z == 0) << 2 | (u.w == 0) << 3) << (4 * i);
            }
        } else {
            for (int i = max(0, -p); i < min(kPagesScan, a.N - p); ++i) free |= (uint32_t)(a.uses[p + i] == 0) << i;
        }
        turn = next();
        look(turn);   // behind this turn's sums
        int sum;
        int at = have + block_before(__popc(free), sh, sum);
        for (; free && at < want; ++at) {
            const int i = __ffs(free) - 1;
            pages[at] = p + i;
            free &= free - 1;
        }
        have += sum;
    }
    __syncthreads();

    // rows: their copies, lengths and, of single tokens, slots
#pragma unroll
    for (int e = 0; e < kPagesEach; ++e) {
        const int r = e * kPagesThreads + tid;
        if (r >= a.R) continue;
        const bool ok = add[e] > 0 && (need[e] == 0 || pre[r] + need[e] <= have);
        const int got = ok && need[e] > 0 ? pages[pre[r]] : -1;
        copies[r] = ok && copy[e] ? make_int4(open[e], got, len[e] & mask, 1) : make_int4(0, 0, 0, ok);
        if (ok && copy[e]) atomicAdd(&a.uses[open[e]], -1);
        a.out[r] = ok ? len[e] + add[e] : a.lens[r];
        if (a.most == 1) a.slots[r] = ok ? ((int64_t)(need[e] > 0 ? got : open[e]) << a.shift) + (len[e] & mask) : -1;
    }
    // new pages, each by the thread whose turn it is: its row is the last one that begins at or before it
    for (int i = tid; i < min(want, have); i += kPagesThreads) {
        int lo = 0, hi = a.R - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (pre[mid] <= i) lo = mid;
            else hi = mid - 1;
        }
        if (pre[lo + 1] > have) continue;
        a.table[(int64_t)lo * a.tab + col0[lo] + i - pre[lo]] = pages[i];
        a.uses[pages[i]] = 1;
    }
    if (!slots_too || a.most == 1) return;
    __syncthreads();
    for (int i = tid; i < a.R * a.most; i += kPagesThreads) a.slots[i] = slot_of(a, i / a.most, i % a.most);
}

// the slots of longer additions
__global__ void __launch_bounds__(256) slots_kernel(ExtendArgs a) {
    const int r = blockIdx.x;
    // (64 bits: `most` may be the largest int)
    for (int64_t j = blockIdx.y * 256 + threadIdx.x; j < a.most; j += gridDim.y * 256) a.slots[(int64_t)r * a.most + j] = slot_of(a, r, (int)j);
}

// pages that rows can want between them, in whole int4
static int64_t extend_most(int32_t R, int32_t M, int32_t N, int32_t shift, int32_t most) {
    const int64_t each = ((int64_t)most >> shift) + 3, all = (each < M + 1 ? each : M + 1) * (int64_t)R;
    return ((all < N ? all : N) + 3) & ~3ll;
}

// (the kernel of eight rows a thread has one form: its registers do not take the other)
static bool pages_counted(int32_t R, int32_t N) { return N >= kPagesCounted || R > kPagesThreads; }

static int64_t extend_writers(int32_t R, int32_t N, bool copies) { return copies && R > kPagesFew ? 2 * (int64_t)N : 0; }

int64_t extend_pages_workspace(int32_t R, int32_t M, int32_t N, int32_t shift, int32_t most, bool copies) {
    if (R < 1 || M < 1 || N < 1 || shift < 0 || shift > 18 || most < 1) return 0;
    return (4 * (int64_t)R + extend_most(R, M, N, shift, most) + extend_writers(R, N, copies) +
            (pages_counted(R, N) ? ((int64_t)N + 3) / kPagesTurn + 1 : 0)) * (int64_t)sizeof(int32_t);
}

int extend_pages(const ExtendArgs& a, void* stream) {
    FX_REQUIRE(a.R >= 1 && a.R <= kPagesRows, "extend_pages: %d rows (1 to %d)", a.R, kPagesRows);
    // (2^18 rows of a page times kPagesRows are the most that order() takes)
    FX_REQUIRE(a.M >= 1 && a.N >= 1 && a.most >= 1 && a.shift >= 0 && a.shift <= 18, "extend_pages: bad shape M=%d N=%d most=%d shift=%d", a.M, a.N,
               a.most, a.shift);
    FX_REQUIRE(((int64_t)a.M << a.shift) <= 0x7fffffff - 128 && (int64_t)a.R * a.M < 0x7fffffff, "extend_pages: a table of %d x %d pages is too large", a.R, a.M);
    FX_REQUIRE(a.N <= 1 << 30, "extend_pages: %d pages are too many", a.N);
    FX_REQUIRE(a.table && a.uses && a.lens && a.add && a.slots && a.out && a.work, "extend_pages: null pointer");
    FX_REQUIRE(((uintptr_t)a.work & 15) == 0, "extend_pages: work must be 16-byte aligned");
    const bool one = (int64_t)a.R * a.most <= 8 * kPagesThreads;   // slots in the same launch
    const int64_t list = extend_most(a.R, a.M, a.N, a.shift, a.most);
    int32_t* counts = nullptr;
    if (pages_counted(a.R, a.N)) {
        counts = a.work + 4 * (int64_t)a.R + list + extend_writers(a.R, a.N, a.copies);
        const int off = (int)((reinterpret_cast<uintptr_t>(a.uses) >> 2) & 3);
        hipLaunchKernelGGL(count_kernel, dim3((unsigned)((a.N + off + kPagesTurn - 1) / kPagesTurn)), dim3(kPagesThreads), 0, (hipStream_t)stream, a.uses, a.N,
                           counts);
        if (int e = check_launch("extend_pages_count")) return e;
    }
    auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(1), dim3(kPagesThreads), 0, (hipStream_t)stream, a, list, counts, one);
    };
    constexpr int kMost = kPagesRows / kPagesThreads;
    if (a.R > kPagesThreads) launch(extend_kernel<kMost, true>);
    else counts ? launch(extend_kernel<1, true>) : launch(extend_kernel<1, false>);
    if (int e = check_launch("extend_pages")) return e;
    if (one) return 0;
    const int y = (a.most - 1) / 1024 + 1;
    hipLaunchKernelGGL(slots_kernel, dim3((unsigned)a.R, (unsigned)(y < 64 ? y : 64)), dim3(256), 0, (hipStream_t)stream, a);
    return check_launch("extend_pages_slots");
}

__global__ void __launch_bounds__(256) copy_pages_kernel(CopyPagesArgs a) {
    const int4 c = reinterpret_cast<const int4*>(a.copies)[blockIdx.x];
    const int t = blockIdx.y, per = a.D / 8, n = c.z * a.H * per;
    uint16_t *const from = a.at[t] + c.x * a.sp[t], *const to = a.at[t] + c.y * a.sp[t];
    constexpr int U = 4;
    for (int i0 = threadIdx.x; i0 < n; i0 += 256 * U) {
        uint4 x[U];
        int64_t in[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = min(i0 + 256 * u, n - 1), d = i % per, hj = i / per, h = hj % a.H, j = hj / a.H;
            in[u] = (int64_t)j * a.st[t] + (int64_t)h * a.sh[t] + d * 8;
            x[u] = ld16(from + in[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + 256 * u < n) st16(to + in[u], x[u]);
    }
}

int copy_pages(const CopyPagesArgs& a, void* stream) {
    FX_REQUIRE(a.R >= 1 && a.R <= kPagesRows && a.count >= 1 && a.count <= kCopyTensors && a.H >= 1 && a.D >= 8 && a.D % 8 == 0 && a.copies,
               "copy_pages: bad arguments");
    hipLaunchKernelGGL(copy_pages_kernel, dim3((unsigned)a.R, (unsigned)a.count), dim3(256), 0, (hipStream_t)stream, a);
    return check_launch("copy_pages");
}

// ---- store -------------------------------------------------------------------------------
//
// HBM-bound: every new row is read once and written once, a thread a 16-byte piece of a key and of its value.  The stores go past
// the caches (24 prompts of up to 4,001 tokens, 525 MB: 98 us without, 90 with, 5.8 TB/s); the loads do not: what a projection
// has just written is still there (33 MB 7.1 us, past them 8.8).  More pieces a thread are the slower: two 91 us, eight 111.

__global__ void __launch_bounds__(256) store_pages_kernel(StorePagesArgs a) {
    const int per = a.D / 8, units = a.H * per, i = blockIdx.x * 256 + threadIdx.x;
    if (i >= a.T * units) return;
    const int r = blockIdx.y, t = i / units, e = i - t * units, h = e / per, d = (e - h * per) * 8;
    const int64_t slot = a.slots[r * a.sr + t * a.st];
    if (slot < 0 || slot >= a.N << a.shift) return;
    const uint4 k = ld16(a.k + r * a.kr + t * a.kt + h * a.kh + d), v = ld16(a.v + r * a.vr + t * a.vt + h * a.vh + d);
    const int64_t page = slot >> a.shift, j = slot & ((1 << a.shift) - 1);
    st16_nt(a.kp + page * a.kpp + j * a.kpt + h * a.kph + d, k);
    st16_nt(a.vp + page * a.vpp + j * a.vpt + h * a.vph + d, v);
}

int store_pages(const StorePagesArgs& a, void* stream) {
    FX_REQUIRE(a.R >= 1 && a.T >= 1 && a.H >= 1 && a.N >= 1 && a.D >= 8 && a.D % 8 == 0 && a.shift >= 0 && a.shift <= 20,
               "store_pages: bad shape R=%d T=%d H=%d D=%d N=%lld shift=%d", a.R, a.T, a.H, a.D, (long long)a.N, a.shift);
    FX_REQUIRE(a.k && a.v && a.slots && a.kp && a.vp, "store_pages: null pointer");
    const int64_t s[] = {a.kr, a.kt, a.kh, a.vr, a.vt, a.vh, a.kpp, a.kpt, a.kph, a.vpp, a.vpt, a.vph};
    for (int64_t x : s) FX_REQUIRE(x % 8 == 0, "store_pages: strides must be multiples of 8 elements");
    FX_REQUIRE((((uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.kp | (uintptr_t)a.vp) & 15) == 0, "store_pages: 16-byte aligned tensors");
    const int64_t n = (int64_t)a.T * a.H * (a.D / 8);
    FX_REQUIRE(n <= 0x7fffff00 && a.R <= 65535, "store_pages: %d rows of %d x %d x %d are too many", a.R, a.T, a.H, a.D);
    hipLaunchKernelGGL(store_pages_kernel, dim3((unsigned)((n + 255) / 256), (unsigned)a.R), dim3(256), 0, (hipStream_t)stream, a);
    return check_launch("store_pages");
}

// ---- reorder -----------------------------------------------------------------------------
//
// A workgroup a few columns of the table, for all rows at once: what the rows held is in LDS before
// any of it is overwritten, so it is done in place.  A page that row p held is now held by as many rows as went on from
// p: its uses change by one less than that.  Bounded by its chain of round trips (lengths, entries, and
// what is written) up to some megabytes of table: 40 rows of 64 pages 3.8 us, 500 of 2,048 9.6.

constexpr int kReorderLds = 32768;   // ints: two a row, and its columns

__global__ void __launch_bounds__(kPagesThreads) reorder_kernel(ReorderArgs a, int cols) {
    __shared__ int32_t lds[kReorderLds];
    int32_t *parent = lds, *state = lds + a.R, *was = state + a.R;   // state: the row's columns here, and 64 times the rows that go on from it
    const int C = 1 << cols, c0 = blockIdx.x * C, threads = blockDim.x;
    bool any = false;
    for (int r = threadIdx.x; r < a.R; r += threads) {
        const int p = a.parents[r], n = min(max(pages_of(pages_len(a.lens[r], a.M, a.shift), a.shift) - c0, 0), C);
        parent[r] = (uint32_t)p < (uint32_t)a.R ? p : -1;
        state[r] = n;
        any |= n > 0;
        if (blockIdx.x == 0) a.out[r] = (uint32_t)p < (uint32_t)a.R ? pages_len(a.lens[p], a.M, a.shift) : 0;
    }
    any = __syncthreads_or(any);
    if (!any) return;   // no row has a page here
    __syncthreads();
    for (int r = threadIdx.x; r < a.R; r += threads)
        if (parent[r] >= 0) atomicAdd(&state[parent[r]], 64);
    const int n = a.R << cols;
    constexpr int U = 4;
    for (int i0 = threadIdx.x; i0 < n; i0 += threads * U) {
        int x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * threads, r = i >> cols, c = i & (C - 1);
            x[u] = i < n && c < (state[r] & 63) ? a.table[(int64_t)r * a.tab + c0 + c] : -1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + u * threads < n) was[i0 + u * threads] = x[u];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += threads) {
        const int r = i >> cols, c = i & (C - 1), s = state[r];
        if (c < (s & 63) && s >> 6 != 1) {
            const int p = was[i];
            if ((uint32_t)p < (uint32_t)a.N) atomicAdd(&a.uses[p], (s >> 6) - 1);
        }
        const int from = parent[r];
        if (from >= 0 && from != r && c < (state[from] & 63)) a.table[(int64_t)r * a.tab + c0 + c] = was[(from << cols) + c];
    }
}

int reorder_pages(const ReorderArgs& a, void* stream) {
    FX_REQUIRE(a.R >= 1 && a.R <= kPagesRows, "reorder_pages: %d rows (1 to %d)", a.R, kPagesRows);
    FX_REQUIRE(a.M >= 1 && a.N >= 1 && a.shift >= 0 && a.shift <= 20 && ((int64_t)a.M << a.shift) <= 0x7fffffff - 128,
               "reorder_pages: bad shape M=%d N=%d shift=%d", a.M, a.N, a.shift);
    FX_REQUIRE(a.table && a.uses && a.lens && a.parents && a.out, "reorder_pages: null pointer");
    int cols = 3;
    while ((int64_t)a.R * ((1 << cols) + 2) > kReorderLds) --cols;
    const int64_t n = (int64_t)a.R << cols;
    hipLaunchKernelGGL(reorder_kernel, dim3((unsigned)((a.M + (1 << cols) - 1) >> cols)), dim3(n <= 512 ? 256 : kPagesThreads), 0, (hipStream_t)stream, a, cols);
    return check_launch("reorder_pages");
}

}  // namespace fx
