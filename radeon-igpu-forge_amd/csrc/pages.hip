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
// are about to write into it, none may; else the lowest of them may.  A row that wants some gets them if
// all rows' wants up to and with its own do not exceed the free pages; else it gets nothing.
//
// One workgroup, bounded by its chain of round trips: lengths, open pages, their uses, who writes there, free
// pages, tables.  The free pages are looked for only as far as they are wanted.

// the workspace: a copy for each row, the page each wanted one is, and for each page (first writer, writers)
__device__ __forceinline__ int32_t* extend_list(const ExtendArgs& a) { return a.work + 4 * (int64_t)a.R; }

enum : uint8_t { kRowWants = 1, kRowCopies = 2, kRowShares = 4 };

__device__ __forceinline__ int64_t slot_of(const ExtendArgs& a, int r, int64_t pos) {
    return ((int64_t)a.table[(int64_t)r * a.tab + (pos >> a.shift)] << a.shift) + (pos & ((1 << a.shift) - 1));
}

__global__ void __launch_bounds__(kPagesThreads) extend_kernel(ExtendArgs a, int64_t list, bool slots_too) {
    extern __shared__ int32_t lds[];   // pre[R + 1], flags[R]
    __shared__ int sh[kPagesWaves];
    int32_t* pre = lds;
    uint8_t* flags = reinterpret_cast<uint8_t*>(lds + a.R + 1);
    int4* copies = reinterpret_cast<int4*>(a.work);
    int32_t *pages = extend_list(a), *writers = pages + list;
    const int tid = threadIdx.x, mask = (1 << a.shift) - 1;

    auto length = [&](int r) { return pages_len(a.lens[r], a.M, a.shift); };
    auto adds = [&](int r) { return min(max(a.add[r], 0), a.most); };
    auto open_page = [&](int r, int len) { return a.table[(int64_t)r * a.tab + (len >> a.shift)]; };

    bool any = false;
    for (int r = tid; r < a.R; r += kPagesThreads) {
        const int len = length(r), add = adds(r);
        uint8_t f = add > 0 && (int64_t)len + add <= (int64_t)a.M << a.shift ? kRowWants : 0;
        if (f && (len & mask)) {
            const int p = open_page(r, len);
            if ((uint32_t)p >= (uint32_t)a.N) f = 0;
            else if (a.uses[p] > 1) {
                f = a.copies ? f | kRowShares : 0;
                if (f) writers[2 * (int64_t)p] = 0x7fffffff, writers[2 * (int64_t)p + 1] = 0;
            }
        }
        flags[r] = f;
        any |= (f & kRowShares) != 0;
    }
    any = __syncthreads_or(any);
    __syncthreads();   // what was written to memory is there
    if (any) {
        for (int r = tid; r < a.R; r += kPagesThreads)
            if (flags[r] & kRowShares) {
                const int64_t p = open_page(r, length(r));
                atomicMin(&writers[2 * p], r);
                atomicAdd(&writers[2 * p + 1], 1);
            }
        __syncthreads();
        for (int r = tid; r < a.R; r += kPagesThreads)
            if (flags[r] & kRowShares) {
                const int64_t p = open_page(r, length(r));
                const int first = __hip_atomic_load(&writers[2 * p], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                const int count = __hip_atomic_load(&writers[2 * p + 1], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                if (count < a.uses[p] || r != first) flags[r] |= kRowCopies;
            }
    }

    int want = 0;   // of all rows so far
    for (int r0 = 0; r0 < a.R; r0 += kPagesThreads) {
        const int r = r0 + tid;
        int n = 0;
        if (r < a.R && (flags[r] & kRowWants)) {
            const int len = length(r);
            n = pages_of((int64_t)len + adds(r), a.shift) - pages_of(len, a.shift) + ((flags[r] & kRowCopies) != 0);
        }
        int sum;
        const int before = block_before(n, sh, sum);
        if (r < a.R) pre[r] = want + before;
        want += sum;
    }
    if (tid == 0) pre[a.R] = want;

    int have = 0;   // free pages found, up to `want`
    const int off = (int)((reinterpret_cast<uintptr_t>(a.uses) >> 2) & 3);   // 16-byte loads at their addresses
    for (int p0 = -off; p0 < a.N && have < want; p0 += kPagesThreads * kPagesScan) {
        const int p = p0 + tid * kPagesScan;
        uint32_t free = 0;
        if (p >= 0 && p + kPagesScan <= a.N) {
#pragma unroll
            for (int i = 0; i < kPagesScan / 4; ++i) {
                const int4 u = *reinterpret_cast<const int4*>(a.uses + p + 4 * i);
                free |= (uint32_t)((u.x == 0) | (u.y == 0) << 1 | (u.z == 0) << 2 | (u.w == 0) << 3) << (4 * i);
            }
        } else {
            for (int i = max(0, -p); i < min(kPagesScan, a.N - p); ++i) free |= (uint32_t)(a.uses[p + i] == 0) << i;
        }
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

    // rows: lengths, and the pages in place of open ones
    auto gets = [&](int r) { return (flags[r] & kRowWants) && (pre[r + 1] == pre[r] || pre[r + 1] <= have); };
    for (int r = tid; r < a.R; r += kPagesThreads) {
        const int len = length(r), add = adds(r);
        const bool ok = gets(r);
        int4 c = make_int4(0, 0, 0, 0);
        if (ok && (flags[r] & kRowCopies)) {
            int32_t* at = a.table + (int64_t)r * a.tab + (len >> a.shift);
            c = make_int4(*at, pages[pre[r]], len & mask, 0);
            *at = c.y;
            a.uses[c.y] = 1;
            atomicAdd(&a.uses[c.x], -1);
        }
        copies[r] = c;
        a.out[r] = ok ? len + add : a.lens[r];
    }
    // new pages, each by the thread whose turn it is: its row is the last one that begins at or before it
    for (int i = tid; i < min(want, have); i += kPagesThreads) {
        int lo = 0, hi = a.R - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (pre[mid] <= i) lo = mid;
            else hi = mid - 1;
        }
        const int r = lo, j = i - pre[r], copy = (flags[r] & kRowCopies) != 0;
        if (pre[r + 1] > have || j < copy) continue;
        a.table[(int64_t)r * a.tab + pages_of(length(r), a.shift) + j - copy] = pages[i];
        a.uses[pages[i]] = 1;
    }
    if (!slots_too) return;
    __syncthreads();
    for (int i = tid; i < a.R * a.most; i += kPagesThreads) {
        const int r = i / a.most, j = i - r * a.most;
        a.slots[i] = j < adds(r) && gets(r) ? slot_of(a, r, (int64_t)length(r) + j) : -1;
    }
}

// the slots of longer additions
__global__ void __launch_bounds__(256) slots_kernel(ExtendArgs a) {
    const int r = blockIdx.x, add = min(max(a.add[r], 0), a.most), len = pages_len(a.lens[r], a.M, a.shift);
    const bool ok = add > 0 && a.out[r] == len + add;   // refused rows keep their lengths
    for (int j = blockIdx.y * 256 + threadIdx.x; j < a.most; j += gridDim.y * 256)
        a.slots[(int64_t)r * a.most + j] = ok && j < add ? slot_of(a, r, (int64_t)len + j) : -1;
}

// pages that rows can want between them, in whole int4
static int64_t extend_most(int32_t R, int32_t M, int32_t N, int32_t shift, int32_t most) {
    const int64_t each = ((int64_t)most >> shift) + 3, all = (each < M + 1 ? each : M + 1) * (int64_t)R;
    return ((all < N ? all : N) + 3) & ~3ll;
}

int64_t extend_pages_workspace(int32_t R, int32_t M, int32_t N, int32_t shift, int32_t most) {
    if (R < 1 || M < 1 || N < 1 || shift < 0 || shift > 20 || most < 1) return 0;
    return (4 * (int64_t)R + extend_most(R, M, N, shift, most) + 2 * (int64_t)N) * (int64_t)sizeof(int32_t);
}

int extend_pages(const ExtendArgs& a, void* stream) {
    FX_REQUIRE(a.R >= 1 && a.R <= kPagesRows, "extend_pages: %d rows (1 to %d)", a.R, kPagesRows);
    FX_REQUIRE(a.M >= 1 && a.N >= 1 && a.most >= 1 && a.shift >= 0 && a.shift <= 20, "extend_pages: bad shape M=%d N=%d most=%d shift=%d", a.M, a.N,
               a.most, a.shift);
    FX_REQUIRE(((int64_t)a.M << a.shift) <= 0x7fffffff - 128 && (int64_t)a.R * a.M < 0x7fffffff, "extend_pages: a table of %d x %d pages is too large", a.R, a.M);
    FX_REQUIRE(a.N <= 0x7fffffff - kPagesThreads * kPagesScan, "extend_pages: %d pages are too many", a.N);
    FX_REQUIRE(a.table && a.uses && a.lens && a.add && a.slots && a.out && a.work, "extend_pages: null pointer");
    FX_REQUIRE(((uintptr_t)a.work & 15) == 0, "extend_pages: work must be 16-byte aligned");
    const bool one = (int64_t)a.R * a.most <= 8 * kPagesThreads;   // slots in the same launch
    const size_t bytes = (size_t)(a.R + 1) * 4 + (size_t)((a.R + 3) & ~3);
    hipLaunchKernelGGL(extend_kernel, dim3(1), dim3(kPagesThreads), bytes, (hipStream_t)stream, a, extend_most(a.R, a.M, a.N, a.shift, a.most), one);
    if (int e = check_launch("extend_pages")) return e;
    if (one) return 0;
    const int y = (a.most + 1023) / 1024;
    hipLaunchKernelGGL(slots_kernel, dim3((unsigned)a.R, (unsigned)(y < 64 ? y : 64)), dim3(256), 0, (hipStream_t)stream, a);
    return check_launch("extend_pages_slots");
}

__global__ void __launch_bounds__(256) copy_pages_kernel(CopyPagesArgs a) {
    const int4 c = reinterpret_cast<const int4*>(a.copies)[blockIdx.x];
    const int t = blockIdx.y, per = a.D / 8, n = c.z * a.H * per;
    uint16_t* const p = a.at[t];
    for (int i = threadIdx.x; i < n; i += 256) {
        const int d = i % per, hj = i / per, h = hj % a.H, j = hj / a.H;
        const int64_t in = (int64_t)j * a.st[t] + (int64_t)h * a.sh[t] + d * 8;
        st16(p + (int64_t)c.y * a.sp[t] + in, ld16(p + (int64_t)c.x * a.sp[t] + in));
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
// HBM-bound: every new row is read once and written once, 16 bytes a lane.  A workgroup takes some tokens of a row of
// the batch, a thread four pieces of them at a time.

struct StorePlan {
    int32_t tokens, units;   // of a workgroup; 16-byte pieces of a token
};

__global__ void __launch_bounds__(256) store_pages_kernel(StorePagesArgs a, StorePlan p) {
    const int r = blockIdx.y, t0 = blockIdx.x * p.tokens, n = min(p.tokens, a.T - t0) * p.units, per = a.D / 8;
    const int64_t* slots = a.slots + r * a.sr;
    const uint16_t *k = a.k + r * a.kr, *v = a.v + r * a.vr;
    constexpr int U = 4;
    for (int i0 = threadIdx.x; i0 < n; i0 += 256 * U) {
        int64_t slot[U];
        uint4 x[U], y[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + 256 * u, t = t0 + i / p.units;
            slot[u] = i < n ? slots[t * a.st] : -1;
            if (slot[u] >= a.N << a.shift) slot[u] = -1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + 256 * u, tt = i / p.units, e = i - tt * p.units, h = e / per, d = (e - h * per) * 8;
            if (slot[u] >= 0) {
                x[u] = ld16_nt(k + (t0 + tt) * a.kt + h * a.kh + d);
                y[u] = ld16_nt(v + (t0 + tt) * a.vt + h * a.vh + d);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + 256 * u, tt = i / p.units, e = i - tt * p.units, h = e / per, d = (e - h * per) * 8;
            if (slot[u] >= 0) {
                const int64_t page = slot[u] >> a.shift, j = slot[u] & ((1 << a.shift) - 1);
                st16(a.kp + page * a.kpp + j * a.kpt + h * a.kph + d, x[u]);
                st16(a.vp + page * a.vpp + j * a.vpt + h * a.vph + d, y[u]);
            }
        }
    }
}

int store_pages(const StorePagesArgs& a, void* stream) {
    FX_REQUIRE(a.R >= 1 && a.T >= 1 && a.H >= 1 && a.N >= 1 && a.D >= 8 && a.D % 8 == 0 && a.shift >= 0 && a.shift <= 20,
               "store_pages: bad shape R=%d T=%d H=%d D=%d N=%lld shift=%d", a.R, a.T, a.H, a.D, (long long)a.N, a.shift);
    FX_REQUIRE(a.k && a.v && a.slots && a.kp && a.vp, "store_pages: null pointer");
    const int64_t s[] = {a.kr, a.kt, a.kh, a.vr, a.vt, a.vh, a.kpp, a.kpt, a.kph, a.vpp, a.vpt, a.vph};
    for (int64_t x : s) FX_REQUIRE(x % 8 == 0, "store_pages: strides must be multiples of 8 elements");
    FX_REQUIRE((((uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.kp | (uintptr_t)a.vp) & 15) == 0, "store_pages: 16-byte aligned tensors");
    FX_REQUIRE((int64_t)a.H * (a.D / 8) < (1 << 24) && a.R <= 65535, "store_pages: %d rows of %d x %d are too many or too wide", a.R, a.H, a.D);
    StorePlan p{};
    p.units = a.H * (a.D / 8);
    p.tokens = p.units >= 2048 ? 1 : 2048 / p.units;   // two turns of a thread
    const dim3 grid((unsigned)((a.T + p.tokens - 1) / p.tokens), (unsigned)a.R);
    FX_REQUIRE((int64_t)grid.x * 256 <= 0xffffffffLL, "store_pages: %d tokens are too many", a.T);
    hipLaunchKernelGGL(store_pages_kernel, grid, dim3(256), 0, (hipStream_t)stream, a, p);
    return check_launch("store_pages");
}

// ---- reorder -----------------------------------------------------------------------------
//
// A workgroup a few columns of the table, for all rows at once: what the rows held is in LDS before
// any of it is overwritten, so it is done in place.  A page that row p held is now held by as many rows as went on from
// p: its uses change by one less than that.  Bounded by its chain of round trips (lengths, entries, and
// what is written) up to some megabytes of table.

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
