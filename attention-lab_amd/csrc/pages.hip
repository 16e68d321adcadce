// The pages of a K/V cache that sequences share: branching, making room, writing, shortening and compacting.
//
// A cache holds, for every layer, pools K, V [pages, G, page, 128] bf16; for the layers together a table [S, W] of int32 (entry
// e of slot i: the page of its positions [e page, (e + 1) page), or -1), lengths [S] and refs [pages], refs[p] the number of
// entries that name page p (0: free). Everything is decided on the device, so that a step can be captured and replayed:
//
//   fork      table'[i] = table[parents[i]], lengths'[i] = lengths[parents[i]]; a parent outside [0, S): an empty slot
//   reserve   lengths'[i] = n + t. If n ends inside a page that others hold too, the slot gets a page of its own with the rows
//             [0, n % page) copied; where all of its holders are written to, the last of them in slot order keeps it. Then
//             ceil((n + t) / page) - ceil(n / page) pages more. In the order of slots and entries, lowest free page first.
//             A slot for whose copy none is left keeps its rows of the shared page in a claim (below)
//   append    a layer's rows of the last t positions, written to their pages
//   truncate  lengths'[i] = min(n, l), the entries from ceil(l / page) on given back
//   compact   with u pages in use: the i-th of them at or past u moves to the i-th free one below u
//
// A claim is an entry of a slot whose length has passed the rows that the entry's page holds for it: the first `rows` of the
// page are the slot's and stay counted, but it had no page of its own to go on in. It reads as an entry without a page, and a
// truncation to those rows or fewer makes the page the entry's again. Written as INT32_MIN + rows pages + page: 1 <= rows < the
// page's, so it lies below -1, and where a page's rows are not known (fork) as in any page, rows < 65536.
//
// Every choice depends on the cache alone, never on the order in which workgroups or atomics run: counts are integer sums,
// and free pages are dealt out by prefix sums over the pool. Entries and lengths are checked before they address memory.
//
// What bounds them: launches and latencies for the bookkeeping, bytes for the copies. The bookkeeping of a reserve is one
// workgroup's, because its parts depend on each other (who keeps a page, how many are wanted, which are free) and a grid would
// have to meet three times; the copies that it asks for are a second launch of as many waves as the chip holds. 8 prompts x 8
// answers, 512 pages: fork 3.5 us, reserve 7, its copies (8 layers, up to 64 half pages) 8, a layer's append 3.4; 124 slots of 98
// entries: fork 4.8, reserve 8.4, truncate 2.2. Compaction of 2048 pages of 64 rows, half in use: ranking 9 us, copies 212 (537
// MB each way, 5.1 TB/s).
#include "common.h"

namespace attnlab {
namespace {

constexpr int kDim = 128;
constexpr int kRowWords = kDim * 2 / 16;     // 16-byte words of a row
constexpr int kMaxSlots = 1024;              // a thread of the reserve's workgroup for each
constexpr int kMaxPage = 1 << 16;
constexpr int kColumns = 16;                 // table entries a fork's workgroup exchanges between the slots
constexpr int kBook = 1024;                  // threads of the reserve's and the compaction's workgroup
constexpr int kScan = 16;                    // pages a thread looks at in a round
constexpr int kCopyRows = 16;                // rows of a page that a wave copies at a time: 4 KB, four loads in flight
constexpr int kAppendRun = 32;               // rows that a workgroup of a long write takes (four appends of 3 x 1003 rows: 44.5
                                             // us with the reserve; 47.2 with 16, 48.2 with 64)
constexpr int kCopyGroups = 2048;            // workgroups of a copy: eight per CU, one wave of each SIMD from each

// What a reserve or a compaction leaves to its copies, in the scratch buffer.
struct Moves {
    int32_t count, used;                     // entries of `src`, `dst`, `rows`; pages in use (compaction)
    int32_t pad[2];
};

struct Book {
    int32_t* table;                          // [S, W]
    int32_t* lengths;                        // [S]
    int32_t* refs;                           // [pages]
    int S, W, pages, shift;
};

__device__ __forceinline__ bool names(int32_t page, int pages) { return (uint32_t)page < (uint32_t)pages; }

// A claim's page and rows; -1 and 0 of an entry that is none. `most`: a page's rows.
struct Claim {
    int page = -1, rows = 0;
    __device__ __forceinline__ Claim(int32_t entry, int pages, int most) {
        if (entry >= -1) return;
        const uint32_t x = (uint32_t)entry ^ 0x80000000u, n = x / (uint32_t)pages;
        if (n < 1 || n >= (uint32_t)most) return;
        page = (int)(x - n * (uint32_t)pages);
        rows = (int)n;
    }
};
__device__ __forceinline__ int32_t claim_of(int page, int rows, int pages) {
    return (int32_t)(0x80000000u + (uint32_t)rows * (uint32_t)pages + (uint32_t)page);
}
// The page that an entry counts for, or -1.
__device__ __forceinline__ int counted(int32_t entry, int pages, int most) {
    return names(entry, pages) ? entry : Claim(entry, pages, most).page;
}

// The slots' rows exchanged, 16 entries of all of them at a time: no workgroup reads what another writes, so the table is
// changed in place. One more workgroup does the lengths.
__global__ __launch_bounds__(256) void page_fork(Book a, const int32_t* parents) {
    __shared__ int32_t was[kMaxSlots * kColumns];
    const int tid = threadIdx.x;
    if (blockIdx.x == gridDim.x - 1) {
        for (int i = tid; i < a.S; i += 256) was[i] = a.lengths[i];
        __syncthreads();
        for (int i = tid; i < a.S; i += 256) {
            const int p = parents[i];
            a.lengths[i] = names(p, a.S) ? was[p] : 0;
        }
        return;
    }
    // eight rows of a thread on their way at a time
    constexpr int kStep = 256 / kColumns, kAhead = 8;
    const int e0 = blockIdx.x * kColumns, col = tid & (kColumns - 1);
    const bool in = e0 + col < a.W;
    for (int i0 = tid / kColumns; i0 < a.S; i0 += kStep * kAhead) {
        int32_t v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            v[u] = in ? a.table[(size_t)min(i0 + kStep * u, a.S - 1) * a.W + e0 + col] : -1;
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (i0 + kStep * u < a.S) was[(i0 + kStep * u) * kColumns + col] = v[u];
    }
    __syncthreads();
    if (!in) return;
    for (int i0 = tid / kColumns; i0 < a.S; i0 += kStep * kAhead) {
        int32_t p[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) p[u] = parents[min(i0 + kStep * u, a.S - 1)];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = i0 + kStep * u;
            if (i >= a.S) break;
            const int32_t old = was[i * kColumns + col], now = names(p[u], a.S) ? was[p[u] * kColumns + col] : -1;
            if (now == old) continue;
            const int from = counted(old, a.pages, kMaxPage), to = counted(now, a.pages, kMaxPage);
            if (from >= 0) atomicSub(a.refs + from, 1);
            if (to >= 0) atomicAdd(a.refs + to, 1);
            a.table[(size_t)i * a.W + e0 + col] = now;
        }
    }
}

__global__ __launch_bounds__(256) void page_truncate(Book a, const int32_t* to, int each) {
    const int i = blockIdx.x, page = 1 << a.shift;
    const int n = a.lengths[i], l = max(to ? to[i] : each, 0);
    if (l >= n) return;
    __syncthreads();
    if (threadIdx.x == 0) a.lengths[i] = l;
    const int first = (int)(((int64_t)l + page - 1) >> a.shift);
    const int end = (int)min((int64_t)a.W, ((int64_t)n + page - 1) >> a.shift);
    for (int e = first + (int)threadIdx.x; e < end; e += 256) {
        int32_t* at = a.table + (size_t)i * a.W + e;
        const int p = counted(*at, a.pages, page);
        if (p >= 0) atomicSub(a.refs + p, 1);
        *at = -1;
    }
    const int part = l & (page - 1);
    if (threadIdx.x == 0 && part && (l >> a.shift) < a.W) {   // a claim of all that is left: the page again
        int32_t* at = a.table + (size_t)i * a.W + (l >> a.shift);
        const Claim c(*at, a.pages, page);
        if (part <= c.rows) *at = c.page;
    }
}

// Inclusive prefix sums of x and y over the workgroup's threads (sh: two words for each of its waves), and their totals.
__device__ __forceinline__ void block_scan(uint32_t& x, uint32_t& y, uint2* sh, uint32_t& all_x, uint32_t& all_y) {
    const int wave = threadIdx.x >> 6, waves = kBook / 64;
    x = wave_incl_scan(x);
    y = wave_incl_scan(y);
    if ((threadIdx.x & 63) == 63) sh[wave] = make_uint2(x, y);
    __syncthreads();
    uint2 before = make_uint2(0, 0);
    all_x = all_y = 0;
#pragma unroll
    for (int w = 0; w < waves; ++w) {
        const uint2 v = sh[w];
        before.x += w < wave ? v.x : 0u;
        before.y += w < wave ? v.y : 0u;
        all_x += v.x;
        all_y += v.y;
    }
    x += before.x;
    y += before.y;
}

// Pages base + 1024 u + thread, u < kScan, of which `flag(page)` says whether they count: for each that does, its rank among
// the pages in ascending order is handed to `take(page, rank)`. `found`: the rank of the first, advanced.
template <typename Flag, typename Take>
__device__ __forceinline__ void rank_pages(int base, int pages, uint32_t& found, uint4* sh, Flag flag, Take take) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    static_assert(kScan * kBook / 64 == 4 * 64, "a count for each wave and round, four to a lane");
    uint64_t hit[kScan];
#pragma unroll
    for (int u = 0; u < kScan; ++u) hit[u] = __ballot(base + kBook * u + tid < pages && flag(u));
    __syncthreads();
    if (lane == 0) {
#pragma unroll
        for (int u = 0; u < kScan; ++u) reinterpret_cast<uint32_t*>(sh)[kBook / 64 * u + wave] = (uint32_t)__popcll(hit[u]);
    }
    __syncthreads();
    // every wave sums the counts up for itself: lane l those of round l / 4, waves 4 (l % 4) ..
    const uint4 c = sh[lane];
    const uint32_t own = c.x + c.y + c.z + c.w, upto = wave_incl_scan(own);
    const int part = wave & 3;
    const uint32_t before = found + upto - own + (part > 0 ? c.x : 0u) + (part > 1 ? c.y : 0u) + (part > 2 ? c.z : 0u);
    found += (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
#pragma unroll
    for (int u = 0; u < kScan; ++u) {
        const uint32_t first = (uint32_t)__builtin_amdgcn_readlane((int)before, 4 * u + (wave >> 2));
        if (hit[u] >> lane & 1) take(base + kBook * u + tid, first + (uint32_t)__popcll(hit[u] & ((1ull << lane) - 1)));
    }
}

__global__ __launch_bounds__(kBook) void page_reserve(Book a, const int32_t* tokens, int each, int32_t* missing, Moves* moves,
                                                      int32_t* src, int32_t* dst, int32_t* rows) {
    __shared__ uint2 wave_sh[kBook / 64];
    __shared__ uint4 scan_sh[64];
    __shared__ __attribute__((aligned(16))) int32_t held_sh[kMaxSlots];   // -1 past the slots
    __shared__ __attribute__((aligned(16))) int32_t first_sh[kMaxSlots];  // a slot's first new entry; then its rows, where it is left
    __shared__ int32_t part_sh[kMaxSlots];
    __shared__ uint32_t upto_sh[kMaxSlots], job_sh[kMaxSlots];   // requests up to and with a slot's; its copy's number + 1, or 0
    const int tid = threadIdx.x, page = 1 << a.shift;
    int32_t pool[kScan];                     // the first pages' counts, on their way from the start; only free ones change below
#pragma unroll
    for (int u = 0; u < kScan; ++u) pool[u] = a.refs[min(kBook * u + tid, a.pages - 1)];
    const bool slot = tid < a.S;
    const int n = slot ? max(a.lengths[tid], 0) : 0, t = slot ? max(tokens ? tokens[tid] : each, 0) : 0;
    const int64_t end = min((int64_t)n + t, (int64_t)INT32_MAX);
    const int last = n >> a.shift, part = n & (page - 1);
    int held = t > 0 && part && last < a.W ? a.table[(size_t)tid * a.W + last] : -1;
    const int refs = names(held, a.pages) ? a.refs[held] : 0;
    if (refs <= 1) held = -1;                // nobody's, or the slot's alone
    held_sh[tid] = held;
    __syncthreads();
    bool copies = false;
    if (held >= 0) {
        int writers = 0, later = 0;
        for (int j = 0; j < a.S; j += 4) {
            const int4 v = *reinterpret_cast<const int4*>(held_sh + j);
            const int same[4] = {v.x == held, v.y == held, v.z == held, v.w == held};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                writers += same[i];
                later |= same[i] && j + i > tid;
            }
        }
        copies = later || writers < refs;
    }
    const int from = (int)(((int64_t)n + page - 1) >> a.shift), upto = (int)((end + page - 1) >> a.shift);
    const int fresh = max(min(upto, a.W) - from, 0);
    const int lost = t > 0 ? max(upto - max(from, a.W), 0) : 0;   // pages that the table has no entry for
    uint32_t wanted, jobs, to = (t > 0 ? (uint32_t)fresh : 0u) + copies, job = copies;
    block_scan(to, job, wave_sh, wanted, jobs);
    if (slot) {
        first_sh[tid] = from;
        part_sh[tid] = part;
        upto_sh[tid] = to;
        job_sh[tid] = copies ? job : 0u;
        if (t > 0) a.lengths[tid] = (int32_t)end;
    }
    __syncthreads();
    // request r -> its slot, and the entry that gets the page (or -1 where there is none left)
    auto give = [&](uint32_t r, int32_t p) {
        int lo = 0, hi = a.S - 1;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (upto_sh[mid] > r) hi = mid;
            else lo = mid + 1;
        }
        const uint32_t k = r - (lo ? upto_sh[lo - 1] : 0u), j = job_sh[lo];
        const bool copy = j && k == 0;
        const int e = first_sh[lo] + (int)k - (j ? 1 : 0);   // a copy's entry is the one before the first new one
        if (p >= 0 || !copy) a.table[(size_t)lo * a.W + e] = p;
        if (copy) {
            src[j - 1] = held_sh[lo];
            dst[j - 1] = p;
            rows[j - 1] = p < 0 ? 0 : part_sh[lo];
        }
    };
    uint32_t found = 0;
    for (int base = 0; base < a.pages && found < wanted; base += kBook * kScan) {
        if (base > 0) {
#pragma unroll
            for (int u = 0; u < kScan; ++u) pool[u] = a.refs[min(base + kBook * u + tid, a.pages - 1)];
        }
        rank_pages(base, a.pages, found, scan_sh, [&](int u) { return pool[u] <= 0; }, [&](int p, uint32_t rank) {
            if (rank >= wanted) return;
            a.refs[p] = 1;
            give(rank, p);
        });
    }
    for (uint32_t r = found + tid; r < wanted; r += kBook) give(r, -1);
    const bool copied = copies && (tid ? upto_sh[tid - 1] : 0u) < found;   // a copy is its slot's first request
    if (copied) atomicSub(a.refs + held, 1);
    int out = lost + (tid == 0 && wanted > found ? (int)(wanted - found) : 0);
    if (found < wanted) {
        // No page was left for every copy. Of the writers that are still on a page, the one with the most rows (the last of those)
        // writes on in place, if its other holders are writers too or claim no more rows than it has; the others claim theirs.
        // (1024 branches of one prompt without a page: 76 us, 65 of them the requests that cannot be met)
        const bool left = held >= 0 && !copied;
        __syncthreads();                     // the requests' entries are dealt
        first_sh[tid] = left ? part << 10 | tid : -1;
        __syncthreads();
        int best = -1, holders = 0, claimed = 0;
        bool on = false;
        if (left) {
            for (int j = 0; j < a.S; j += 4) {
                const int4 h = *reinterpret_cast<const int4*>(held_sh + j), f = *reinterpret_cast<const int4*>(first_sh + j);
                holders += (h.x == held) + (h.y == held) + (h.z == held) + (h.w == held);
                best = max(max(max(best, h.x == held ? f.x : -1), max(h.y == held ? f.y : -1, h.z == held ? f.z : -1)),
                           h.w == held ? f.w : -1);
            }
            on = best == (part << 10 | tid);
        }
        // claims, at the same entry of their slots, or holders that do not grow: a wave looks for those of its pages, one by one
        for (uint64_t open = __ballot(on && holders < refs); open; open &= open - 1) {
            const int x = __builtin_ctzll(open), p = __shfl(held, x, 64), e = __shfl(last, x, 64);
            int more = 0, rows_of = 0;
            for (int j = tid & 63; j < a.S; j += 64) {
                const Claim c(a.table[(size_t)j * a.W + e], a.pages, page);
                if (c.page != p || held_sh[j] == p) continue;
                ++more;
                rows_of = max(rows_of, c.rows);
            }
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                more += __shfl_xor(more, d, 64);
                rows_of = max(rows_of, __shfl_xor(rows_of, d, 64));
            }
            if ((tid & 63) == x) {
                holders += more;
                claimed = rows_of;
            }
        }
        if (left) {
            on = on && holders == refs && claimed <= part;
            if (!on) a.table[(size_t)tid * a.W + last] = claim_of(held, part, a.pages);
            out += !on - copies;             // its copy, if it asked for one, is counted above
        }
    }
    if (tid == 0) moves->count = (int32_t)jobs;
    if (missing && out) atomicAdd(missing, out);
}

__global__ __launch_bounds__(kBook) void page_compact(Book a, Moves* moves, int32_t* src, int32_t* dst, int32_t* rank_of) {
    __shared__ uint2 wave_sh[kBook / 64];
    __shared__ uint4 scan_sh[64];
    const int tid = threadIdx.x;
    uint32_t mine = 0, none = 0, used, all;
    for (int base = 0; base < a.pages; base += kBook * kScan) {
        int32_t r[kScan];
#pragma unroll
        for (int u = 0; u < kScan; ++u) r[u] = a.refs[min(base + kBook * u + tid, a.pages - 1)];
#pragma unroll
        for (int u = 0; u < kScan; ++u) mine += base + kBook * u + tid < a.pages && r[u] > 0;
    }
    block_scan(mine, none, wave_sh, used, all);
    uint32_t holes = 0, high = 0;
    for (int base = 0; base < a.pages; base += kBook * kScan) {
        int32_t r[kScan];
#pragma unroll
        for (int u = 0; u < kScan; ++u) r[u] = a.refs[min(base + kBook * u + tid, a.pages - 1)];
        auto page_of = [&](int u) { return base + kBook * u + tid; };
        rank_pages(base, a.pages, holes, scan_sh, [&](int u) { return page_of(u) < (int)used && r[u] <= 0; },
                   [&](int p, uint32_t rank) { dst[rank] = p; });
        rank_pages(base, a.pages, high, scan_sh, [&](int u) { return page_of(u) >= (int)used && r[u] > 0; },
                   [&](int p, uint32_t rank) { src[rank] = p; rank_of[p] = (int32_t)rank; });
#pragma unroll
        for (int u = 0; u < kScan; ++u)
            if (page_of(u) >= (int)used && page_of(u) < a.pages && r[u] <= 0) rank_of[page_of(u)] = -1;
    }
    __syncthreads();   // as many pages at or past `used` are in use as are free below it
    for (uint32_t i = tid; i < high; i += kBook) {
        a.refs[dst[i]] = a.refs[src[i]];
        a.refs[src[i]] = 0;
    }
    if (tid == 0) {
        moves->count = (int32_t)high;
        moves->used = (int32_t)used;
    }
}

struct CopyArgs {
    uint16_t* pool[2];                       // K and V of every layer
    int64_t layer_stride;                    // elements
    int layers, G, page, pages;
    const Moves* moves;
    const int32_t* src;
    const int32_t* dst;
    const int32_t* rows;                     // rows of each copy; null: whole pages
    int32_t* table;                          // compaction: entries at or past moves->used follow their pages
    int64_t entries;
    const int32_t* rank_of;
};

// The pages of `src` copied to `dst` in every layer, K and V. A wave takes up to 16 rows of one (copy, layer, K or V, group) at a
// time and the grid walks over them; nothing is copied onto a page that another copy reads.
__global__ __launch_bounds__(256) void page_copy(CopyArgs a) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)), waves = gridDim.x * 4;
    const int count = a.moves->count;
    const int chunks = (a.page + kCopyRows - 1) / kCopyRows;
    const int per = a.layers * 2 * a.G * chunks;
    const int64_t units = (int64_t)count * per;
    for (int64_t unit = wave; unit < units; unit += waves) {
        const int j = (int)(unit / per);
        int x = (int)(unit - (int64_t)j * per);
        const int c = x % chunks;
        x /= chunks;
        const int g = x % a.G;
        x /= a.G;
        const int rows = min((a.rows ? a.rows[j] : a.page) - kCopyRows * c, kCopyRows);
        const int s = a.src[j], d = a.dst[j];
        if (rows <= 0 || !names(s, a.pages) || !names(d, a.pages)) continue;
        uint16_t* base = a.pool[x & 1] + (size_t)(x >> 1) * a.layer_stride + (size_t)kCopyRows * c * kDim;
        const size_t step = (size_t)a.page * kDim;
        const u32x4_t* from = reinterpret_cast<const u32x4_t*>(base + ((size_t)s * a.G + g) * step);
        u32x4_t* to = reinterpret_cast<u32x4_t*>(base + ((size_t)d * a.G + g) * step);
        const int words = rows * kRowWords;
        u32x4_t w[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (64 * u + lane < words) w[u] = from[64 * u + lane];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (64 * u + lane < words) to[64 * u + lane] = w[u];
    }
    if (a.table && count) {
        const int used = a.moves->used;
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.entries; i += (int64_t)gridDim.x * 256) {
            const int32_t entry = a.table[i];
            const Claim c(entry, a.pages, a.page);
            const int32_t p = c.rows ? c.page : entry;
            if (p < used || p >= a.pages) continue;
            const int32_t r = a.rank_of[p];
            if (r >= 0) a.table[i] = c.rows ? claim_of(a.dst[r], c.rows, a.pages) : a.dst[r];
        }
    }
}

struct AppendArgs {
    const uint16_t* x[2];                    // K and V rows: (slot, group, row, dim) at x + i sb + g sg + t st + dim
    int64_t sb[2], sg[2], st[2];
    uint16_t* pool[2];                       // the layer's K and V pages
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* tokens;                   // rows of each slot, or null: T
    int S, W, pages, shift, G, T;
};

// Where row t of slot i goes: its (page, group, row) in the pool, or -1.
__device__ __forceinline__ int64_t row_of(const AppendArgs& a, int i, int g, int t, int count, int64_t first) {
    const int64_t pos = first + t, e = pos >> a.shift;
    const int p = t < count && pos >= 0 && e < a.W ? a.table[(size_t)i * a.W + e] : -1;
    return names(p, a.pages) ? (((int64_t)p * a.G + g) << a.shift) + (pos & ((1 << a.shift) - 1)) : -1;
}

// Sixteen lanes a row, K or V by blockIdx.y. Few tokens (LONG false): rows of all slots and groups in line, sixteen to a
// workgroup; else kAppendRun consecutive rows of one (slot, group).
template <bool LONG>
__global__ __launch_bounds__(256) void page_append(AppendArgs a, int runs) {
    constexpr int kRows = LONG ? kAppendRun / 16 : 1;
    const int kv = blockIdx.y, lane16 = threadIdx.x & 15, line = threadIdx.x >> 4;
    int i, g, t0;
    if constexpr (LONG) {
        const int ig = blockIdx.x / runs;
        t0 = (blockIdx.x - ig * runs) * kAppendRun + line;
        i = ig / a.G;
        g = ig - i * a.G;
    } else {
        const int64_t x = (int64_t)blockIdx.x * 16 + line;
        const int64_t ig = x / a.T;
        t0 = (int)(x - ig * a.T);
        i = (int)(ig / a.G);
        g = (int)(ig - (int64_t)i * a.G);
        if (i >= a.S) return;
    }
    const int tokens = a.tokens ? a.tokens[i] : a.T, count = min(tokens, a.T);
    if (t0 >= count) return;
    const int length = a.lengths[i];
    if (length == INT32_MAX) return;         // where a reserve stops counting: which positions the rows have is not known
    const int64_t first = (int64_t)length - tokens;
    const uint16_t* from = a.x[kv] + i * a.sb[kv] + g * a.sg[kv] + 8 * lane16;
    u32x4_t w[kRows];
    int64_t at[kRows];
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
        at[u] = row_of(a, i, g, t0 + 16 * u, count, first);
        w[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(from + min(t0 + 16 * u, count - 1) * a.st[kv]));
    }
#pragma unroll
    for (int u = 0; u < kRows; ++u)
        if (at[u] >= 0) *reinterpret_cast<u32x4_t*>(a.pool[kv] + at[u] * kDim + 8 * lane16) = w[u];
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Whether two arrays of na and nb int32 share memory.
bool meet(const int32_t* a, int64_t na, const int32_t* b, int64_t nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + 4 * (uintptr_t)nb && y < x + 4 * (uintptr_t)na;
}

int check_book(const int32_t* table, const int32_t* lengths, const int32_t* refs, int S, int W, int pages, int page) {
    ATTNLAB_REQUIRE(1 <= S && S <= kMaxSlots, "slots S=%d outside [1, %d]", S, kMaxSlots);
    ATTNLAB_REQUIRE(W >= 1 && pages >= 1, "max_pages=%d and num_pages=%d must be positive", W, pages);
    ATTNLAB_REQUIRE(page >= 1 && page <= (1 << 16) && (page & (page - 1)) == 0,
                    "page_size=%d must be a power of two in [1, 65536]", page);
    ATTNLAB_REQUIRE((int64_t)W * page <= INT32_MAX, "max_pages * page_size exceeds 2^31 positions");
    // a reserve counts its requests in 32 bits
    ATTNLAB_REQUIRE((int64_t)S * W <= INT32_MAX, "a table of %d slots x %d pages exceeds 2^31 entries", S, W);
    ATTNLAB_REQUIRE(table && lengths && refs, "table, lengths and refs must be device pointers");
    return ATTNLAB_OK;
}

int check_pools(const uint16_t* k, const uint16_t* v, int layers, int pages, int G, int page) {
    ATTNLAB_REQUIRE(layers >= 1 && G >= 1, "layers=%d and G=%d must be positive", layers, G);
    ATTNLAB_REQUIRE((int64_t)pages * G * page <= INT32_MAX, "the pool of %d pages x %d groups x %d rows exceeds 2^31 rows", pages,
                    G, page);
    ATTNLAB_REQUIRE(k && v && aligned(k, 16) && aligned(v, 16), "k and v must be 16-byte aligned device pointers");
    return ATTNLAB_OK;
}

Book book_of(int32_t* table, int32_t* lengths, int32_t* refs, int S, int W, int pages, int page) {
    return Book{table, lengths, refs, S, W, pages, __builtin_ctz((unsigned)page)};
}

// Scratch: the header, then src, dst and rows of at most `slots` copies, or src, dst and rank_of of the pages.
int64_t scratch_words(int S, int pages) { return (int64_t)(sizeof(Moves) / 4) + 3 * (int64_t)(S > pages ? S : pages); }

int launch_copy(const CopyArgs& a, int64_t most, hipStream_t s, const char* what) {
    const int chunks = (a.page + kCopyRows - 1) / kCopyRows;
    int64_t groups = (most * a.layers * 2 * a.G * chunks + 3) / 4;
    if (a.table && groups < (a.entries + 255) / 256) groups = (a.entries + 255) / 256;
    if (groups > kCopyGroups) groups = kCopyGroups;
    hipLaunchKernelGGL(page_copy, dim3((unsigned)groups), dim3(256), 0, s, a);
    return check_launch(what);
}

}  // namespace
}  // namespace attnlab

using namespace attnlab;

extern "C" int64_t attnlab_page_scratch_bytes(int S, int num_pages) {
    return S < 1 || num_pages < 1 ? -1 : 4 * scratch_words(S, num_pages);
}

extern "C" int attnlab_page_fork(int32_t* table, int32_t* lengths, int32_t* refs, const int32_t* parents, int S, int max_pages,
                                 int num_pages, void* stream) {
    const int rc = check_book(table, lengths, refs, S, max_pages, num_pages, 1);
    if (rc) return rc;
    ATTNLAB_REQUIRE(parents, "parents must be a device pointer");
    // read by workgroups that others' writes would overtake
    ATTNLAB_REQUIRE(!meet(parents, S, lengths, S) && !meet(parents, S, refs, num_pages) &&
                        !meet(parents, S, table, (int64_t)S * max_pages),
                    "parents must not lie in the cache's own tensors");
    const int groups = (max_pages + kColumns - 1) / kColumns + 1;
    hipLaunchKernelGGL(page_fork, dim3((unsigned)groups), dim3(256), 0, reinterpret_cast<hipStream_t>(stream),
                       book_of(table, lengths, refs, S, max_pages, num_pages, 1), parents);
    return check_launch("page_fork");
}

extern "C" int attnlab_page_truncate(int32_t* table, int32_t* lengths, int32_t* refs, const int32_t* to, int length, int S,
                                     int max_pages, int num_pages, int page_size, void* stream) {
    const int rc = check_book(table, lengths, refs, S, max_pages, num_pages, page_size);
    if (rc) return rc;
    ATTNLAB_REQUIRE(to || length >= 0, "length=%d must not be negative", length);
    // a slot's workgroup reads to[i] beside others' writes; the lengths themselves change nothing
    ATTNLAB_REQUIRE(!to || ((to == lengths || !meet(to, S, lengths, S)) && !meet(to, S, refs, num_pages) &&
                            !meet(to, S, table, (int64_t)S * max_pages)),
                    "the lengths to truncate to must not lie in the cache's own tensors");
    hipLaunchKernelGGL(page_truncate, dim3((unsigned)S), dim3(256), 0, reinterpret_cast<hipStream_t>(stream),
                       book_of(table, lengths, refs, S, max_pages, num_pages, page_size), to, length);
    return check_launch("page_truncate");
}

extern "C" int attnlab_page_reserve(uint16_t* k, uint16_t* v, int layers, int num_pages, int G, int page_size, int32_t* table,
                                    int32_t* lengths, int32_t* refs, const int32_t* tokens, int each, int S, int max_pages,
                                    int32_t* missing, void* scratch, int64_t scratch_bytes, void* stream) {
    int rc = check_book(table, lengths, refs, S, max_pages, num_pages, page_size);
    if (!rc) rc = check_pools(k, v, layers, num_pages, G, page_size);
    if (rc) return rc;
    ATTNLAB_REQUIRE(tokens || each >= 0, "tokens=%d must not be negative", each);
    ATTNLAB_REQUIRE(scratch && aligned(scratch, 16) && scratch_bytes >= 4 * scratch_words(S, num_pages),
                    "scratch must be a 16-byte aligned device buffer of %lld bytes", (long long)(4 * scratch_words(S, num_pages)));
    Moves* moves = static_cast<Moves*>(scratch);
    int32_t* src = reinterpret_cast<int32_t*>(moves + 1);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(page_reserve, dim3(1), dim3(kBook), 0, s,
                       book_of(table, lengths, refs, S, max_pages, num_pages, page_size), tokens, each, missing, moves, src,
                       src + S, src + 2 * S);
    rc = check_launch("page_reserve");
    if (rc || page_size == 1) return rc;   // a length ends inside no page of one row
    const CopyArgs c{{k, v}, (int64_t)num_pages * G * page_size * kDim, layers, G, page_size, num_pages, moves, src, src + S,
                     src + 2 * S, nullptr, 0, nullptr};
    return launch_copy(c, S, s, "page_reserve (copies)");
}

extern "C" int attnlab_page_append(const uint16_t* k, int64_t k_b_stride, int64_t k_g_stride, int64_t k_t_stride,
                                   const uint16_t* v, int64_t v_b_stride, int64_t v_g_stride, int64_t v_t_stride,
                                   uint16_t* k_pages, uint16_t* v_pages, int num_pages, int G, int page_size,
                                   const int32_t* table, const int32_t* lengths, const int32_t* tokens, int S, int max_pages,
                                   int T, void* stream) {
    ATTNLAB_REQUIRE(T >= 0, "T=%d must not be negative", T);
    int rc = check_book(table, lengths, table, S, max_pages, num_pages, page_size);
    if (!rc) rc = check_pools(k_pages, v_pages, 1, num_pages, G, page_size);
    if (rc || T == 0) return rc;
    ATTNLAB_REQUIRE(k && v && aligned(k, 16) && aligned(v, 16) &&
                        ((k_b_stride | k_g_stride | k_t_stride | v_b_stride | v_g_stride | v_t_stride) & 7) == 0,
                    "k and v must be device pointers with 16-byte aligned rows");
    const AppendArgs a{{k, v}, {k_b_stride, v_b_stride}, {k_g_stride, v_g_stride}, {k_t_stride, v_t_stride},
                       {k_pages, v_pages}, table, lengths, tokens, S, max_pages, num_pages,
                       __builtin_ctz((unsigned)page_size), G, T};
    // runs and lines of rows: 3 x 1003 rows 7.1 and 8.0 us, 64 x 100 rows 13.5 and 15.2; up to 3 x 48 rows 2.9 either way
    const bool lengthy = T > 16;
    const int64_t runs = ((int64_t)T + kAppendRun - 1) / kAppendRun;
    const int64_t groups = lengthy ? (int64_t)S * G * runs : ((int64_t)S * G * T + 15) / 16;
    ATTNLAB_REQUIRE(groups < (int64_t)1 << 31, "grid of %lld workgroups is too large", (long long)groups);
    const dim3 grid((unsigned)groups, 2), wg(256);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (lengthy) hipLaunchKernelGGL(page_append<true>, grid, wg, 0, s, a, (int)runs);
    else hipLaunchKernelGGL(page_append<false>, grid, wg, 0, s, a, 0);
    return check_launch("page_append");
}

extern "C" int attnlab_page_compact(uint16_t* k, uint16_t* v, int layers, int num_pages, int G, int page_size, int32_t* table,
                                    int32_t* lengths, int32_t* refs, int S, int max_pages, void* scratch,
                                    int64_t scratch_bytes, void* stream) {
    int rc = check_book(table, lengths, refs, S, max_pages, num_pages, page_size);
    if (!rc) rc = check_pools(k, v, layers, num_pages, G, page_size);
    if (rc) return rc;
    ATTNLAB_REQUIRE(scratch && aligned(scratch, 16) && scratch_bytes >= 4 * scratch_words(S, num_pages),
                    "scratch must be a 16-byte aligned device buffer of %lld bytes", (long long)(4 * scratch_words(S, num_pages)));
    Moves* moves = static_cast<Moves*>(scratch);
    int32_t* src = reinterpret_cast<int32_t*>(moves + 1);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(page_compact, dim3(1), dim3(kBook), 0, s,
                       book_of(table, lengths, refs, S, max_pages, num_pages, page_size), moves, src, src + num_pages,
                       src + 2 * (int64_t)num_pages);
    rc = check_launch("page_compact");
    if (rc) return rc;
    const CopyArgs c{{k, v}, (int64_t)num_pages * G * page_size * kDim, layers, G, page_size, num_pages, moves, src,
                     src + num_pages, nullptr, table, (int64_t)S * max_pages, src + 2 * (int64_t)num_pages};
    return launch_copy(c, num_pages / 2, s, "page_compact (copies)");
}
