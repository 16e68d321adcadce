// Attention of sequences that share prompts, over a paged cache: sequence b's T queries sit at the last positions of its length,
//   out[b,g,i,t] = sum_j softmax_j(scale q[b,g,i,t] . k_j) v_j    over j <= lengths[b] - T + t, k_j and v_j by b's table
// Consecutive sequences form runs; the whole pages of a run's first prefix[r] positions are the same for all of its sequences. So
// the keys fall into two parts, each with its own softmax, and the parts (m, l, o) are merged at the end:
//   the shared part   a run's rows, n sequences x T queries x h heads, against its prefix: a matrix product, the keys read once
//   the own part      a sequence's T h rows against its positions from the prefix on
// A sequence that ends inside its run's prefix takes no part in the shared read and reads all of its positions in the own part, so
// the shared one has no masked positions at all.
//
// Both parts are split over workgroups by keys; each leaves its rows' partials, and a last launch merges a row's. How a
// prompt's keys are split is worked out on the device, from runs and prefixes that the host need not know: the blocks of all
// tiles of rows over the workgroups that the chip holds at once give a share; a tile's whole shares go first, and what is left
// of the tiles, shorter pieces, fills the gaps. A count beside each row says how many partials it has.
//
// Two kernels. `wide`: 128 rows, four waves of 32; blocks of 64 keys, S^T = K Q^T, the softmax on its accumulators, O^T += V^T P^T
// (v_mfma_f32_32x32x16_bf16), K and V copied into LDS a block ahead without passing through registers. `narrow`: up to 16 rows;
// each wave walks tiles of 32 keys of its own (v_mfma_f32_16x16x32_bf16), K from memory to the matrix core, V through the wave's
// LDS. A part begins at a page's first position, so in pages of 16 positions or more every 16 keys of a block share one: its
// entry is looked up a block ahead, and the 16 rows are a buffer that ends where they do (or at once, where there is no page),
// behind which loads give zeros. Smaller pages are looked up key by key. Keys without a row are masked.
//
// One launch does both parts, the own part's workgroups behind the shared part's.
//
// What bounds it (8 groups). 16 questions of 211 tokens, h=2, on 16K: 455 to 485 us with the merge's 16, 1.0 PFLOP/s in the shared
// part; the matrix cores are busy half of the time, and the softmax lies between a wave's products. 4 x 13 answers, h=8, on 9K,
// up to 1K of their own: 70 to 75 us, 3.6 to 3.8 TB/s: one block's copies in flight a workgroup, and a block's own chain of
// products, softmax and products (16 answers, h=8, on 128K: 149 us, 120 where K and V are in the caches). 16 answers, h=4, on 8K:
// 22.5 us, and 4 answers on 512: 15 (the host; 12 on the GPU), chains of latencies: the share 2.3, the first copies 2.7, four
// blocks 5.8, partials 1, the merge 5.
//
// Weights go to the matrix cores as bf16, the operand's type. Of one query each, what that rounding left is multiplied by V
// too, so they keep 16 bits, as in the package's other one-query reads (us, with the rest and without: 16 answers, h=4, on 8K
// 24.8 and 24.5; 4 x 13, h=8, on 9K 64.5 and 60.0; 2 x 30, h=4, on 16K 50.1 and 46.6; 16, h=8, on 32K 50.2 and 44.0, on 128K 149
// and 127; 8 x 4, h=4, on 16K 116 and 116); a chunk's are rounded once (2^-8 of each at most), as in its other chunk reads: the
// second product lies in what bounds the kernel (16 questions on 16K 642 and 473). Their sum is of the unrounded ones, sums fp32.
#include <cfloat>
#include <type_traits>

#include "mfma_attend.h"

namespace attnlab {
namespace {

constexpr int kDim = 128;
constexpr int kWide = 128, kNarrow = 16;    // rows of a workgroup
constexpr int kKeys = 64;                   // keys of a wide block
constexpr int kTile = 32;                   // keys of a narrow wave's tile
constexpr int kWaves = 4;
constexpr float kLazy = 8.0f;               // a row's shift is set 2^8 above its largest score and moves when one passes it
constexpr int kPart = 132;                  // m, l, two unused words, the 128 unnormalised outputs
constexpr int kMaxSplits = 64;              // partials that a row has of either part, at most
// Shares that the shared part is cut into: two workgroups per CU where all are wide, three where all are narrow. One where wide
// ones go with narrow ones of the own part, which take the other half of each CU: 4 prompts of 9K with 13 answers each take 67
// us, 79 with two, 69 and 71 with 224 and 320 shares; 48 answers (h=8) of 1500 to 14K 83 and 101; with little to read behind
// the prompt they are alike.
constexpr int kWideWorkers = 512, kMixedWorkers = 256, kNarrowWorkers = 768;

struct SharedArgs {
    const uint16_t* q;        // [B, G, h, T, 128]
    const uint16_t* K;        // [pages, G, page, 128]
    const uint16_t* V;
    const int32_t* table;     // [B, W], row stride table_stride
    int64_t table_stride;
    const int32_t* lengths;   // [B], or null: `length`
    const int32_t* prefixes;  // [R], or null: `prefix`
    const int32_t* runs;      // [R + 1], or null: one run of all
    int length, prefix;
    int B, G, h, T, W, R, pages, shift;
    float scale_log2;
    uint16_t* out;            // [B, G, h, T, 128]
    float* part;              // [B, G, h, T, shared + own, 132], or null: the own part's one partial is the output
    int2* counts;             // [B, G, h, T] partials that a row has of the two parts
    int shared, own;          // partials of the two parts that there is room for (shared 0: no shared part)
    int own_items, shared_turns, own_turns;   // workgroups of the own part, and an eighth of those of either
};

// What a masked key's row is read from.
__device__ __attribute__((aligned(16))) uint32_t shared_zeros[4];

__device__ __forceinline__ int length_of(const SharedArgs& a, int b) {
    const int64_t cap = (int64_t)a.W << a.shift;
    return (int)min((int64_t)max(a.lengths ? a.lengths[b] : a.length, 0), cap);
}
__device__ __forceinline__ int prefix_of(const SharedArgs& a, int r) {
    const int64_t cap = (int64_t)a.W << a.shift;
    return (int)min((int64_t)max(a.prefixes ? a.prefixes[r] : a.prefix, 0), cap) >> a.shift << a.shift;
}

struct Run {
    int first, count, prefix;   // its sequences; its whole pages' positions (0: nothing shared)
};

// Inclusive running maximum over the wave's lanes, of values of at least 0.
__device__ __forceinline__ int wave_incl_max(int x) {
    auto up = [&](uint32_t y) { x = max(x, (int)y); };
    up(dpp_u32_or_zero<0x111, 0xf>((uint32_t)x));
    up(dpp_u32_or_zero<0x112, 0xf>((uint32_t)x));
    up(dpp_u32_or_zero<0x114, 0xf>((uint32_t)x));
    up(dpp_u32_or_zero<0x118, 0xf>((uint32_t)x));
    up(dpp_u32_or_zero<0x142, 0xa>((uint32_t)x));
    up(dpp_u32_or_zero<0x143, 0xc>((uint32_t)x));
    return x;
}

// The runs, 64 at a time: lane x holds run 64 i + x. Run r is [S_r, S_{r+1}) with S_r the largest of runs[0 .. r] within [0, B], so
// they never overlap. Up to 64 stay in registers.
struct Runs {
    Run own;       // of the first 64
    int after;     // where those end
    __device__ __forceinline__ static Run load(const SharedArgs& a, int r0, int& before) {
        const int lane = threadIdx.x & 63, r = min(r0 + lane, a.R - 1);   // past the last: that one again, empty
        int upto = a.runs ? min(max(a.runs[r + 1], 0), a.B) : a.B;
        const int prefix = prefix_of(a, r);      // loaded with the bound, not behind it
        upto = max(wave_incl_max(upto), before);
        const int left = __shfl_up(upto, 1, 64), from = lane == 0 ? before : left;
        before = __builtin_amdgcn_readlane(upto, 63);
        return Run{from, upto - from, prefix};
    }
    __device__ __forceinline__ explicit Runs(const SharedArgs& a) {
        after = a.runs ? min(max(a.runs[0], 0), a.B) : 0;
        own = load(a, 0, after);
    }
    // step(64 runs, a lane's one each) until it returns true
    template <typename Step>
    __device__ __forceinline__ void walk(const SharedArgs& a, Step step) const {
        if (step(own)) return;
        int before = after;
        for (int r0 = 64; r0 < a.R; r0 += 64)
            if (step(load(a, r0, before))) return;
    }
};
// The shared positions of sequence b's run (0: none).
__device__ __forceinline__ int prefix_of_sequence(const SharedArgs& a, int b) {
    int found = 0;
    Runs(a).walk(a, [&](const Run& run) {
        const uint64_t hit = __ballot(run.count > 0 && run.first <= b && b < run.first + run.count);
        if (hit) found = __builtin_amdgcn_readlane(run.prefix, __builtin_ctzll(hit));
        return hit != 0;
    });
    return found;
}
// Whether all queries of sequence b see all of `prefix` positions; if not, it reads none of them in the shared part.
__device__ __forceinline__ bool sees(const SharedArgs& a, int b, int prefix) { return length_of(a, b) - a.T + 1 >= prefix; }

// What a workgroup does: `rows` rows from row r0 of `count` sequences from b0 on, over the blocks [i0, i1) of the keys [base, end)
// of sequence tb's table, its partials in slot `slot`. partials > 0: it says that the rows have so many of this part.
struct Item {
    int b0, tb, count, r0, rows, base, end, i0, i1, slot, partials, g;
    bool shared;
};

// A share is of 256 keys at least (16 answers on 8K: 28.5 us, with 128 keys 35.8)
constexpr int kLeastBlocks = 4, kLeastTiles = 8;
// More tiles than workgroups: tiles of fewer blocks go whole, in as many rounds as it takes, longer ones are shared out evenly.
// Even and whole, questions of 211 tokens: 20 on 2K 125 and 133 us, on 4K 198 and 224, on 16K 649 and 781; 36 on 2K 221 and
// 197, on 4K 330 and 307, on 8K 551 and 548, on 16K 1014 and 1034.
constexpr uint32_t kLongBlocks = 64;

// The shared part's workgroup `turn` of XCD `xcd`: a group, a run, a share of its blocks of kBlock keys, and a tile of kRows of its
// rows. The tiles that read the same keys lie next to each other, on one XCD. False: there are fewer.
template <int kRows, int kBlock, uint32_t kWorkers>
__device__ __forceinline__ bool shared_item(const SharedArgs& a, int xcd, int turn, Item& w) {
    auto tiles = [&](const Run& r) { return r.prefix > 0 ? (uint32_t)(((int64_t)r.count * a.T * a.h + kRows - 1) / kRows) : 0u; };
    auto blocks = [&](const Run& r) { return (uint32_t)(r.prefix + kBlock - 1) / kBlock; };
    auto sum = [&](uint32_t x) { return (uint32_t)__builtin_amdgcn_readlane((int)wave_incl_scan(x), 63); };
    // the blocks of all tiles (sums of 16, 24 and 24 bits of them), and of the longest
    const Runs runs(a);
    uint64_t total = 0;
    uint32_t longest = 1;
    runs.walk(a, [&](const Run& run) {
        const uint32_t n = tiles(run), k = blocks(run);
        const uint64_t own = (uint64_t)n * k;
        total += sum((uint32_t)own & 0xffffu) + ((uint64_t)sum((uint32_t)(own >> 16) & 0xffffffu) << 16) +
                 ((uint64_t)sum((uint32_t)(own >> 40)) << 40);
        longest = max(longest, (uint32_t)__builtin_amdgcn_readlane(wave_incl_max(n ? (int)k : 0), 63));
        return false;
    });
    // a share: even over the workgroups in as many rounds as the tiles would take whole. In several rounds only where a tile is
    // long enough for a second partial of its rows to pay
    total *= a.G;
    uint32_t share = longest;
    if (total <= (uint64_t)kWorkers * longest) {
        share = (uint32_t)((total + kWorkers - 1) / kWorkers);
    } else if (longest >= kLongBlocks && total < (uint64_t)kWorkers * longest * 8) {
        const uint32_t rounds = (uint32_t)((total + (uint64_t)kWorkers * longest - 1) / ((uint64_t)kWorkers * longest));
        share = (uint32_t)(total / ((uint64_t)kWorkers * rounds)) + 1;
    }
    const uint32_t least = max((longest + a.shared - 1) / a.shared, (uint32_t)(kBlock == kKeys ? kLeastBlocks : kLeastTiles));
    share = min(longest, max(share, least));
    // whole shares of a group, and pieces
    uint32_t whole = 0, pieces = 0;
    runs.walk(a, [&](const Run& run) {
        const uint32_t n = tiles(run), k = blocks(run);
        whole += sum(n * (k / share));
        pieces += sum(k % share ? n : 0u);
        return false;
    });
    const uint32_t turns = (whole * a.G + 7) / 8, piece_turns = (pieces * a.G + 7) / 8;
    const bool piece = (uint32_t)turn >= turns;
    const uint32_t lin = piece ? xcd * piece_turns + turn - turns : xcd * turns + turn, group = piece ? pieces : whole;
    if (piece && (uint32_t)turn - turns >= piece_turns) return false;
    if (lin >= group * a.G) return false;
    w.g = (int)(lin / group);
    uint32_t rest = lin - w.g * group;
    runs.walk(a, [&](const Run& run) {
        const uint32_t n = tiles(run), k = blocks(run), full = k / share, mine = piece ? (k % share ? n : 0u) : n * full;
        const uint32_t upto = wave_incl_scan(mine);
        const uint64_t hit = __ballot(upto > rest);
        if (!hit) {
            rest -= (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
            return false;
        }
        const int x = __builtin_ctzll(hit);
        auto of = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, x); };
        const uint32_t at = rest - of(upto - mine), part = piece ? of(full) : at / of(n), tile = piece ? at : at - part * of(n);
        w.b0 = (int)of(run.first);
        w.count = (int)of(run.count);
        w.end = (int)of(run.prefix);
        w.r0 = (int)tile * kRows;
        w.slot = (int)part;
        w.i0 = (int)(part * share);
        w.i1 = (int)min((uint32_t)w.i0 + share, of(k));
        w.partials = part == 0 ? (int)((of(k) + share - 1) / share) : 0;
        return true;
    });
    // The table of the first sequence that sees the whole prefix: one that has ended or been cut back need not name its pages any
    // more. None: nothing to read, but the rows are to be told so.
    const int lane = threadIdx.x & 63;
    w.tb = -1;
    for (int b = 0; b < w.count && w.tb < 0; b += 64) {
        const uint64_t hit = __ballot(b + lane < w.count && sees(a, w.b0 + min(b + lane, w.count - 1), w.end));
        if (hit) w.tb = w.b0 + b + (int)__builtin_ctzll(hit);
    }
    if (w.tb < 0) {
        w.tb = w.b0;
        w.i1 = w.i0;
    }
    w.rows = (int)min((int64_t)w.count * a.T * a.h - w.r0, (int64_t)kRows);
    w.base = 0;
    w.shared = true;
    return true;
}

// The own part: false where the sequence has no keys for this split.
template <int kRows, int kBlock>
__device__ __forceinline__ bool own_item(const SharedArgs& a, int lin, Item& w) {
    const int tiles = (a.T * a.h + kRows - 1) / kRows;
    const int split = lin % a.own;
    lin /= a.own;
    w.r0 = (tiles - 1 - lin % tiles) * kRows;   // later queries read more keys: first
    lin /= tiles;
    w.g = lin % a.G;
    w.tb = w.b0 = lin / a.G;
    w.count = 1;
    w.rows = min(a.T * a.h - w.r0, kRows);
    const int n = length_of(a, w.b0), prefix = a.shared ? prefix_of_sequence(a, w.b0) : 0;
    w.base = n - a.T + 1 >= prefix ? prefix : 0;
    w.end = max(n - a.T + min(a.T - 1, (w.r0 + kRows - 1) / a.h) + 1, w.base);
    const int blocks = (w.end - w.base + kBlock - 1) / kBlock;
    const int share = max((blocks + a.own - 1) / a.own, kBlock == kKeys ? kLeastBlocks : kLeastTiles);
    w.i0 = split * share;
    if (split > 0 && w.i0 >= blocks) return false;
    w.i1 = min(w.i0 + share, blocks);
    w.slot = a.shared + split;
    w.partials = split == 0 ? max((blocks + share - 1) / share, 1) : 0;
    w.shared = false;
    // nobody else counts the shared partials of a sequence that shares nothing
    if (a.part && prefix == 0 && split == 0)
        for (int x = threadIdx.x; x < w.rows; x += 64 * kWaves) {
            const int t = (w.r0 + x) / a.h, head = w.r0 + x - t * a.h;
            a.counts[(((size_t)w.b0 * a.G + w.g) * a.h + head) * a.T + t].x = 0;
        }
    return true;
}
// A row's count of this part's partials: none where the sequence takes no part in the shared read.
__device__ __forceinline__ void count_partials(const SharedArgs& a, const Item& w, size_t row, bool dead) {
    if (w.shared) a.counts[row].x = dead ? 0 : w.partials;
    else a.counts[row].y = w.partials;
}

struct Row {
    int b, t, head;
    __device__ __forceinline__ Row(const SharedArgs& a, const Item& w, int r) {
        const int x = w.r0 + min(r, w.rows - 1), th = a.T * a.h, s = x / th, y = x - s * th;
        b = w.b0 + s;
        t = y / a.h;
        head = y - t * a.h;
    }
    __device__ __forceinline__ size_t at(const SharedArgs& a, int g) const {
        return (((size_t)b * a.G + g) * a.h + head) * a.T + t;
    }
};

// The address of key `key`'s row in page p of group g, `chunk` bytes in; zeros where p names none.
__device__ __forceinline__ const char* key_row(const SharedArgs& a, const uint16_t* pool, int p, int g, int key, int chunk) {
    const bool ok = (uint32_t)p < (uint32_t)a.pages;
    const size_t row = (((size_t)(ok ? p : 0) * a.G + g) << a.shift) + (key & ((1 << a.shift) - 1));
    uint64_t at = reinterpret_cast<uint64_t>(pool) + row * (2 * kDim) + chunk;
    asm volatile("" : "+v"(at));   // computed by every lane: a select, not a branch
    return reinterpret_cast<const char*>(ok ? at : reinterpret_cast<uint64_t>(shared_zeros));
}
// Sixteen rows of a page from key k16 on, or fewer up to `end`, or none: where they lie and how many bytes.
struct Sixteen {
    size_t at;
    uint32_t rows;
    __device__ __forceinline__ Sixteen(const SharedArgs& a, int p, int g, int k16, int end) {
        // uniform, and in scalar registers: with a descriptor in vector ones every load is a loop over its values (16 questions
        // on 16K: 503 us, and 459)
        auto scalar = [](uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); };
        rows = scalar((uint32_t)p < (uint32_t)a.pages ? (uint32_t)min(max(end - k16, 0), 16) : 0u);
        at = (size_t)scalar((((uint32_t)p * a.G + g) << a.shift) + (k16 & ((1 << a.shift) - 1))) * kDim;
    }
    __device__ __forceinline__ uint32_t bytes() const { return rows * 2 * kDim; }
    __device__ __forceinline__ uint32_t have() const { return (1u << rows) - 1u; }
};

// The scale (log2 domain), made positive: a negative one flips the sign of q instead (exact), and zero becomes the smallest normal
// float, which gives the same weights while a masked key's -inf * scale stays -inf.
__device__ __forceinline__ float positive_scale(float x) { return x == 0.0f ? FLT_MIN : fabsf(x); }

// What rounding x and y to the pair `w` left, a bf16 pair too.
__device__ __forceinline__ uint32_t rest_of(float x, float y, uint32_t w) { return pack_bf16x2(x - bf16_lo(w), y - bf16_hi(w)); }

__device__ __forceinline__ uint32_t bf16x2_finite(uint32_t w, uint32_t& flags) {   // NaN and infinity zeroed, and flagged 1.0
    const uint32_t lo = (w & 0x00007f80u) == 0x00007f80u ? 0x0000ffffu : 0u;
    const uint32_t hi = (w & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u;
    flags = (lo & 0x3f80u) | (hi & 0x3f800000u);
    return w & ~(lo | hi);
}

// K and V blocks in LDS: 64 rows of 16 16-byte chunks, permuted within the row so that the reads meet no bank twice: K's chunk c of
// row j at slot c ^ (j & 15) (a read takes 16 rows, one chunk), V's at c ^ (4 (j & 3)) (a transposing read takes 4 chunks of 4
// consecutive rows). Key 16 z + 8 g + 4 a + b of a 32-key tile is row 16 z + 8 a + 4 g + b of its product, so that a lane's weights
// are those of eight consecutive keys, the ones whose V its operand holds.
// ONE: one query a sequence, of which only the shared part is read here, and the weights' rest has its product with V.
template <bool SMALL, bool ONE>
__device__ __forceinline__ void wide(const SharedArgs& a, const Item& w, char* kt0, char* vt0, char* kt1, char* vt1, int& again) {
    constexpr int kRow = 2 * kDim;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, g = lane >> 5;
    const int R = 32 * wave + n;
    const Row row(a, w, R);              // rows past the last repeat it and are not written
    bf16x8_t qb[8];
    {
        const uint16_t* qr = a.q + row.at(a, w.g) * kDim;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
            qb[kk] = __builtin_bit_cast(bf16x8_t, *reinterpret_cast<const u32x4_t*>(qr + 16 * kk + 8 * g));
    }
    // keys before `lim` are this lane's row's; the least and the most of the wave's rows
    const int len = w.shared ? 0 : length_of(a, w.b0);
    auto limit = [&](int r) { return w.shared ? INT32_MAX : len - a.T + min(w.r0 + min(r, w.rows - 1), a.T * a.h - 1) / a.h + 1; };
    // (a wave without a row of its own only copies)
    const int lim = limit(R), lim_min = limit(32 * wave), lim_max = 32 * wave < w.rows ? limit(32 * wave + 31) : 0;
    const bool dead = w.shared && !sees(a, row.b, w.end);

    // staging: a load of a wave fills 1 KB of a tile, four rows, lane l slot l % 16 of row l / 16 of them
    const int srow = lane >> 4, slot = lane & 15;
    const int kchunk = 16 * (slot ^ (4 * wave + srow)), vchunk = 16 * (slot ^ (4 * srow));
    const int32_t* pages = a.table + (size_t)w.tb * a.table_stride;
    auto first_key = [&](int i) { return w.base + kKeys * i; };
    const int stop = min(w.end, first_key(w.i1));
    // the entries of block i's pages, as they stand in the table: lane u of four that of keys 16 u .., or lane j key j's
    auto look = [&](int i) {
        const int key = first_key(min(i, w.i1 - 1)) + (SMALL ? lane : 16 * (lane & 3));
        return pages[min(key, w.end - 1) >> a.shift];
    };
    // block i's copies, and the entries of the next one's pages; which of the block's keys have a row, a bit each
    // (the entries leave their register before the next ones are loaded into it: moved there later, they would be waited for)
    int next = 0;
    auto issue = [&](int i, char* kt, char* vt) -> uint64_t {
        const int kb = first_key(i);
        if constexpr (SMALL) {
            const int page = kb + lane < stop ? next : -1;
            __builtin_amdgcn_sched_barrier(0);
            next = look(i + 1);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int j = 16 * u + 4 * wave + srow, p = __shfl(page, j, 64);
                load_lds16(reinterpret_cast<const uint16_t*>(key_row(a, a.K, p, w.g, kb + j, kchunk)),
                           reinterpret_cast<uint16_t*>(kt + 4096 * u + 1024 * wave));
                load_lds16(reinterpret_cast<const uint16_t*>(key_row(a, a.V, p, w.g, kb + j, vchunk)),
                           reinterpret_cast<uint16_t*>(vt + 4096 * u + 1024 * wave));
            }
            return __ballot((uint32_t)page < (uint32_t)a.pages);
        } else {
            uint64_t have = 0;
            const uint32_t at = kRow * (4 * wave + srow);
            int entry[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                entry[u] = __builtin_amdgcn_readlane(next, u);
                asm volatile("" : "+s"(entry[u]));
            }
            __builtin_amdgcn_sched_barrier(0);
            next = look(i + 1);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const Sixteen r(a, entry[u], w.g, kb + 16 * u, stop);
                load_lds16_buf(a.K + r.at, r.bytes(), at + kchunk, reinterpret_cast<uint16_t*>(kt + 4096 * u + 1024 * wave));
                load_lds16_buf(a.V + r.at, r.bytes(), at + vchunk, reinterpret_cast<uint16_t*>(vt + 4096 * u + 1024 * wave));
                have |= (uint64_t)r.have() << (16 * u);
            }
            return have;
        }
    };
    // operand reads, as byte offsets into a tile. K: this lane's key of a 32-key tile, chunk 2 kk + g. V: rows 16 ks + 8 g + 4 hf +
    // e, dims 32 dt + 16 (lane / 16 % 2) + 4 j .. + 3, e = lane % 16 / 4, j = lane % 4. `pin` keeps the compiler from holding
    // a copy of each per tile.
    const int key = (n & 16) + 8 * ((n >> 2) & 1) + 4 * ((n >> 3) & 1) + (n & 3);
    uint32_t kof[8], vof[4];
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) kof[kk] = kRow * key + 16 * ((2 * kk + g) ^ (key & 15));
    const int ve = (lane & 15) >> 2;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) vof[dt] = kRow * (8 * g + ve) + 64 * (dt ^ ve) + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
    auto pin = [&]() {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) asm volatile("" : "+v"(kof[kk]));
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) asm volatile("" : "+v"(vof[dt]));
    };

    float m_run = -INFINITY, l_run = 0.0f;
    const float sc = positive_scale(a.scale_log2);
    if (a.scale_log2 < 0.0f) {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
            qb[kk] = __builtin_bit_cast(bf16x8_t, __builtin_bit_cast(u32x4_t, qb[kk]) ^ 0x80008000u);
    }
    f32x16_t o[4];
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[dt][i] = 0.0f;

    // `have`: the block's keys that have a row to read, a bit each
    auto block = [&](auto careful, int kb, uint64_t have, const char* ks, const char* vs) __attribute__((always_inline)) {
        if (kb >= lim_max || have == 0) return;
        const bool ahead = !ONE && kb + kKeys > lim_min, gaps = ~have != 0;
        auto value = [&](int ks2, int dt) -> bf16x8_t {   // V^T's operand of 16-key step ks2, dims 32 dt ..
            const char* vp = vs + 16 * kRow * ks2 + vof[dt];
            const u32x2v_t lo4 = read_tr16(vp), hi4 = read_tr16(vp + 4 * kRow);
            return __builtin_bit_cast(bf16x8_t, u32x4_t{lo4.x, lo4.y, hi4.x, hi4.y});
        };
        bool spoilt = false;   // some V of a block with keys that only some rows see is NaN or infinite
        if (careful && ahead) {
            float chk = 0.0f;  // 0 times it, which is NaN
#pragma unroll
            for (int ks2 = 0; ks2 < 4; ++ks2)
#pragma unroll
                for (int dt = 0; dt < 4; ++dt) {
                    const u32x4_t x = __builtin_bit_cast(u32x4_t, value(ks2, dt));
                    chk = dot2_bf16(x.x, 0u, chk);
                    chk = dot2_bf16(x.y, 0u, chk);
                    chk = dot2_bf16(x.z, 0u, chk);
                    chk = dot2_bf16(x.w, 0u, chk);
                    __builtin_amdgcn_sched_barrier(0);   // an operand at a time: registers
                }
            spoilt = __any(chk != 0.0f);
        }
        f32x16_t s[2];
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[x][i] = 0.0f;
        constexpr int kAhead = 3;   // steps that K's reads are ahead of their products
        u32x4_t kw[8][2];
        auto read_k = [&](int kk) __attribute__((always_inline)) {
#pragma unroll
            for (int x = 0; x < 2; ++x) kw[kk][x] = *reinterpret_cast<const u32x4_t*>(ks + 32 * kRow * x + kof[kk]);
        };
#pragma unroll
        for (int kk = 0; kk < kAhead; ++kk) read_k(kk);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
#pragma unroll
            for (int x = 0; x < 2; ++x)
                s[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, kw[kk][x]), qb[kk], s[x], 0, 0, 0);
            if (kk + kAhead < 8) {
                read_k(kk + kAhead);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        // this lane's scores: row R, keys kb + 8 g + c, c = 32 x + 16 (i / 8) + i % 8
        if (ahead) {
            const int most = lim - 1 - kb - 8 * g;
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[x][i] = 32 * x + 16 * (i >> 3) + (i & 7) <= most ? s[x][i] : -INFINITY;
        }
        if (gaps) {
            const uint64_t mine = have >> (8 * g);
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    s[x][i] = (uint32_t)(mine >> (32 * x)) & 1u << (16 * (i >> 3) + (i & 7)) ? s[x][i] : -INFINITY;
        }
        uint32_t see = 0;   // a spoilt block's visible keys, a bit for each of this lane's scores
        if (careful && spoilt) {
#pragma unroll
            for (int i = 0; i < 32; ++i) see |= s[i >> 4][i & 15] == -INFINITY ? 0u : 1u << i;
        }
        float bm = -INFINITY;
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int i = 0; i < 16; ++i) bm = fmaxf(bm, s[x][i]);
        bm = max_xor32(bm) * sc;
        if (bm > m_run) {   // also the first keys of the row (m_run = -inf)
            bm += kLazy;
            const float al = fast_exp2(m_run - bm);   // exp2(-inf) = 0
            l_run *= al;
#pragma unroll
            for (int dt = 0; dt < 4; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[dt][i] *= al;
            m_run = bm;
        }
        bf16x8_t pb[4], rest[ONE ? 4 : 1];
        const float nm = m_run == -INFINITY ? 0.0f : -m_run;   // no score above -inf yet: weights 0, or NaN for a NaN score
#pragma unroll
        for (int ks2 = 0; ks2 < 4; ++ks2) {
            uint32_t w4[4], r4[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x0 = s[ks2 >> 1][8 * (ks2 & 1) + 2 * e], x1 = s[ks2 >> 1][8 * (ks2 & 1) + 2 * e + 1];
                const float p0 = fast_exp2(fmaf(x0, sc, nm));
                const float p1 = fast_exp2(fmaf(x1, sc, nm));
                l_run += p0 + p1;
                w4[e] = pack_bf16x2(p0, p1);
                if constexpr (ONE) r4[e] = rest_of(p0, p1, w4[e]);
            }
            pb[ks2] = __builtin_bit_cast(bf16x8_t, u32x4_t{w4[0], w4[1], w4[2], w4[3]});
            if constexpr (ONE) rest[ks2] = __builtin_bit_cast(bf16x8_t, u32x4_t{r4[0], r4[1], r4[2], r4[3]});
        }
        if (!careful || !spoilt) {
#pragma unroll
            for (int ks2 = 0; ks2 < 4; ++ks2)
#pragma unroll
                for (int dt = 0; dt < 4; ++dt) {
                    const bf16x8_t v = value(ks2, dt);
                    o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, pb[ks2], o[dt], 0, 0, 0);
                    if constexpr (ONE) o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, rest[ks2], o[dt], 0, 0, 0);
                }
        } else {   // the finite values' products, and NaN where a visible key's value is not finite
#pragma unroll
            for (int dt = 0; dt < 4; ++dt) {
                f32x16_t f;
#pragma unroll
                for (int i = 0; i < 16; ++i) f[i] = 0.0f;
#pragma unroll
                for (int ks2 = 0; ks2 < 4; ++ks2) {
                    u32x4_t v = __builtin_bit_cast(u32x4_t, value(ks2, dt)), flag, one;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint32_t bits;
                        v[e] = bf16x2_finite(v[e], bits);
                        flag[e] = bits;
                        const uint32_t two = see >> (8 * ks2 + 2 * e);
                        one[e] = (two & 1u ? 0x3f80u : 0u) | (two & 2u ? 0x3f800000u : 0u);
                    }
                    o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, v), pb[ks2], o[dt], 0, 0, 0);
                    f = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, flag),
                                                                __builtin_bit_cast(bf16x8_t, one), f, 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) o[dt][i] = f[i] > 0.0f ? __builtin_nanf("") : o[dt][i];
            }
        }
    };
    // Two tile pairs: the next block's copies are issued when every wave has left the tiles they overwrite, the barrier that also
    // publishes the current block, and land while it is computed; its pages were looked up a block before that. Past the last block
    // there is nothing to copy (no rows, no traffic), and the copies are issued all the same: a wait behind a branch is for the
    // most that either side may have left, which would be for the copies that are to be on their way (us, of single weights, with the branch and
    // without: 16 answers, h=8, on 32K 47.3 and 44.5, on 128K 135 and 121; 8 x 4, h=4, on 16K 110 and 100; 16 questions on 16K
    // 467 and 461; the own part's workgroups beside it lose: 4 x 13 answers, h=8, on 9K 66.2 and 67.7, 2 x 30, h=4, on 16K 52.8
    // and 55.3).
    uint64_t have = 0;
    auto publish = [&](auto left) {   // this wave's copies have landed but for the last `left` loads, and its reads are done
        if constexpr (decltype(left)::value == 8) __builtin_amdgcn_s_waitcnt(0x0078);   // vmcnt(8) lgkmcnt(0)
        else __builtin_amdgcn_s_waitcnt(0x0070);                                        // vmcnt(0) lgkmcnt(0)
        asm volatile("s_barrier" ::: "memory");
        pin();
    };
    using All = std::integral_constant<int, 0>;
    using Eight = std::integral_constant<int, 8>;
    if (tid == 0) again = 0;   // published by the first block's barrier
    if (w.i0 < w.i1) {
        next = look(w.i0);
        have = issue(w.i0, kt0, vt0);
        // q has landed, with the entries behind it: said here, as a wait for it in the loop would be one for the copies
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) asm volatile("" : "+v"(qb[kk]));
        __builtin_amdgcn_sched_barrier(0);   // in this order: the wait for the first block's counts the second's eight
        uint64_t now = have;
        have = issue(w.i0 + 1, kt1, vt1);
        publish(Eight{});
        block(std::false_type{}, first_key(w.i0), now, kt0, vt0);
        for (int i = w.i0 + 1; i < w.i1; i += 2) {
            publish(All{});
            now = have;
            have = issue(i + 1, kt0, vt0);
            block(std::false_type{}, first_key(i), now, kt1, vt1);
            if (i + 1 >= w.i1) break;
            publish(All{});
            now = have;
            have = issue(i + 2, kt1, vt1);
            block(std::false_type{}, first_key(i + 1), now, kt0, vt0);
        }
        __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0): nothing is written to LDS behind the last block
    }
    // A result that is not finite: a visible key's doing, or zero weights times one that only later queries see. All rows
    // again, with the blocks that have such keys looked over. The shared part has none.
    if (!ONE && !w.shared) {
        float finite = 0.0f * l_run;
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) finite = fmaf(0.0f, o[dt][i], finite);
        __syncthreads();   // `again` is set, with or without a block
        if (__any(finite != 0.0f) && lane == 0) again = 1;
        __syncthreads();
        if (again) {
            m_run = -INFINITY;
            l_run = 0.0f;
#pragma unroll
            for (int dt = 0; dt < 4; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[dt][i] = 0.0f;
            if (w.i0 < w.i1) next = look(w.i0);
            for (int i = w.i0; i < w.i1; ++i) {
                have = issue(i, kt0, vt0);
                publish(All{});
                block(std::true_type{}, first_key(i), have, kt0, vt0);
                __syncthreads();
            }
        }
    }
    const float l_tot = l_run + shfl_xor_f32(l_run, 32);
    if (R >= w.rows) return;
    if (a.part) {
        const size_t at = row.at(a, w.g);
        float* pp = a.part + (at * (a.shared + a.own) + w.slot) * kPart;
        if (g == 0) {
            pp[0] = m_run;
            pp[1] = l_tot;
            if (w.partials) count_partials(a, w, at, dead);
        }
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4)
                *reinterpret_cast<float4*>(pp + 4 + 32 * dt + 8 * i4 + 4 * g) =
                    make_float4(o[dt][4 * i4], o[dt][4 * i4 + 1], o[dt][4 * i4 + 2], o[dt][4 * i4 + 3]);
        return;
    }
    const float inv = l_tot == 0.0f ? 0.0f : 1.0f / l_tot;
    uint16_t* orow = a.out + row.at(a, w.g) * kDim;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4)   // dims 32 dt + 8 i4 + 4 g + 0..3
            *reinterpret_cast<u32x2v_t*>(orow + 32 * dt + 8 * i4 + 4 * g) =
                u32x2v_t{pack_bf16x2(o[dt][4 * i4] * inv, o[dt][4 * i4 + 1] * inv),
                         pack_bf16x2(o[dt][4 * i4 + 2] * inv, o[dt][4 * i4 + 3] * inv)};
}

// `low`, `high`: 32 KB of LDS in two halves, a wave's V tile in 8 KB of them, then the merge. AHEAD: a tile is on its way while
// another is computed, where registers allow it anyway.
struct Tile {
    u32x4_t k[2][4], v[8];
    uint32_t have;
};
template <bool SMALL, bool AHEAD>
__device__ __forceinline__ void narrow(const SharedArgs& a, const Item& w, char* low, char* high, float (*ml_sh)[kNarrow][2]) {
    constexpr int kRow = 2 * kDim;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n16 = lane & 15, g4 = lane >> 4;
    auto tile_of = [&](int x) { return (x < 2 ? low : high) + kTile * kRow * (x & 1); };
    // Q^T as the B operand: column n16 is the workgroup's row n16 (past the last: that one again)
    bf16x8_t qb[4];
    const float sc = positive_scale(a.scale_log2);
    {
        const uint16_t* qr = a.q + Row(a, w, n16).at(a, w.g) * kDim + 8 * g4;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            u32x4_t x = *reinterpret_cast<const u32x4_t*>(qr + 32 * kk);
            if (a.scale_log2 < 0.0f) x ^= 0x80008000u;
            qb[kk] = __builtin_bit_cast(bf16x8_t, x);
        }
    }
    // Tile t2 of a product holds keys 16 t2 .. + 15, so a lane's weights are of keys 4 g4 .. + 3 and 16 + 4 g4 .. + 3: the rows
    // whose V it reads. V in LDS: chunk c of row r at c ^ (4 (r % 4)), so that the rows a transposing read takes together lie in
    // different banks (lane 4 e + j of 16 reads four elements of row 4 g4 + e, and gets 4 rows).
    const int vrow = lane >> 4;
    char* vt = tile_of(wave);
    const int vst = kRow * vrow + 16 * (n16 ^ (4 * vrow));
    int vof = kRow * (4 * g4 + (n16 >> 2)) + 64 * (n16 >> 2) + 8 * (n16 & 3);   // dims 32 x .. at vof ^ 64 x

    float m = -INFINITY, l = 0.0f;
    f32x4_t o[8];
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) o[dt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

    const int32_t* pages = a.table + (size_t)w.tb * a.table_stride;
    auto look = [&](int i) {
        const int key = w.base + kTile * min(i, w.i1 - 1) + (SMALL ? lane & 31 : 16 * (lane & 1));
        return pages[min(key, w.end - 1) >> a.shift];
    };
    int next = w.i0 < w.i1 ? look(w.i0 + wave) : 0;
    auto issue = [&](int i, Tile& f) {   // tile i's loads, and the pages of the wave's next one
        const int entry = next, kb = w.base + kTile * i;
        next = look(i + kWaves);
        if constexpr (SMALL) {
            const int page = kb + (lane & 31) < w.end ? entry : -1;
#pragma unroll
            for (int t2 = 0; t2 < 2; ++t2) {
                const int j = 16 * t2 + n16;
                const char* r = key_row(a, a.K, __shfl(page, j, 64), w.g, kb + j, 16 * g4);
                const int step = r == reinterpret_cast<const char*>(shared_zeros) ? 0 : 64;
#pragma unroll
                for (int c = 0; c < 4; ++c) f.k[t2][c] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(r + step * c));
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int j = 4 * u + vrow;
                f.v[u] = __builtin_nontemporal_load(
                    reinterpret_cast<const u32x4_t*>(key_row(a, a.V, __shfl(page, j, 64), w.g, kb + j, 16 * n16)));
            }
            f.have = (uint32_t)__ballot((uint32_t)page < (uint32_t)a.pages);
        } else {
            constexpr int kNt = 2;   // non-temporal
            f.have = 0;
#pragma unroll
            for (int t2 = 0; t2 < 2; ++t2) {
                const Sixteen r(a, __builtin_amdgcn_readlane(entry, t2), w.g, kb + 16 * t2, w.end);
                const __amdgpu_buffer_rsrc_t kr =
                    __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(a.K + r.at), 0, (int)r.bytes(), 0x00020000);
                const __amdgpu_buffer_rsrc_t vr =
                    __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(a.V + r.at), 0, (int)r.bytes(), 0x00020000);
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    f.k[t2][c] = __builtin_bit_cast(
                        u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(kr, kRow * n16 + 16 * g4 + 64 * c, 0, kNt));
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    f.v[4 * t2 + u] = __builtin_bit_cast(
                        u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(vr, 16 * lane + 1024 * u, 0, kNt));
                f.have |= r.have() << (16 * t2);
            }
        }
        __builtin_amdgcn_sched_barrier(0);   // every load is on its way before the first result is waited for
    };
    auto compute = [&](const Tile& f) {
        const uint32_t have = f.have;
        asm volatile("" : "+v"(vof));   // its other forms are made where they are used: registers
        f32x4_t sv[2];
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
            sv[t2] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
                sv[t2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, f.k[t2][kk]), qb[kk], sv[t2], 0, 0,
                                                                0);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) *reinterpret_cast<u32x4_t*>(vt + vst + 1024 * u) = f.v[u];
        // this lane's scores: column n16, keys 16 t2 + 4 g4 + e
        if (~have) {
#pragma unroll
            for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (!(have >> (16 * t2 + 4 * g4 + e) & 1)) sv[t2][e] = -INFINITY;
        }
        float bm = -INFINITY;
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
            for (int e = 0; e < 4; ++e) bm = fmaxf(bm, sv[t2][e]);
        if (__any(bm * sc > m)) {
            bm = max_xor32(max_xor16(bm)) * sc;
            if (bm > m) {   // also a column's first rows (m = -inf)
                bm += kLazy;
                const float al = fast_exp2(m - bm);
                l *= al;
#pragma unroll
                for (int dt = 0; dt < 8; ++dt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[dt][e] *= al;
                m = bm;
            }
        }
        const float nm = m == -INFINITY ? 0.0f : -m;   // no score above -inf yet: every weight 0
        float pr[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) pr[e] = fast_exp2(fmaf(sv[e >> 2][e & 3], sc, nm));
        l += ((pr[0] + pr[1]) + (pr[2] + pr[3])) + ((pr[4] + pr[5]) + (pr[6] + pr[7]));
        // a wave's LDS operations take effect in order; these keep the compiler from moving them past each other
        asm volatile("" ::: "memory");
        uint32_t w4[4], r4[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            w4[e] = pack_bf16x2(pr[2 * e], pr[2 * e + 1]);
            r4[e] = rest_of(pr[2 * e], pr[2 * e + 1], w4[e]);
        }
        const bf16x8_t pb = __builtin_bit_cast(bf16x8_t, u32x4_t{w4[0], w4[1], w4[2], w4[3]});
        const bf16x8_t rest = __builtin_bit_cast(bf16x8_t, u32x4_t{r4[0], r4[1], r4[2], r4[3]});
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
            const char* r = vt + (vof ^ 64 * (dt >> 1)) + 32 * (dt & 1);
            const u32x2v_t w0 = read_tr16(r), w1 = read_tr16(r + 16 * kRow);
            const bf16x8_t v = __builtin_bit_cast(bf16x8_t, u32x4_t{w0.x, w0.y, w1.x, w1.y});
            o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pb, o[dt], 0, 0, 0);
            o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, rest, o[dt], 0, 0, 0);
            if constexpr (AHEAD) __builtin_amdgcn_sched_barrier(0);   // an operand at a time: registers
        }
        asm volatile("" ::: "memory");
    };
    int i = w.i0 + wave;
    if constexpr (AHEAD) {
        Tile f0, f1;
        if (i < w.i1) issue(i, f0);
        for (; i < w.i1; i += 2 * kWaves) {
            if (i + kWaves < w.i1) issue(i + kWaves, f1);
            compute(f0);
            if (i + kWaves >= w.i1) break;
            if (i + 2 * kWaves < w.i1) issue(i + 2 * kWaves, f0);
            compute(f1);
        }
    } else {
        for (; i < w.i1; i += kWaves) {
            Tile f;
            issue(i, f);
            compute(f);
        }
    }
    l += shfl_xor_f32(l, 16);
    l += shfl_xor_f32(l, 32);

    // the waves' (m, l, O) through LDS: [row][dim] floats in each wave's V tile
    static_assert(kTile * kRow >= kNarrow * kDim * sizeof(float), "the merge lies in the V tiles");
    __syncthreads();
    if (g4 == 0) {
        ml_sh[wave][n16][0] = m;
        ml_sh[wave][n16][1] = l;
    }
#pragma unroll
    for (int dt = 0; dt < 8; ++dt)
        *reinterpret_cast<f32x4_t*>(reinterpret_cast<float*>(vt) + n16 * kDim + 16 * dt + 4 * g4) = o[dt];
    __syncthreads();
    for (int r = wave; r < w.rows; r += kWaves) {   // wave -> row, lane l -> dims 2 l, 2 l + 1
        const Row row(a, w, r);
        float ms = -INFINITY;
#pragma unroll
        for (int x = 0; x < kWaves; ++x) ms = fmaxf(ms, ml_sh[x][r][0]);
        float ls = 0.0f;
        float2 os = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int x = 0; x < kWaves; ++x) {
            const float mx = ml_sh[x][r][0], lx = ml_sh[x][r][1];
            const float y = mx == -INFINITY ? (lx == 0.0f ? 0.0f : 1.0f) : fast_exp2(mx - ms);
            const float2 v = *reinterpret_cast<const float2*>(reinterpret_cast<const float*>(tile_of(x)) + r * kDim + 2 * lane);
            ls += y * lx;
            os.x += y * v.x;
            os.y += y * v.y;
        }
        if (a.part) {
            const size_t at = row.at(a, w.g);
            float* pp = a.part + (at * (a.shared + a.own) + w.slot) * kPart;
            if (lane == 0) {
                pp[0] = ms;
                pp[1] = ls;
                if (w.partials) count_partials(a, w, at, w.shared && !sees(a, row.b, w.end));
            }
            *reinterpret_cast<float2*>(pp + 4 + 2 * lane) = os;
        } else {
            const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
            *reinterpret_cast<uint32_t*>(a.out + row.at(a, w.g) * kDim + 2 * lane) = pack_bf16x2(os.x * inv, os.y * inv);
        }
    }
}

// Both parts, the shared one by tiles of 128 rows (WIDE) or 16, the own one too (OWN_WIDE).
template <bool WIDE, bool OWN_WIDE, bool SMALL>
__global__ __launch_bounds__(64 * kWaves, WIDE ? 2 : 3) void shared_read(SharedArgs a) {
    static_assert(WIDE || !OWN_WIDE, "several queries of a sequence are read wide in both parts");
    __shared__ __attribute__((aligned(1024))) char t0[kKeys * 2 * kDim], t1[kKeys * 2 * kDim];
    __shared__ __attribute__((aligned(1024))) char t2[WIDE ? kKeys * 2 * kDim : 1], t3[WIDE ? kKeys * 2 * kDim : 1];
    __shared__ float ml_sh[kWaves][kNarrow][2];
    __shared__ int again;
    // each XCD an eighth of either part's items, in line, the shared part's, which are longer, first
    const int xcd = blockIdx.x & 7, turn = blockIdx.x >> 3;
    const bool first = turn < a.shared_turns;
    const int own = __builtin_amdgcn_readfirstlane(xcd * a.own_turns + turn - a.shared_turns);
    if (!first && own >= a.own_items) return;
    Item w;
    if constexpr (WIDE && !OWN_WIDE) {
        if (first) {
            if (shared_item<kWide, kKeys, kMixedWorkers>(a, xcd, turn, w)) wide<SMALL, true>(a, w, t0, t1, t2, t3, again);
        } else {
            if (own_item<kNarrow, kTile>(a, own, w)) narrow<SMALL, !SMALL>(a, w, t0, t1, ml_sh);
        }
    } else {
        constexpr int kRows = WIDE ? kWide : kNarrow, kBlock = WIDE ? kKeys : kTile;
        constexpr uint32_t kWorkers = WIDE ? kWideWorkers : kNarrowWorkers;
        if (!(first ? shared_item<kRows, kBlock, kWorkers>(a, xcd, turn, w) : own_item<kRows, kBlock>(a, own, w))) return;
        if constexpr (WIDE) wide<SMALL, false>(a, w, t0, t1, t2, t3, again);
        else narrow<SMALL, false>(a, w, t0, t1, ml_sh);
    }
}

// A row's partials merged by GROUPS half waves, each every GROUPS-th of them: lane -> four dims, and the weight of every 32nd.
template <int GROUPS>
__global__ __launch_bounds__(256) void shared_combine(const float* part, const int2* counts, uint16_t* out, int shared, int slots,
                                                      int64_t rows) {
    constexpr int kHold = 2 * kMaxSplits / 32, kAhead = 4;
    __shared__ __attribute__((aligned(16))) float sum_sh[8][kDim];
    const int half = threadIdx.x >> 5, lane = threadIdx.x & 31, group = half % GROUPS;
    const int64_t row = min((int64_t)blockIdx.x * (8 / GROUPS) + half / GROUPS, rows - 1);   // past the last: that one again
    const float* pp = part + row * slots * kPart;
    const int2 n = counts[row];
    const int count = min(n.x, shared) + min(n.y, slots - shared);
    auto slot = [&](int x) { return (size_t)(x < n.x ? x : shared + x - n.x) * kPart; };
    float wt[kHold], ls[kHold], mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
        wt[i] = -INFINITY;
        ls[i] = 0.0f;
        if (32 * i + lane < count) {
            const float2 ml = *reinterpret_cast<const float2*>(pp + slot(32 * i + lane));
            wt[i] = ml.x;
            ls[i] = ml.y;
        }
        mx = fmaxf(mx, wt[i]);
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) mx = fmaxf(mx, shfl_xor_f32(mx, d));
    float l = 0.0f;
#pragma unroll
    for (int i = 0; i < kHold; ++i) {   // no score above -inf in the split: nothing, unless its scores were NaN
        wt[i] = wt[i] == -INFINITY ? (ls[i] == 0.0f ? 0.0f : 1.0f) : fast_exp2(wt[i] - mx);
        l += wt[i] * ls[i];
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) l += shfl_xor_f32(l, d);
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s0 = group; s0 < count; s0 += kAhead * GROUPS) {
        float4 v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            v[u] = *reinterpret_cast<const float4*>(pp + slot(min(s0 + u * GROUPS, count - 1)) + 4 + 4 * lane);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int x = s0 + u * GROUPS;
            const float held = x < 32 ? wt[0] : x < 64 ? wt[1] : x < 96 ? wt[2] : wt[3];
            const float w = __shfl(held, x & 31, 32);
            if (x < count) {
                o.x += w * v[u].x;
                o.y += w * v[u].y;
                o.z += w * v[u].z;
                o.w += w * v[u].w;
            }
        }
    }
    if constexpr (GROUPS > 1) {
        *reinterpret_cast<float4*>(&sum_sh[half][4 * lane]) = o;
        __syncthreads();
        if (group != 0) return;
#pragma unroll
        for (int u = 1; u < GROUPS; ++u) {
            const float4 v = *reinterpret_cast<const float4*>(&sum_sh[half + u][4 * lane]);
            o.x += v.x;
            o.y += v.y;
            o.z += v.z;
            o.w += v.w;
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    *reinterpret_cast<uint2*>(out + row * kDim + 4 * lane) =
        make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
}

template <bool WIDE, bool OWN_WIDE>
void launch_read(const SharedArgs& a, int64_t items, hipStream_t s) {
    const dim3 grid((unsigned)items), wg(64 * kWaves);
    if (a.shift < 4) hipLaunchKernelGGL((shared_read<WIDE, OWN_WIDE, true>), grid, wg, 0, s, a);
    else hipLaunchKernelGGL((shared_read<WIDE, OWN_WIDE, false>), grid, wg, 0, s, a);
}

}  // namespace
}  // namespace attnlab

using namespace attnlab;

extern "C" int64_t attnlab_shared_part_bytes(int B, int G, int h, int T, int shared_splits, int own_splits) {
    if (B < 1 || G < 1 || h < 1 || T < 0 || shared_splits < 0 || own_splits < 1) return -1;
    const int64_t slots = (int64_t)shared_splits + own_splits, rows = (int64_t)B * G * h * T;
    return slots > 1 ? (rows + 1) / 2 * 16 + rows * slots * kPart * 4 : 0;   // the counts, then the partials
}

extern "C" int attnlab_shared_prefix_attend(const uint16_t* q, const uint16_t* k_pages, const uint16_t* v_pages, int num_pages,
                                            int page_size, const int32_t* block_table, int64_t bt_stride, int max_pages,
                                            const int32_t* lengths, int length, const int32_t* prefix_lengths, int prefix_length,
                                            const int32_t* runs, int R, int B, int G, int h, int T, float scale, int wide,
                                            int shared_splits, int own_splits, uint16_t* out, float* part, int64_t part_bytes,
                                            void* stream) {
    ATTNLAB_REQUIRE(B >= 1 && G >= 1 && T >= 0, "B, G must be positive and T >= 0 (B=%d G=%d T=%d)", B, G, T);
    ATTNLAB_REQUIRE(1 <= h && h <= 16, "query heads per group h=%d outside [1, 16]", h);
    ATTNLAB_REQUIRE(page_size >= 1 && page_size <= (1 << 16) && (page_size & (page_size - 1)) == 0,
                    "page_size=%d must be a power of two in [1, 65536]", page_size);
    ATTNLAB_REQUIRE(num_pages >= 1 && max_pages >= 1, "num_pages=%d and max_pages=%d must be positive", num_pages, max_pages);
    ATTNLAB_REQUIRE((int64_t)max_pages * page_size <= INT32_MAX - 128, "max_pages * page_size exceeds 2^31 positions");
    ATTNLAB_REQUIRE((int64_t)num_pages * G * page_size <= INT32_MAX, "the pool of %d pages x %d groups x %d rows exceeds 2^31 rows",
                    num_pages, G, page_size);
    ATTNLAB_REQUIRE(lengths || length >= 0, "length=%d must not be negative", length);
    ATTNLAB_REQUIRE(prefix_lengths || prefix_length >= 0, "prefix_length=%d must not be negative", prefix_length);
    ATTNLAB_REQUIRE(R >= 1 && (runs || R == 1), "R=%d runs need their bounds", R);
    ATTNLAB_REQUIRE(0 <= shared_splits && shared_splits <= kMaxSplits && 1 <= own_splits && own_splits <= kMaxSplits,
                    "key splits %d and %d outside [0, %d] and [1, %d]", shared_splits, own_splits, kMaxSplits, kMaxSplits);
    if (T == 0) return ATTNLAB_OK;
    ATTNLAB_REQUIRE(q && k_pages && v_pages && out && block_table && bt_stride >= max_pages,
                    "q, k_pages, v_pages, out and a block_table of max_pages=%d entries per sequence are required", max_pages);
    ATTNLAB_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages) |
                      reinterpret_cast<uintptr_t>(out)) & 15) == 0, "q, k_pages, v_pages and out must be 16-byte aligned");
    const int64_t need = attnlab_shared_part_bytes(B, G, h, T, shared_splits, own_splits);
    ATTNLAB_REQUIRE(need == 0 || (part && (reinterpret_cast<uintptr_t>(part) & 15) == 0 && part_bytes >= need),
                    "%d + %d key splits need a 16-byte aligned part buffer of %lld bytes", shared_splits, own_splits,
                    (long long)need);
    SharedArgs a{};
    a.q = q;
    a.K = k_pages;
    a.V = v_pages;
    a.table = block_table;
    a.table_stride = bt_stride;
    a.lengths = lengths;
    a.prefixes = prefix_lengths;
    a.runs = runs;
    a.length = length;
    a.prefix = prefix_length;
    a.B = B;
    a.G = G;
    a.h = h;
    a.T = T;
    a.W = max_pages;
    a.R = R;
    a.pages = num_pages;
    a.shift = __builtin_ctz((unsigned)page_size);
    a.scale_log2 = scale * kLog2e;
    a.out = out;
    const int64_t rows = (int64_t)B * G * h * T;
    ATTNLAB_REQUIRE(rows < (int64_t)1 << 31 && R < 1 << 30, "%lld rows of %d runs are too many", (long long)rows, R);
    if (need) {
        a.counts = reinterpret_cast<int2*>(part);
        a.part = part + (rows + 1) / 2 * 4;
    }
    a.shared = shared_splits;
    a.own = own_splits;
    const bool own_wide = T > 1;
    if (own_wide) wide = 1;
    const int own_rows = own_wide ? kWide : kNarrow;
    const int64_t own = (int64_t)B * G * ((T * (int64_t)h + own_rows - 1) / own_rows) * own_splits;
    const int workers = !wide ? kNarrowWorkers : own_wide ? kWideWorkers : kMixedWorkers;
    // Workgroups of the shared part: a piece of every tile of rows (a run's last one can be partly empty: one such for each run
    // that has a row) beside the shares that the chip holds at once, or one of every tile; or all shares of the longest
    // prefixes that the tables have room for
    const int64_t tiles = G * ((int64_t)B * T * h / (wide ? kWide : kNarrow) + (R < B ? R : B));
    const int64_t keys = (int64_t)max_pages * page_size, longest = prefix_lengths || prefix_length > keys ? keys : prefix_length;
    const int least = wide ? kKeys * kLeastBlocks : kTile * kLeastTiles;
    const int64_t shares = (longest + least - 1) / least;
    int64_t first = 0;
    if (shared_splits) {
        first = (tiles > workers ? tiles : workers) + tiles;
        if (tiles * shares < first) first = tiles * shares;
    }
    ATTNLAB_REQUIRE(first + own + 16 < (int64_t)1 << 31 && tiles * kMaxSplits < (int64_t)1 << 31,
                    "a grid of %lld workgroups is too large", (long long)(first + own));
    a.own_items = (int)own;
    a.shared_turns = (int)((first + 7) / 8) + (first ? 1 : 0);   // whole shares and pieces are eighths of their own
    a.own_turns = (a.own_items + 7) / 8;
    const int64_t items = 8 * ((int64_t)a.shared_turns + a.own_turns);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (own_wide) launch_read<true, true>(a, items, s);
    else if (wide && shared_splits) launch_read<true, false>(a, items, s);
    else launch_read<false, false>(a, items, s);
    if (need) {
        // four half waves a row where it can have many partials (16 answers on 8K: 26.8 us, with one 29.0), else one (16 questions:
        // 461 us, with four 478)
        const int slots = shared_splits + own_splits;
        const dim3 wg(256);
        if (slots > 8) hipLaunchKernelGGL(shared_combine<4>, dim3((unsigned)((rows + 1) / 2)), wg, 0, s, a.part, a.counts, out,
                                          shared_splits, slots, rows);
        else hipLaunchKernelGGL(shared_combine<1>, dim3((unsigned)((rows + 7) / 8)), wg, 0, s, a.part, a.counts, out, shared_splits,
                                slots, rows);
    }
    return check_launch("shared_prefix_attend");
}
