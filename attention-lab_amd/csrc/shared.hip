// Attention of sequences that share prompts, over a paged cache: sequence b's T queries sit at the last positions of its length,
//   out[b,g,i,t] = sum_j softmax_j(scale q[b,g,i,t] . k_j) v_j    over j <= lengths[b] - T + t, k_j and v_j by b's table
// Consecutive sequences form runs; the whole pages of a run's first prefix[r] positions are the same for all of its sequences. So
// the keys fall into two parts, each with its own softmax, and the parts (m, l, o) are merged at the end:
//   the shared part   a run's rows, n sequences x T queries x h heads, against its prefix: a matrix product, the keys read once
//   the own part      a sequence's T h rows against its positions from the prefix on
// A sequence that ends inside its run's prefix takes no part in the shared read and reads all of its positions in the own part, so
// the shared one has no masked positions at all.
//
// Both parts are split over workgroups by keys; every (row, split) leaves a partial, and a last launch merges a row's.
//
// Two kernels. `wide`: 128 rows, four waves of 32; blocks of 64 keys, S^T = K Q^T, the softmax on its accumulators, O^T += V^T P^T
// (v_mfma_f32_32x32x16_bf16), K and V copied into LDS a block ahead without passing through registers. `narrow`: up to 16 rows;
// each wave walks tiles of 32 keys of its own (v_mfma_f32_16x16x32_bf16), K from memory to the matrix core, V through the wave's
// LDS. Both look a key's page up a block ahead, one entry a lane, so pages may be of any size and end anywhere in a block; a
// key without a page is read as zeros and masked.
//
// Weights are rounded to bf16, the operand's type, before their product with V; their sum is of the unrounded ones, sums fp32.
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
constexpr int kMaxSplits = 64;

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
    float* part;              // [B, G, h, T, shared + own, 132]
    int shared, own;          // key splits of the two parts
    int tiles;                // row tiles of the shared part, at most
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

// Calls step(runs of 64 lanes, how many) until it returns true: lane x holds run r0 + x. Runs are [S_r, S_{r+1}) with S_r the
// largest of runs[0 .. r] within [0, B], so they never overlap.
template <typename Step>
__device__ __forceinline__ void walk_runs(const SharedArgs& a, Step step) {
    const int lane = threadIdx.x & 63;
    int before = a.runs ? min(max(a.runs[0], 0), a.B) : 0;
    for (int r0 = 0; r0 < a.R; r0 += 64) {
        const int r = r0 + lane;
        int upto = a.runs ? (r < a.R ? min(max(a.runs[r + 1], 0), a.B) : 0) : a.B;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int x = __shfl_up(upto, d, 64);
            if (lane >= d) upto = max(upto, x);
        }
        upto = max(upto, before);
        int from = __shfl_up(upto, 1, 64);
        if (lane == 0) from = before;
        before = __builtin_amdgcn_readlane(upto, 63);
        Run run{from, r < a.R ? upto - from : 0, 0};
        if (run.count > 0) run.prefix = prefix_of(a, r);
        if (step(run)) return;
    }
}
__device__ __forceinline__ Run lane_run(const Run& run, int at) {
    return Run{__builtin_amdgcn_readlane(run.first, at), __builtin_amdgcn_readlane(run.count, at),
               __builtin_amdgcn_readlane(run.prefix, at)};
}
// The run of row tile `tile` (of `rows` rows) of the shared part, and the tile's number in it; count 0: none.
__device__ __forceinline__ Run run_of_tile(const SharedArgs& a, int tile, int rows, int& in_run) {
    Run found{0, 0, 0};
    int base = 0;
    walk_runs(a, [&](const Run& run) {
        const uint32_t tiles = run.prefix > 0 ? (uint32_t)(((int64_t)run.count * a.T * a.h + rows - 1) / rows) : 0u;
        const uint32_t upto = wave_incl_scan(tiles) + (uint32_t)base;
        const uint64_t hit = __ballot((int)upto > tile);
        if (hit) {
            const int at = __builtin_ctzll(hit);
            found = lane_run(run, at);
            in_run = tile - (__builtin_amdgcn_readlane((int)upto, at) - __builtin_amdgcn_readlane((int)tiles, at));
            return true;
        }
        base = __builtin_amdgcn_readlane((int)upto, 63);
        return false;
    });
    return found;
}
// The shared positions of sequence b's run (0: none).
__device__ __forceinline__ int prefix_of_sequence(const SharedArgs& a, int b) {
    int found = 0;
    walk_runs(a, [&](const Run& run) {
        const uint64_t hit = __ballot(run.count > 0 && run.first <= b && b < run.first + run.count);
        if (hit) found = __builtin_amdgcn_readlane(run.prefix, __builtin_ctzll(hit));
        return hit != 0;
    });
    return found;
}
// Whether all queries of sequence b see all of `prefix` positions; if not, it reads none of them in the shared part.
__device__ __forceinline__ bool sees(const SharedArgs& a, int b, int prefix) { return length_of(a, b) - a.T + 1 >= prefix; }

// What a workgroup does: `rows` rows from row r0 of `count` sequences from b0 on, over the blocks [i0, i1) of the keys [base, end)
// of sequence b0's table, its partials in slot `slot`.
struct Item {
    int b0, count, r0, rows, base, end, i0, i1, slot, g;
    bool shared;
};
template <int kRows, int kBlock>
__device__ __forceinline__ bool item_of(const SharedArgs& a, int lin, Item& w) {
    const int shared_items = a.G * a.shared * a.tiles;
    int split, splits;
    if (lin < shared_items) {   // the tiles that read the same keys lie next to each other, on one XCD
        const int gs = lin / a.tiles;
        int tile = 0;
        const Run run = run_of_tile(a, lin - gs * a.tiles, kRows, tile);
        if (run.count == 0) return false;
        w.g = gs / a.shared;
        split = gs - w.g * a.shared;
        splits = a.shared;
        w.b0 = run.first;
        w.count = run.count;
        w.r0 = tile * kRows;
        w.base = 0;
        w.end = run.prefix;
        w.slot = split;
        w.shared = true;
    } else {
        lin -= shared_items;
        const int tiles = (a.T * a.h + kRows - 1) / kRows;
        split = lin % a.own;
        lin /= a.own;
        const int tile = tiles - 1 - lin % tiles;   // later queries read more keys: first
        lin /= tiles;
        w.g = lin % a.G;
        w.b0 = lin / a.G;
        w.count = 1;
        w.r0 = tile * kRows;
        const int prefix = a.shared ? prefix_of_sequence(a, w.b0) : 0, n = length_of(a, w.b0);
        w.base = sees(a, w.b0, prefix) ? prefix : 0;
        w.end = max(n - a.T + min(a.T - 1, (w.r0 + kRows - 1) / a.h) + 1, w.base);
        splits = a.own;
        w.slot = a.shared + split;
        w.shared = false;
        // nobody else writes the shared slots of a sequence that shares nothing
        if (prefix == 0 && a.shared && split == 0) {
            const int rows = min(kRows, a.T * a.h - w.r0);
            for (int x = threadIdx.x; x < rows * a.shared; x += 64 * kWaves) {
                const int row = w.r0 + x / a.shared, t = row / a.h, head = row - t * a.h;
                float* pp = a.part + ((((size_t)w.b0 * a.G + w.g) * a.h + head) * a.T + t) * (a.shared + a.own) * kPart +
                            (size_t)(x % a.shared) * kPart;
                pp[0] = -INFINITY;
                pp[1] = 0.0f;
            }
        }
    }
    w.rows = (int)min((int64_t)w.count * a.T * a.h - w.r0, (int64_t)kRows);
    const int blocks = (w.end - w.base + kBlock - 1) / kBlock, share = (blocks + splits - 1) / splits;
    w.i0 = min(split * share, blocks);
    w.i1 = min(w.i0 + share, blocks);
    return true;
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

// This lane's key's page (key `key` of sequence b's table), or -1.
__device__ __forceinline__ int page_of(const SharedArgs& a, const int32_t* row, int key, int end) {
    if (key >= end) return -1;
    const int p = row[key >> a.shift];
    return (uint32_t)p < (uint32_t)a.pages ? p : -1;
}
// The address of key `key` in page p, or zeros.
__device__ __forceinline__ const char* key_row(const SharedArgs& a, const uint16_t* pool, int p, int g, int key, int chunk) {
    const size_t row = (((size_t)(uint32_t)p * a.G + g) << a.shift) + (key & ((1 << a.shift) - 1));
    return p < 0 ? reinterpret_cast<const char*>(shared_zeros) : reinterpret_cast<const char*>(pool) + row * (2 * kDim) + chunk;
}

// The scale (log2 domain), made positive: a negative one flips the sign of q instead (exact), and zero becomes the smallest normal
// float, which gives the same weights while a masked key's -inf * scale stays -inf.
__device__ __forceinline__ float positive_scale(float x) { return x == 0.0f ? FLT_MIN : fabsf(x); }

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
__global__ __launch_bounds__(256, 2) void shared_wide(SharedArgs a, int first_item) {
    constexpr int kRow = 2 * kDim;
    __shared__ __attribute__((aligned(1024))) char kt0[kKeys * kRow], vt0[kKeys * kRow];
    __shared__ __attribute__((aligned(1024))) char kt1[kKeys * kRow], vt1[kKeys * kRow];
    __shared__ int again;
    Item w;
    if (!item_of<kWide, kKeys>(a, __builtin_amdgcn_readfirstlane(xcd_contiguous_block()) + first_item, w)) return;
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
    const int lim = limit(R), lim_min = limit(32 * wave), lim_max = limit(32 * wave + 31);
    const bool dead = w.shared && !sees(a, row.b, w.end);

    // staging: a load of a wave fills 1 KB of a tile, four rows, lane l slot l % 16 of row l / 16 of them
    const int srow = lane >> 4, slot = lane & 15;
    const int kchunk = 16 * (slot ^ (4 * wave + srow)), vchunk = 16 * (slot ^ (4 * srow));
    const int32_t* pages = a.table + (size_t)w.b0 * a.table_stride;
    auto first_key = [&](int i) { return w.base + kKeys * i; };
    auto look = [&](int i) { return i < w.i1 ? page_of(a, pages, first_key(i) + lane, w.end) : -1; };
    auto copy = [&](int kb, int page, char* kt, char* vt) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int j = 16 * u + 4 * wave + srow, p = __shfl(page, j, 64);
            load_lds16(reinterpret_cast<const uint16_t*>(key_row(a, a.K, p, w.g, kb + j, kchunk)),
                       reinterpret_cast<uint16_t*>(kt + 4096 * u + 1024 * wave));
            load_lds16(reinterpret_cast<const uint16_t*>(key_row(a, a.V, p, w.g, kb + j, vchunk)),
                       reinterpret_cast<uint16_t*>(vt + 4096 * u + 1024 * wave));
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
        const bool ahead = kb + kKeys > lim_min, gaps = ~have != 0;
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
        bf16x8_t pb[4];
        const float nm = m_run == -INFINITY ? 0.0f : -m_run;   // no score above -inf yet: weights 0, or NaN for a NaN score
#pragma unroll
        for (int ks2 = 0; ks2 < 4; ++ks2) {
            uint32_t w4[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x0 = s[ks2 >> 1][8 * (ks2 & 1) + 2 * e], x1 = s[ks2 >> 1][8 * (ks2 & 1) + 2 * e + 1];
                const float p0 = fast_exp2(fmaf(x0, sc, nm));
                const float p1 = fast_exp2(fmaf(x1, sc, nm));
                l_run += p0 + p1;
                w4[e] = pack_bf16x2(p0, p1);
            }
            pb[ks2] = __builtin_bit_cast(bf16x8_t, u32x4_t{w4[0], w4[1], w4[2], w4[3]});
        }
        if (!careful || !spoilt) {
#pragma unroll
            for (int ks2 = 0; ks2 < 4; ++ks2)
#pragma unroll
                for (int dt = 0; dt < 4; ++dt)
                    o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(value(ks2, dt), pb[ks2], o[dt], 0, 0, 0);
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
    // publishes the current block, and land while it is computed; its pages were looked up a block before that.
    uint64_t have = 0;
    int next = look(w.i0);
    auto issue = [&](int i, char* kt, char* vt) {   // block i's copies; the pages of block i + 1
        const int page = next;
        next = look(i + 1);
        copy(first_key(i), page, kt, vt);
        return (uint64_t)__ballot(page >= 0);
    };
    auto publish = [&]() {
        __builtin_amdgcn_s_waitcnt(0x0070);   // vmcnt(0) lgkmcnt(0): this wave's copies have landed, its reads are done
        asm volatile("s_barrier" ::: "memory");
        pin();
    };
    if (tid == 0) again = 0;   // published by the first block's barrier
    if (w.i0 < w.i1) have = issue(w.i0, kt0, vt0);
    for (int i = w.i0; i < w.i1; i += 2) {
        publish();
        uint64_t now = have;
        if (i + 1 < w.i1) have = issue(i + 1, kt1, vt1);
        block(std::false_type{}, first_key(i), now, kt0, vt0);
        if (i + 1 >= w.i1) break;
        publish();
        now = have;
        if (i + 2 < w.i1) have = issue(i + 2, kt0, vt0);
        block(std::false_type{}, first_key(i + 1), now, kt1, vt1);
    }
    // A result that is not finite: a visible key's doing, or zero weights times one that only later queries see. All rows again, with
    // the blocks that have such keys looked over. The shared part has none.
    if (!w.shared) {
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
            next = look(w.i0);
            for (int i = w.i0; i < w.i1; ++i) {
                have = issue(i, kt0, vt0);
                publish();
                block(std::true_type{}, first_key(i), have, kt0, vt0);
                __syncthreads();
            }
        }
    }
    const float l_tot = l_run + shfl_xor_f32(l_run, 32);
    if (R >= w.rows) return;
    const int slots = a.shared + a.own;
    if (slots > 1) {
        float* pp = a.part + (row.at(a, w.g) * slots + w.slot) * kPart;
        if (g == 0) {
            pp[0] = dead ? -INFINITY : m_run;
            pp[1] = dead ? 0.0f : l_tot;
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

// One tile of a wave: K's rows krow and krow + 4, 16 bytes of every 64; V's rows 4 u + lane / 16.
struct Tile {
    u32x4_t k[2][4], v[8];
};

__global__ __launch_bounds__(64 * kWaves, 3) void shared_narrow(SharedArgs a, int first_item) {
    constexpr int kRow = 2 * kDim;
    __shared__ __attribute__((aligned(1024))) uint16_t v_sh[kWaves][kTile * kDim];   // a wave's V tile; then the merge
    __shared__ float ml_sh[kWaves][kNarrow][2];
    Item w;
    if (!item_of<kNarrow, kTile>(a, __builtin_amdgcn_readfirstlane(xcd_contiguous_block()) + first_item, w)) return;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n16 = lane & 15, g4 = lane >> 4;
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
    const int krow = 8 * (n16 >> 2) + (n16 & 3), vrow = lane >> 4;
    // V in LDS: chunk c of row r at c ^ (4 (r % 4)), so that the rows a transposing read takes together lie in different banks
    // (lane 4 e + j of 16 reads four elements of row 8 g4 + 4 t + e, and gets 4 rows)
    char* vt = reinterpret_cast<char*>(v_sh[wave]);
    const int vst = 256 * vrow + 16 * (n16 ^ (4 * vrow));
    int vof[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) vof[x] = 256 * (8 * g4 + (n16 >> 2)) + 64 * (x ^ (n16 >> 2)) + 8 * (n16 & 3);

    float m = -INFINITY, l = 0.0f;
    f32x4_t o[8];
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) o[dt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

    const int32_t* pages = a.table + (size_t)w.b0 * a.table_stride;
    auto look = [&](int i) { return i < w.i1 ? page_of(a, pages, w.base + kTile * i + (lane & 31), w.end) : -1; };
    int next = look(w.i0 + wave);
    for (int i = w.i0 + wave; i < w.i1; i += kWaves) {
        const int page = next, kb = w.base + kTile * i;
        Tile f;
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
            const int j = krow + 4 * t2;
            const char* r = key_row(a, a.K, __shfl(page, j, 64), w.g, kb + j, 16 * g4);
            const bool none = r == reinterpret_cast<const char*>(shared_zeros);
#pragma unroll
            for (int c = 0; c < 4; ++c)
                f.k[t2][c] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(r + (none ? 0 : 64 * c)));
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int j = 4 * u + vrow;
            f.v[u] = __builtin_nontemporal_load(
                reinterpret_cast<const u32x4_t*>(key_row(a, a.V, __shfl(page, j, 64), w.g, kb + j, 16 * n16)));
        }
        next = look(i + kWaves);
        __builtin_amdgcn_sched_barrier(0);   // every load is on its way before the first result is waited for
        const uint32_t have = (uint32_t)__ballot(page >= 0);
        f32x4_t sv[2];
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
            sv[t2] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
                sv[t2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, f.k[t2][kk]), qb[kk], sv[t2], 0, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) *reinterpret_cast<u32x4_t*>(vt + vst + 1024 * u) = f.v[u];
        // this lane's scores: column n16, keys 8 g4 + 4 t2 + i
        if (~have) {
#pragma unroll
            for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (!(have >> (8 * g4 + 4 * t2 + e) & 1)) sv[t2][e] = -INFINITY;
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
        uint32_t w4[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w4[e] = pack_bf16x2(pr[2 * e], pr[2 * e + 1]);
        const bf16x8_t pb = __builtin_bit_cast(bf16x8_t, u32x4_t{w4[0], w4[1], w4[2], w4[3]});
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
            const char* r = vt + vof[dt >> 1] + 32 * (dt & 1);
            const u32x2v_t w0 = read_tr16(r), w1 = read_tr16(r + 4 * kRow);
            o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, u32x4_t{w0.x, w0.y, w1.x, w1.y}), pb, o[dt],
                                                           0, 0, 0);
        }
        asm volatile("" ::: "memory");
    }
    l += shfl_xor_f32(l, 16);
    l += shfl_xor_f32(l, 32);

    // the waves' (m, l, O) through LDS: [wave][row][dim] floats, in the V tiles' memory
    __syncthreads();
    float* red = reinterpret_cast<float*>(&v_sh[0][0]);
    static_assert(sizeof(v_sh) >= kWaves * kNarrow * kDim * sizeof(float), "the merge lies in the V tiles");
    if (g4 == 0) {
        ml_sh[wave][n16][0] = m;
        ml_sh[wave][n16][1] = l;
    }
#pragma unroll
    for (int dt = 0; dt < 8; ++dt)
        *reinterpret_cast<f32x4_t*>(red + (wave * kNarrow + n16) * kDim + 16 * dt + 4 * g4) = o[dt];
    __syncthreads();
    const int slots = a.shared + a.own;
    for (int r = wave; r < w.rows; r += kWaves) {   // wave -> row, lane l -> dims 2 l, 2 l + 1
        const Row row(a, w, r);
        const bool dead = w.shared && !sees(a, row.b, w.end);
        float ms = -INFINITY;
#pragma unroll
        for (int x = 0; x < kWaves; ++x) ms = fmaxf(ms, ml_sh[x][r][0]);
        float ls = 0.0f;
        float2 os = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int x = 0; x < kWaves; ++x) {
            const float mx = ml_sh[x][r][0], lx = ml_sh[x][r][1];
            const float y = mx == -INFINITY ? (lx == 0.0f ? 0.0f : 1.0f) : fast_exp2(mx - ms);
            const float2 v = *reinterpret_cast<const float2*>(red + (x * kNarrow + r) * kDim + 2 * lane);
            ls += y * lx;
            os.x += y * v.x;
            os.y += y * v.y;
        }
        if (slots > 1) {
            float* pp = a.part + (row.at(a, w.g) * slots + w.slot) * kPart;
            if (lane == 0) {
                pp[0] = dead ? -INFINITY : ms;
                pp[1] = dead ? 0.0f : ls;
            }
            *reinterpret_cast<float2*>(pp + 4 + 2 * lane) = os;
        } else {
            const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
            *reinterpret_cast<uint32_t*>(a.out + row.at(a, w.g) * kDim + 2 * lane) = pack_bf16x2(os.x * inv, os.y * inv);
        }
    }
}

// A row's partials merged in their order: thread -> (row, four dims).
__global__ __launch_bounds__(256) void shared_combine(const float* part, uint16_t* out, int slots, int64_t rows) {
    const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (item >= rows * 32) return;
    const int64_t row = item >> 5;
    const int d4 = 4 * (int)(item & 31);
    const float* pp = part + row * slots * kPart;
    float mx = -INFINITY;
    for (int s = 0; s < slots; ++s) mx = fmaxf(mx, pp[s * kPart]);
    float l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s = 0; s < slots; ++s) {
        const float m = pp[s * kPart], ls = pp[s * kPart + 1];
        // no score above -inf in the split: nothing, unless its scores were NaN
        if (m == -INFINITY && ls == 0.0f) continue;
        const float w = m == -INFINITY ? 1.0f : fast_exp2(m - mx);
        const float4 v = *reinterpret_cast<const float4*>(pp + s * kPart + 4 + d4);
        l += w * ls;
        o.x += w * v.x;
        o.y += w * v.y;
        o.z += w * v.z;
        o.w += w * v.w;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    *reinterpret_cast<uint2*>(out + row * kDim + d4) =
        make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
}

}  // namespace
}  // namespace attnlab

using namespace attnlab;

extern "C" int64_t attnlab_shared_part_bytes(int B, int G, int h, int T, int shared_splits, int own_splits) {
    if (B < 1 || G < 1 || h < 1 || T < 0 || shared_splits < 0 || own_splits < 1) return -1;
    const int64_t slots = (int64_t)shared_splits + own_splits;
    return slots > 1 ? (int64_t)B * G * h * T * slots * kPart * 4 : 0;
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
                    "%d + %d key splits need a 16-byte aligned part buffer of %lld bytes", shared_splits, own_splits, (long long)need);
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
    a.part = part;
    a.shared = shared_splits;
    a.own = own_splits;
    const int64_t rows = (int64_t)B * G * h * T, per_group = (int64_t)B * T * h;
    ATTNLAB_REQUIRE(rows < (int64_t)1 << 31 && per_group + 128 * (int64_t)R < (int64_t)1 << 31, "%lld rows are too many", (long long)rows);
    const bool own_wide = T > 1;
    const int shared_rows = wide ? kWide : kNarrow, own_rows = own_wide ? kWide : kNarrow;
    // a run's last tile can be partly empty: at most one such for each run that has a row
    a.tiles = shared_splits ? (int)(per_group / shared_rows + (R < B ? R : B)) : 0;
    const int64_t shared_items = (int64_t)G * shared_splits * a.tiles;
    const int64_t own_items = (int64_t)B * G * ((T * (int64_t)h + own_rows - 1) / own_rows) * own_splits;
    ATTNLAB_REQUIRE(shared_items + own_items < (int64_t)1 << 31 && rows * 32 / 256 < (int64_t)1 << 31,
                    "grids of %lld and %lld workgroups are too large", (long long)shared_items, (long long)own_items);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const dim3 wg(256);
    auto launch = [&](bool wide_rows, int64_t items, int first) {
        if (items == 0) return;
        if (wide_rows) hipLaunchKernelGGL(shared_wide, dim3((unsigned)items), wg, 0, s, a, first);
        else hipLaunchKernelGGL(shared_narrow, dim3((unsigned)items), wg, 0, s, a, first);
    };
    if ((wide != 0) == own_wide) {
        launch(own_wide, shared_items + own_items, 0);
    } else {
        launch(wide != 0, shared_items, 0);
        launch(own_wide, own_items, (int)shared_items);
    }
    if (need) hipLaunchKernelGGL(shared_combine, dim3((unsigned)((rows * 32 + 255) / 256)), wg, 0, s, part, out,
                                 shared_splits + own_splits, rows);
    return check_launch("shared_prefix_attend");
}
