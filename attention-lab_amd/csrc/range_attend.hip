// One query's attention over part of a cache, on the matrix cores: the positions of a sliding window and a few first
// tokens (sinks), every legal position, or a listed set of rows; over a bf16 cache or an 8-bit one (quant.h).
//   out[b,g,i] = sum_j softmax_j(scale q[b,g,i] . k_j) v_j    over j in [0, s) U [lo, n), or over the listed rows
//
// A wave takes 32 rows at a time: S^T[keys, heads] = K Q^T, two 16-key tiles of v_mfma_f32_16x16x32_bf16, then
// O^T[dims, heads] += V^T P^T, eight 16-dim tiles. K's rows are loaded in the operand's order (16 keys over the lanes, a
// row's bytes over the four lane groups) and go from the load to the matrix core; V's rows pass through the wave's own LDS
// and are read transposed. Key 8 g + 4 t + i is row 4 g + i of tile t, so that a lane's eight weights are those of the
// eight consecutive keys whose V it reads. The waves wait for each other only at the end.
// An 8-bit code becomes a bf16 exactly, its block's scale included, in one conversion (v_cvt_scalef32_pk_bf16_fp8). The
// matrix cores' own fp8 products would save K's, but they sum with about 16 bits (2^-16 of the summed magnitudes off on
// N(0, 1) rows, 2^-13 on rows of mixed magnitudes, where the bf16 products stay within fp32's rounding).
//
// The 16 columns of a tile are 8 heads twice: columns 0..7 multiply V by P rounded to bf16, columns 8..15 by what that
// rounding left, and the two are added at the end, so the weights keep 16 bits without a second product. Softmax is
// online in the log2 domain; a row's shift m is set 2^8 above its largest score so far and moves, with the sums rescaled,
// only when a score passes it, so most tiles need no exchange between lanes and no weight is above 1: n rows of values
// below 2^128 / n have finite sums, as with the exact maximum. Sums and outputs are fp32. The waves of a workgroup merge
// through LDS, the P workgroups of a (b, g) through partials: the last to arrive merges them in split order, or, without
// counters, a second small launch does, with the same sums.
//
// What bounds it: the bytes of the rows. A kernel of as many workgroups that only reads a large buffer reaches 7.1 TB/s; 16
// requests of 32K (8 groups, h=4), 8-bit, take 158 us: 6.8 TB/s. Eight 128K caches with a window of 4096 over bf16: 25.6 us,
// 5.2 TB/s; five of 5K to 20K (h=8): 29.5 us, 4.4; 1092 listed rows of 16 requests: 14.1 us, 2.6 TB/s of rows apart; one
// request of 2K: 8 us, the latencies of a launch (5.2 with one tile a wave and nothing to merge) and of the merge. Ranges take
// three waves a SIMD with one tile each over two with two, and four waves a workgroup over eight or sixteen.
//
// Masked rows: their scores are replaced, and their V rows are zeros of scale 1, so whatever they and their scale bytes hold
// (NaN, infinity) leaves the output alone. A query with no row to read, or whose scores are all -inf, gets zeros.
#include <cfloat>

#include "mfma_attend.h"
#include "quant.h"

namespace attnlab {

int check_quant_cache(const void* k_codes, const void* v_codes, const void* k_exp, const void* v_exp, int B, int G,
                      int C, int block);

namespace {

constexpr int kDim = 128;
constexpr int kWaves = 4;
constexpr int kTile = 32;           // rows a wave takes at a time
constexpr int kListChunk = 2048;    // listed positions staged in LDS at a time
constexpr float kLazy = 8.0f;       // the shift lies 2^8 above the largest score when it is set
constexpr int kPartWords = kDim + 2;

struct RangeArgs {
    const uint8_t* K;         // [B, G, C, 128] bf16 or codes, as bytes
    const uint8_t* V;
    const uint8_t* ke;        // [B, G, nb] scale bytes (8-bit cache)
    const uint8_t* ve;
    const uint16_t* q;        // [B, G, h, 128]
    const int32_t* lengths;   // [B] valid lengths, the query at the last position; or null: `n` and `qend`
    const int32_t* rows;      // [B * G, S] (listed rows)
    int64_t rows_stride;
    int B, G, h, C, P, shift, nb;
    int n;                    // keys [0, n); the number of listed rows
    int64_t qend;             // the query's position + 1, where the window ends
    int window, sinks;        // window 0: none
    float scale_log2;
    void* out;
    int out_bf16;
    uint32_t* arrive;         // [B * G] arrival counters, zero on entry and left zero: the last workgroup of a (b, g) merges
                              // its partials (P <= kMergeSlots); null: a second launch does
    float* part;              // [slot, h, 130]: m, l, the unnormalised outputs (P > 1; B * G * P slots)
};

// The rows a sequence of n keys reads: positions [0, s) and [lo, n), in aligned tiles of 32 (a scale block is 16 positions
// or more, so a tile's eights share a scale); the second range's first tile may begin before lo.
struct Span {
    int s, lo, n;
    __device__ __forceinline__ int first_tiles() const { return (s + kTile - 1) / kTile; }
    __device__ __forceinline__ int from() const { return lo & ~(kTile - 1); }
    __device__ __forceinline__ int tiles() const {
        return first_tiles() + (n > lo ? (n - from() + kTile - 1) / kTile : 0);
    }
};
__device__ __forceinline__ Span span_of(const RangeArgs& a, int n, int64_t qend) {
    Span r{0, 0, n};
    if (a.window > 0) {
        r.s = min(a.sinks, n);
        r.lo = (int)min((int64_t)n, max(qend - a.window, (int64_t)r.s));
    }
    return r;
}
__device__ __forceinline__ Span span_of_sequence(const RangeArgs& a, int b) {
    const int n = min(max(a.lengths[b], 0), a.C);
    return span_of(a, n, n);
}

// With a length per sequence and P > 1 the B P slots of a group go to the sequences by their tiles: sequence b takes
// ceil(tiles_b / share), one at least, the share being the least (of 4 tiles or more) with which B (P - 1) slots would hold
// them all evenly, so B more hold every remainder. Each workgroup works this out for itself, 64 sequences at a time.
__device__ __forceinline__ int share_of(const RangeArgs& a) {
    const int lane = threadIdx.x & 63;
    uint32_t total = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const uint32_t x = b0 + lane < a.B ? (uint32_t)span_of_sequence(a, b0 + lane).tiles() : 0u;
        total += (uint32_t)__builtin_amdgcn_readlane((int)wave_incl_scan(x), 63);
    }
    const uint32_t even = (uint32_t)(a.B * (a.P - 1));
    return (int)max((uint32_t)kWaves, (total + even - 1) / even);
}
// The sequence `by_slot` belongs to (or, by_slot < 0, `b` itself): b, its first slot and its number of slots. b = a.B where
// the slot is nobody's.
__device__ __forceinline__ void slots_of(const RangeArgs& a, int share, int by_slot, int& b, int& first, int& count) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const uint32_t x =
            b0 + lane < a.B ? (uint32_t)max((span_of_sequence(a, b0 + lane).tiles() + share - 1) / share, 1) : 0u;
        const uint32_t to = wave_incl_scan(x) + (uint32_t)base;   // the slots of this lane's sequence end here
        const uint64_t hit = by_slot < 0 ? (b >= b0 && b < b0 + 64 ? 1ull << (b - b0) : 0ull)
                                         : __ballot((int)to > by_slot);
        if (hit) {
            const int at = __builtin_ctzll(hit);
            b = b0 + at;
            count = __builtin_amdgcn_readlane((int)x, at);
            first = __builtin_amdgcn_readlane((int)to, at) - count;
            return;
        }
        base = __builtin_amdgcn_readlane((int)to, 63);
    }
    b = a.B;
    first = count = 0;
}

// One tile of a wave. 8-bit: K two 16-byte loads a row (bytes 16 g .. and 64 + 16 g ..), V eight lanes a row; bf16: twice
// as many. Scale bytes: of this lane's K row of tile 0 and 1, and of V (of its eight keys; in a list of key
// 8 g4 + n16 % 8).
template <bool Q8>
struct Tile {
    u32x4_t k[2][Q8 ? 2 : 4];
    u32x4_t v[Q8 ? 4 : 8];
    uint32_t kx[2], vx;
};

// P up to which the last workgroup of a (b, g) to arrive merges its partials (with lengths, a sequence can have more slots
// than P); past it they take a launch of their own.
constexpr int kMergeSlots = 16;

// A partial's weight against the maximum mt. No score above -inf (m = -inf): nothing to add, unless they were NaN.
__device__ __forceinline__ float slot_weight(float m, float l, float mt) {
    return m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : fast_exp2(m - mt);
}

// `count` partials `step` words apart merged in order, kGroup in flight: lane l holds dims 2 l, 2 l + 1. COHERENT: written
// by workgroups of this launch, read past the caches of this XCD.
template <bool COHERENT, int kGroup>
__device__ __forceinline__ void merge_groups(const float* pb, size_t step, int count, float& m, float& l, float2& o) {
    const int lane = threadIdx.x & 63;
    m = -INFINITY;
    l = 0.0f;
    o = make_float2(0.0f, 0.0f);
    for (int p0 = 0; p0 < count; p0 += kGroup) {
        float mv[kGroup], lv[kGroup];
        float2 ov[kGroup];
#pragma unroll
        for (int u = 0; u < kGroup; ++u) {   // past the last slot: that one again, with no weight
            const float* pp = pb + min(p0 + u, count - 1) * step;
            if constexpr (COHERENT) {
                mv[u] = load_coherent(pp);
                lv[u] = load_coherent(pp + 1);
                ov[u] = make_float2(load_coherent(pp + 2 + 2 * lane), load_coherent(pp + 3 + 2 * lane));
            } else {
                const float2 ml = *reinterpret_cast<const float2*>(pp);
                mv[u] = ml.x;
                lv[u] = ml.y;
                ov[u] = *reinterpret_cast<const float2*>(pp + 2 + 2 * lane);
            }
        }
        float mn = m;
#pragma unroll
        for (int u = 0; u < kGroup; ++u) mn = fmaxf(mn, mv[u]);
        const float w0 = slot_weight(m, l, mn);
        l *= w0;
        o.x *= w0;
        o.y *= w0;
#pragma unroll
        for (int u = 0; u < kGroup; ++u) {
            if (p0 + u < count) {
                const float w = slot_weight(mv[u], lv[u], mn);
                l += w * lv[u];
                o.x += w * ov[u].x;
                o.y += w * ov[u].y;
            }
        }
        m = mn;
    }
}

// Sixteen in flight where there are more than eight (in a launch of its own 0.3 to 0.5 us less), else eight (0.3 less).
template <bool COHERENT>
__device__ __forceinline__ void merge_slots(const float* pb, size_t step, int count, float& m, float& l, float2& o) {
    if (count > 8) merge_groups<COHERENT, 16>(pb, step, count, m, l, o);
    else merge_groups<COHERENT, 8>(pb, step, count, m, l, o);
}

// Outputs 2 l, 2 l + 1 of a (b, g, head); zeros where nothing was summed.
__device__ __forceinline__ void store_row(const RangeArgs& a, size_t row, float l, float2 o) {
    const float2 r = l == 0.0f ? make_float2(0.0f, 0.0f) : make_float2(o.x / l, o.y / l);
    const size_t to = row * kDim + 2 * (threadIdx.x & 63);
    if (a.out_bf16) *reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(a.out) + to) = pack_bf16x2(r.x, r.y);
    else *reinterpret_cast<float2*>(reinterpret_cast<float*>(a.out) + to) = r;
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const uint8_t* base, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, (int)bytes, 0x00020000);
}

template <bool Q8, bool LIST>
__global__ __launch_bounds__(64 * kWaves, LIST ? 2 : 3) void range_attend(RangeArgs a) {
    constexpr int kRow = Q8 ? kDim : 2 * kDim;          // bytes of a row
    constexpr int kLanes = kRow / 16;                   // lanes of a V row
    constexpr int kKLoads = Q8 ? 2 : 4, kVLoads = Q8 ? 4 : 8;
    __shared__ __attribute__((aligned(1024))) uint16_t v_sh[kWaves][kTile * kDim];   // a wave's V tile; then the merge
    __shared__ float ml_sh[kWaves][16][2];
    __shared__ int list_sh[LIST ? kListChunk : 1];
    __shared__ __attribute__((aligned(8))) uint8_t vx_sh[kWaves][kTile];
    __shared__ uint32_t last_sh;
    const int lin = __builtin_amdgcn_readfirstlane(xcd_contiguous_block());
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n16 = lane & 15, g4 = lane >> 4;

    // this workgroup's (b, g), its rows, and its tiles [t0, t1) of them
    int bg, p, share, slots = a.P;
    Span rows{0, 0, a.n};   // the list's entries, or a range
    if (!LIST && a.lengths && a.P > 1) {
        const int g = lin / (a.B * a.P);
        int b, first;
        share = share_of(a);
        slots_of(a, share, lin - g * a.B * a.P, b, first, slots);
        if (b >= a.B) return;
        p = lin - g * a.B * a.P - first;
        bg = b * a.G + g;
        rows = span_of_sequence(a, b);
    } else {
        bg = lin / a.P;
        p = lin - bg * a.P;
        if constexpr (!LIST) rows = a.lengths ? span_of_sequence(a, bg / a.G) : span_of(a, a.n, a.qend);
        share = (rows.tiles() + a.P - 1) / a.P;
    }
    const int s = rows.s, lo = rows.lo, n = rows.n, from = rows.from();
    const int na = rows.first_tiles(), tiles = rows.tiles();
    if (!LIST && a.lengths && a.P > 1) share = (tiles + slots - 1) / slots;   // evenly: 16 to 32K 108 us for 111
    const int t0 = (int)min((int64_t)p * share, (int64_t)tiles), t1 = min(t0 + share, tiles);

    // Q^T as the B operand: column n16 is head n16 % 8; its 8 dims of step kk, in the order K's bytes are loaded in
    bf16x8_t qb[4];
    {
        const int head = n16 & 7;
        const uint16_t* qr = a.q + ((size_t)bg * a.h + min(head, a.h - 1)) * kDim;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            const int d = Q8 ? 64 * (kk >> 1) + 16 * g4 + 8 * (kk & 1) : 32 * kk + 8 * g4;
            u32x4_t w = *reinterpret_cast<const u32x4_t*>(qr + d);
            if (head >= a.h) w = u32x4_t{0, 0, 0, 0};
            qb[kk] = __builtin_bit_cast(bf16x8_t, w);
        }
    }
    // the scale (log2 domain), made positive: a negative one flips the sign of q instead (exact), and zero becomes the
    // smallest normal float, which gives the same weights while a masked key's -inf * scale stays -inf
    const float sc = a.scale_log2 == 0.0f ? FLT_MIN : fabsf(a.scale_log2);
    if (a.scale_log2 < 0.0f) {
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
            qb[kk] = __builtin_bit_cast(bf16x8_t, __builtin_bit_cast(u32x4_t, qb[kk]) ^ 0x80008000u);
    }
    const uint8_t* Kb = a.K + (size_t)bg * a.C * kRow;
    const uint8_t* Vb = a.V + (size_t)bg * a.C * kRow;
    const uint8_t* keb = Q8 ? a.ke + (size_t)bg * a.nb : nullptr;
    const uint8_t* veb = Q8 ? a.ve + (size_t)bg * a.nb : nullptr;
    // This lane's rows of a tile: K row 8 (n16 / 4) + 4 t + n16 % 4 of operand t; V rows u (64 / kLanes) + vrow.
    const int krow = 8 * (n16 >> 2) + (n16 & 3), vrow = lane / kLanes;
    // V in LDS. 8-bit: 128-byte rows of 8 chunks, chunk c of row r at c ^ (r / 2 % 8); bf16: 256-byte rows of 16 chunks,
    // chunk c of row r at c ^ (4 (r % 4)): the rows that a transposing read takes together then lie in different banks
    // (8-bit: lane 2 e + j of 16 reads 8 bytes of row 8 g4 + e and gets 8 rows of one dim; bf16: lane 4 e + j four
    // elements of row 8 g4 + 4 t + e, and gets 4 rows).
    char* vt = reinterpret_cast<char*>(v_sh[wave]);
    const int vst = Q8 ? 128 * vrow + 16 * ((lane & 7) ^ (vrow >> 1)) : 256 * vrow + 16 * ((lane & 15) ^ (4 * (vrow & 3)));
    const int vof8 = 128 * (8 * g4 + (n16 >> 1)) + 16 * (4 * (g4 & 1) + (n16 >> 2)) + 8 * (n16 & 1);
    int vof[4];
    if constexpr (!Q8) {
#pragma unroll
        for (int x = 0; x < 4; ++x) vof[x] = 256 * (8 * g4 + (n16 >> 2)) + 64 * (x ^ (n16 >> 2)) + 8 * (n16 & 3);
    }

    float m = -INFINITY, l = 0.0f;
    f32x4_t o[8];
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) o[dt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

    int c0 = 0;   // first tile of the list chunk in LDS
    // first position of a range's tile, the end of its range, and where the range begins
    auto range_tile = [&](int t, int& base, int& end, int& begin) {
        const bool first = t < na;
        base = first ? kTile * t : from + kTile * (t - na);
        end = first ? s : n;
        begin = first ? 0 : lo;
    };
    auto entry = [&](int t, int r) -> int { return list_sh[kTile * (t - c0) + r]; };   // position of row r, or -1
    auto issue = [&](int t, Tile<Q8>& f) {
        if constexpr (LIST) {
            int kp[2];
#pragma unroll
            for (int t2 = 0; t2 < 2; ++t2) {
                kp[t2] = max(entry(t, krow + 4 * t2), 0);
                f.kx[t2] = keb[kp[t2] >> a.shift];
            }
            // a skipped slot has no scale byte: its weight is zero, and zero times the scale of some byte would be NaN
            const int vp = entry(t, 8 * g4 + (n16 & 7));
            const uint32_t vx = veb[max(vp, 0) >> a.shift];
            f.vx = vp < 0 ? 127u : vx;
#pragma unroll
            for (int t2 = 0; t2 < 2; ++t2) {
                const uint8_t* r = Kb + (size_t)kp[t2] * kRow + 16 * g4;
#pragma unroll
                for (int c = 0; c < kKLoads; ++c)
                    f.k[t2][c] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(r + 64 * c));
            }
#pragma unroll
            for (int u = 0; u < kVLoads; ++u) {
                const uint8_t* r = Vb + (size_t)max(entry(t, (64 / kLanes) * u + vrow), 0) * kRow + 16 * (lane % kLanes);
                f.v[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(r));
            }
        } else {   // rows past the range read as zeros: the buffer ends there
            int base, end, begin;
            range_tile(t, base, end, begin);
            const uint32_t bytes = (uint32_t)min(kTile, end - base) * kRow;
            const __amdgpu_buffer_rsrc_t kr = buffer(Kb + (size_t)base * kRow, bytes);
            const __amdgpu_buffer_rsrc_t vr = buffer(Vb + (size_t)base * kRow, bytes);
            if constexpr (Q8) {
                f.kx[0] = f.kx[1] = __builtin_amdgcn_raw_buffer_load_b8(buffer(keb, (uint32_t)a.nb),
                                                                        (base + 8 * (n16 >> 2)) >> a.shift, 0, 0);
                f.vx = __builtin_amdgcn_raw_buffer_load_b8(buffer(veb, (uint32_t)a.nb), (base + 8 * g4) >> a.shift, 0, 0);
            }
            constexpr int kNt = 2;   // non-temporal
#pragma unroll
            for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
                for (int c = 0; c < kKLoads; ++c)
                    f.k[t2][c] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                                                                 kr, krow * kRow + 16 * g4 + 4 * t2 * kRow + 64 * c, 0, kNt));
#pragma unroll
            for (int u = 0; u < kVLoads; ++u)
                f.v[u] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(vr, 16 * lane + 1024 * u, 0, kNt));
        }
        // every load is on its way before the first result is waited for
        __builtin_amdgcn_sched_barrier(0);
    };
    auto compute = [&](int t, Tile<Q8>& f) {
        uint32_t ok;   // rows of the tile to read
        if constexpr (LIST) {
            ok = (uint32_t)__ballot(entry(t, lane & 31) >= 0);
        } else {
            int base, end, begin;
            range_tile(t, base, end, begin);
            const int rows = end - base, skip = begin - base;
            ok = rows >= kTile ? 0xffffffffu : (1u << rows) - 1u;
            if (skip > 0) ok &= 0xffffffffu << skip;
        }
        f32x4_t sv[2];
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
            sv[t2] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
            float ks = 1.0f;
            if constexpr (Q8) ks = scale_of(f.kx[t2]);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                u32x4_t w;
                if constexpr (Q8) {
                    const u32x4_t c = f.k[t2][kk >> 1];
                    const uint32_t w0 = kk & 1 ? c.z : c.x, w1 = kk & 1 ? c.w : c.y;
                    w = u32x4_t{e4m3_to_bf16x2<false>(w0, ks), e4m3_to_bf16x2<true>(w0, ks),
                                e4m3_to_bf16x2<false>(w1, ks), e4m3_to_bf16x2<true>(w1, ks)};
                } else {
                    w = f.k[t2][kk];
                }
                sv[t2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, w), qb[kk], sv[t2], 0, 0, 0);
            }
        }
        // V on its way to LDS while the scores are made
        if (ok != 0xffffffffu) {
            asm volatile("");   // a branch, not selects: few tiles are partial
#pragma unroll
            for (int u = 0; u < kVLoads; ++u)
                if (!(ok >> ((64 / kLanes) * u + vrow) & 1)) f.v[u] = u32x4_t{0, 0, 0, 0};
        }
#pragma unroll
        for (int u = 0; u < kVLoads; ++u) {
            // 8-bit: r / 2 % 8 of row 8 u + vrow is vrow / 2 ^ 4 (u % 2)
            const int at = Q8 ? (vst ^ (64 * (u & 1))) + 1024 * u : vst + 1024 * u;
            *reinterpret_cast<u32x4_t*>(vt + at) = f.v[u];
        }
        if constexpr (LIST) {   // the scale bytes of V's 32 rows, to be read by eights
            if (n16 < 8) vx_sh[wave][8 * g4 + n16] = (uint8_t)f.vx;
        }
        // this lane's scores: column n16, keys 8 g4 + 4 t2 + i
        if (ok != 0xffffffffu) {
            asm volatile("");
#pragma unroll
            for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (!(ok >> (8 * g4 + 4 * t2 + i) & 1)) sv[t2][i] = -INFINITY;
        }
        float bm = -INFINITY;
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
            for (int i = 0; i < 4; ++i) bm = fmaxf(bm, sv[t2][i]);
        if (__any(bm * sc > m)) {
            bm = max_xor32(max_xor16(bm)) * sc;
            if (bm > m) {   // also a column's first rows (m = -inf)
                bm += kLazy;
                const float al = fast_exp2(m - bm);
                l *= al;
#pragma unroll
                for (int dt = 0; dt < 8; ++dt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[dt][i] *= al;
                m = bm;
            }
        }
        const float nm = m == -INFINITY ? 0.0f : -m;   // no score above -inf yet: every weight 0
        float pr[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) pr[i] = fast_exp2(fmaf(sv[i >> 2][i & 3], sc, nm));
        l += ((pr[0] + pr[1]) + (pr[2] + pr[3])) + ((pr[4] + pr[5]) + (pr[6] + pr[7]));
        // a wave's LDS operations take effect in order; these keep the compiler from moving them past each other
        asm volatile("" ::: "memory");
        if constexpr (LIST) {   // V's rows have scales of their own: they go into the weights
            const uint2 x = *reinterpret_cast<const uint2*>(&vx_sh[wave][8 * g4]);
#pragma unroll
            for (int i = 0; i < 8; ++i) pr[i] *= scale_of((i < 4 ? x.x : x.y) >> (8 * (i & 3)) & 255u);
        }
        uint32_t w4[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t hi = pack_bf16x2(pr[2 * i], pr[2 * i + 1]);
            const uint32_t rest = pack_bf16x2(pr[2 * i] - bf16_lo(hi), pr[2 * i + 1] - bf16_hi(hi));
            w4[i] = n16 < 8 ? hi : rest;
        }
        const bf16x8_t pb = __builtin_bit_cast(bf16x8_t, u32x4_t{w4[0], w4[1], w4[2], w4[3]});
        // 8-bit: the scale of this lane's eight keys. Where all are masked it can be any byte, one that is no number among them
        const float vs = Q8 && !LIST && (ok >> (8 * g4) & 255u) != 0 ? scale_of(f.vx) : 1.0f;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
            u32x4_t w;
            if constexpr (Q8) {
                const u32x2v_t c = read_tr8(vt + (vof8 ^ (16 * dt)));
                w = u32x4_t{e4m3_to_bf16x2<false>(c.x, vs), e4m3_to_bf16x2<true>(c.x, vs), e4m3_to_bf16x2<false>(c.y, vs),
                            e4m3_to_bf16x2<true>(c.y, vs)};
            } else {
                const char* r = vt + vof[dt >> 1] + 32 * (dt & 1);
                const u32x2v_t w0 = read_tr16(r), w1 = read_tr16(r + 4 * 256);
                w = u32x4_t{w0.x, w0.y, w1.x, w1.y};
            }
            o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, w), pb, o[dt], 0, 0, 0);
        }
        asm volatile("" ::: "memory");
    };
    auto walk = [&](int ta, int tb) {   // tile t of [ta, tb) belongs to wave (t - ta) % kWaves
        int t = ta + wave;
        if constexpr (LIST) {
            // a tile ahead, at two waves a SIMD: 1092 rows of 16 requests 14.9 us for 15.8 (ranges gain nothing by it)
            Tile<Q8> f0, f1;
            if (t < tb) issue(t, f0);
            for (; t < tb; t += 2 * kWaves) {
                if (t + kWaves < tb) issue(t + kWaves, f1);
                compute(t, f0);
                if (t + kWaves >= tb) break;
                if (t + 2 * kWaves < tb) issue(t + 2 * kWaves, f0);
                compute(t + kWaves, f1);
            }
        } else {
            for (; t < tb; t += kWaves) {
                Tile<Q8> f;
                issue(t, f);
                compute(t, f);
            }
        }
    };
    if constexpr (LIST) {
        for (c0 = t0; c0 < t1; c0 += kListChunk / kTile) {
            const int tb = min(c0 + kListChunk / kTile, t1);
            const int32_t* src = a.rows + (size_t)bg * a.rows_stride + (size_t)kTile * c0;
            const int len = min(kTile * (tb - c0), n - kTile * c0);
            if (c0 != t0) __syncthreads();
            for (int i = tid; i < kTile * (tb - c0); i += 64 * kWaves) {
                const int pos = i < len ? src[i] : -1;
                list_sh[i] = (unsigned)pos < (unsigned)a.C ? pos : -1;
            }
            __syncthreads();
            walk(c0, tb);
        }
    } else {
        walk(t0, t1);
    }
    l += shfl_xor_f32(l, 16);
    l += shfl_xor_f32(l, 32);

    // the waves' (m, l, O) through LDS: [wave][column][dim] floats, in the V tiles' memory
    __syncthreads();
    float* red = reinterpret_cast<float*>(&v_sh[0][0]);
    static_assert(sizeof(v_sh) >= kWaves * 16 * kDim * sizeof(float), "the merge lies in the V tiles");
    if (g4 == 0) {
        ml_sh[wave][n16][0] = m;
        ml_sh[wave][n16][1] = l;
    }
#pragma unroll
    for (int dt = 0; dt < 8; ++dt)
        *reinterpret_cast<f32x4_t*>(red + (wave * 16 + n16) * kDim + 16 * dt + 4 * g4) = o[dt];
    __syncthreads();
    const bool alone = a.P == 1 || (a.arrive != nullptr && slots == 1), merge_here = a.arrive != nullptr && slots > 1;
    for (int i = wave; i < a.h; i += kWaves) {   // wave -> head, lane l -> dims 2 l, 2 l + 1
        float ms = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) ms = fmaxf(ms, ml_sh[w][i][0]);
        float ls = 0.0f;
        float2 os = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float x = slot_weight(ml_sh[w][i][0], ml_sh[w][i][1], ms);
            const float2 hi = *reinterpret_cast<const float2*>(red + (w * 16 + i) * kDim + 2 * lane);
            const float2 rest = *reinterpret_cast<const float2*>(red + (w * 16 + 8 + i) * kDim + 2 * lane);
            ls += x * ml_sh[w][i][1];
            os.x += x * (hi.x + rest.x);
            os.y += x * (hi.y + rest.y);
        }
        if (alone) {
            store_row(a, (size_t)bg * a.h + i, ls, os);
            continue;
        }
        float* pp = a.part + ((size_t)lin * a.h + i) * kPartWords;
        if (merge_here) {   // written through to memory, so the merging workgroup reads them on any XCD
            if (lane == 0) {
                store_coherent(pp, ms);
                store_coherent(pp + 1, ls);
            }
            store_coherent(pp + 2 + 2 * lane, os.x);
            store_coherent(pp + 3 + 2 * lane, os.y);
        } else {
            if (lane == 0) *reinterpret_cast<float2*>(pp) = make_float2(ms, ls);
            *reinterpret_cast<float2*>(pp + 2 + 2 * lane) = os;
        }
    }
    if (!merge_here) return;
    // Arrival: every partial store of this workgroup has completed before its count (the wait and the barrier), so the
    // workgroup that counts all others before itself finds every partial in memory. It leaves the counter zero.
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0)
        last_sh = __hip_atomic_fetch_add(a.arrive + bg, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)(slots - 1);
    __syncthreads();
    if (!last_sh) return;
    for (int i = wave; i < a.h; i += kWaves) {
        float m2, l2;
        float2 o2;
        merge_slots<true>(a.part + ((size_t)(lin - p) * a.h + i) * kPartWords, (size_t)a.h * kPartWords, slots, m2, l2, o2);
        store_row(a, (size_t)bg * a.h + i, l2, o2);
    }
    if (tid == 0) __hip_atomic_store(a.arrive + bg, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The partials of a (b, g, head) merged: one wave up to kMergeSlots slots, the sums those of the merge inside
// range_attend; past them four waves that take every fourth slot and meet in LDS.
__global__ __launch_bounds__(256) void range_combine(RangeArgs a) {
    __shared__ float ml_sh[4][2];
    __shared__ float2 acc_sh[4][64];
    const int bg = blockIdx.x / a.h, i = blockIdx.x - bg * a.h;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), W = blockDim.x >> 6;
    int first = bg * a.P, count = a.P;
    if (a.lengths) {
        int b = bg / a.G;
        slots_of(a, share_of(a), -1, b, first, count);
        first += (bg - b * a.G) * a.B * a.P;
    }
    const size_t step = (size_t)a.h * kPartWords;
    float m, l;
    float2 o;
    merge_slots<false>(a.part + ((size_t)first * a.h + i) * kPartWords + wave * step, W * step, (count - wave + W - 1) / W,
                       m, l, o);
    if (W > 1) {
        if (lane == 0) {
            ml_sh[wave][0] = m;
            ml_sh[wave][1] = l;
        }
        acc_sh[wave][lane] = o;
        __syncthreads();
        if (wave != 0) return;
        float mt = m;
        for (int w = 1; w < W; ++w) mt = fmaxf(mt, ml_sh[w][0]);
        l = 0.0f;
        o = make_float2(0.0f, 0.0f);
        for (int w = 0; w < W; ++w) {
            const float x = slot_weight(ml_sh[w][0], ml_sh[w][1], mt);
            l += x * ml_sh[w][1];
            o.x += x * acc_sh[w][lane].x;
            o.y += x * acc_sh[w][lane].y;
        }
    }
    store_row(a, (size_t)bg * a.h + i, l, o);
}

template <bool LIST>
int launch_range(const RangeArgs& a, hipStream_t s) {
    const int64_t blocks = (int64_t)a.B * a.G * a.P;
    ATTNLAB_REQUIRE(blocks < (int64_t)1 << 31, "grid of %lld workgroups is too large", (long long)blocks);
    const dim3 grid((unsigned)blocks), wg(64 * kWaves);
    if constexpr (LIST) hipLaunchKernelGGL((range_attend<true, true>), grid, wg, 0, s, a);
    else if (a.ke) hipLaunchKernelGGL((range_attend<true, false>), grid, wg, 0, s, a);
    else hipLaunchKernelGGL((range_attend<false, false>), grid, wg, 0, s, a);
    if (a.P > 1 && a.arrive == nullptr)
        hipLaunchKernelGGL(range_combine, dim3((unsigned)(a.B * a.G * a.h)), dim3(a.P <= kMergeSlots ? 64 : 256), 0, s, a);
    return check_launch(LIST ? "range_attend (rows)" : "range_attend");
}

int check_range(const void* K, const void* V, const uint8_t* k_exp, const uint8_t* v_exp, int block, const uint16_t* q,
                int B, int G, int h, int C, int P, const void* out, int out_bf16, const float* part) {
    if (k_exp || v_exp) {
        const int rc = check_quant_cache(K, V, k_exp, v_exp, B, G, C, block);
        if (rc) return rc;
    }
    ATTNLAB_REQUIRE(B >= 1 && G >= 1 && C >= 1, "B=%d G=%d C=%d must be positive", B, G, C);
    ATTNLAB_REQUIRE(1 <= h && h <= 8, "h=%d outside [1, 8]", h);
    ATTNLAB_REQUIRE(1 <= P && P <= 256, "partitions P=%d outside [1, 256]", P);
    ATTNLAB_REQUIRE((int64_t)B * G * h < (int64_t)1 << 31, "B * G * h too large");
    ATTNLAB_REQUIRE(K && V && q && out, "K, V, q and out must be device pointers");
    ATTNLAB_REQUIRE(((reinterpret_cast<uintptr_t>(K) | reinterpret_cast<uintptr_t>(V) | reinterpret_cast<uintptr_t>(q)) &
                     15) == 0, "K, V and q must be 16-byte aligned");
    ATTNLAB_REQUIRE((reinterpret_cast<uintptr_t>(out) & (out_bf16 ? 3 : 7)) == 0,
                    "out must be aligned to two of its elements (stored in pairs)");
    ATTNLAB_REQUIRE(P == 1 || (part != nullptr && (reinterpret_cast<uintptr_t>(part) & 7) == 0),
                    "P > 1 needs the partial buffer, 8-byte aligned");
    return ATTNLAB_OK;
}

RangeArgs range_args(const void* K, const void* V, const uint8_t* k_exp, const uint8_t* v_exp, int block,
                     const uint16_t* q, int B, int G, int h, int C, int P, float scale, void* out, int out_bf16,
                     float* part, uint32_t* arrive) {
    RangeArgs a{};
    a.B = B;
    a.K = static_cast<const uint8_t*>(K);
    a.V = static_cast<const uint8_t*>(V);
    a.ke = k_exp;
    a.ve = v_exp;
    a.q = q;
    a.G = G;
    a.h = h;
    a.C = C;
    a.P = P;
    if (k_exp) {
        a.shift = block == 16 ? 4 : block == 32 ? 5 : 6;
        a.nb = (C + block - 1) / block;
    }
    a.scale_log2 = scale * kLog2e;
    a.out = out;
    a.out_bf16 = out_bf16;
    a.part = part;
    a.arrive = P > 1 && P <= kMergeSlots ? arrive : nullptr;
    return a;
}

}  // namespace
}  // namespace attnlab

using namespace attnlab;

extern "C" int attnlab_range_decode(const void* K, const void* V, const uint8_t* k_exp, const uint8_t* v_exp, int block,
                                    const uint16_t* q, const int32_t* lengths, int length, int64_t q_pos, int window,
                                    int sinks, int B, int G, int h, int C, int P, float scale, void* out, int out_bf16,
                                    float* part, uint32_t* arrive, void* stream) {
    const int rc = check_range(K, V, k_exp, v_exp, block, q, B, G, h, C, P, out, out_bf16, part);
    if (rc) return rc;
    ATTNLAB_REQUIRE(lengths != nullptr || (0 <= length && length <= C), "valid length %d outside [0, C=%d]", length, C);
    ATTNLAB_REQUIRE(lengths != nullptr || q_pos >= 0, "the query's position %lld must not be negative",
                    (long long)q_pos);
    ATTNLAB_REQUIRE(window >= 0 && sinks >= 0, "window=%d and sinks=%d must not be negative", window, sinks);
    RangeArgs a = range_args(K, V, k_exp, v_exp, block, q, B, G, h, C, P, scale, out, out_bf16, part, arrive);
    a.lengths = lengths;
    a.n = lengths ? 0 : (int)(q_pos + 1 < length ? q_pos + 1 : length);   // causal: no key past the query
    a.qend = q_pos + 1;
    a.window = window;
    a.sinks = sinks;
    return launch_range<false>(a, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int attnlab_quant_attend(const uint8_t* k_codes, const uint8_t* v_codes, const uint8_t* k_exp,
                                    const uint8_t* v_exp, int block, const uint16_t* q, const int32_t* rows,
                                    int64_t rows_stride, int B, int G, int h, int S, int C, int P, float scale,
                                    void* out, int out_bf16, float* part, uint32_t* arrive, void* stream) {
    ATTNLAB_REQUIRE(k_exp && v_exp, "the scale bytes must be device pointers");
    const int rc = check_range(k_codes, v_codes, k_exp, v_exp, block, q, B, G, h, C, P, out, out_bf16, part);
    if (rc) return rc;
    ATTNLAB_REQUIRE(S >= 1, "at least one row must be selected (S=%d)", S);
    ATTNLAB_REQUIRE(rows != nullptr && rows_stride >= S, "rows must hold S=%d positions per (b, g)", S);
    RangeArgs a = range_args(k_codes, v_codes, k_exp, v_exp, block, q, B, G, h, C, P, scale, out, out_bf16, part, arrive);
    a.rows = rows;
    a.rows_stride = rows_stride;
    a.n = S;
    return launch_range<true>(a, reinterpret_cast<hipStream_t>(stream));
}
