// Causal attention of a chunk of queries over a cache whose visible positions end in a sliding window and a few first
// tokens (sinks), or are all the legal ones; over a bf16 cache or an 8-bit one (quant.h). Query t sits at p = q_pos0 + t:
//   out[b,g,i,t] = sum_j softmax_j(scale q[b,g,i,t] . k_j) v_j    over j <= p, j < legal, (j > p - window or j < sinks)
//
// A workgroup owns 128 (query, head) rows, 128 / h consecutive queries with all h heads, and walks blocks of 64 keys: the
// blocks of the sinks, then those from the first query's window on. Per block S^T = K Q^T, the softmax on its
// accumulators, O^T += V^T P^T (v_mfma_f32_32x32x16_bf16; a row's softmax state and outputs stay in lanes n and n + 32).
// K and V are copied into LDS in the cache's own format without passing through registers, a block ahead, one barrier a
// block; an 8-bit operand becomes bf16 (exactly, its scale included) as it is read, which costs each wave 128 conversions
// a block and halves what it reads from LDS.
//
// The weights are rounded to bf16, the operand's type, before their product with V; their sum is of the unrounded ones.
// Outputs are off the 64-bit ones by 0.0023 of them (root mean square), where rounding the output alone costs 0.0016. The
// one-query kernel's weights of two parts would be half as many products again.
//
// What bounds it: the matrix cores are busy 50 % of the time at about 2.1 GHz, the vector units 60 % with the softmax and
// the conversions; LDS reads wait between (without them the kernel took 320 us where it took 535, without the copies 428).
// An 8K prompt (8 groups, h=4; 0.55 TFLOP) takes 509 us over bf16 (1.08 PFLOP/s) and 510 to 520 over 8 bits, where tiles
// widened on their way into LDS took 562. 1000 queries after 29011 (h=2), 8-bit: 246 us (0.98 PFLOP/s); 1501 queries,
// window 2047, 8-bit: 74; two 8K prompts (h=4) with a window of 1024 over bf16: 310. There 4096 workgroups take 80 us apart
// from their blocks (eight rounds of 10: Q, the first copies with nothing to hide behind, the output) and 14 us for each
// block: windows of 64, 512, 1024, 2048 and 4096 take 117, 204, 312, 489 and 779 us, none 995. A wave with 64 rows
// halves the reads per product and holds too many registers (632 us and 828); eight waves over 256 rows take 493 us over
// bf16, 540 over 8 bits and 311 under the window, and are coarser on short prompts; equal runs of all tiles' blocks for each
// workgroup balance the chip and write twice the partials (86 us for 76 under the window); a wave's priority, half blocks
// or V read ahead gave nothing.
//
// A masked key has weight zero, but zero times a V row that holds NaN or infinity is NaN. Rows past the visible range are
// copied as zeros; inside it a key can be masked for one row and visible to the next. So a workgroup with a result that is
// not finite takes its rows again, looks over the blocks that have masked keys and multiplies those that hold such values
// by way of flags.
#include <cfloat>
#include <type_traits>

#include "mfma_attend.h"
#include "quant.h"

namespace attnlab {

int check_quant_cache(const void* k_codes, const void* v_codes, const void* k_exp, const void* v_exp, int B, int G,
                      int C, int block);

namespace {

constexpr int kDim = 128;
constexpr int kRows = 128;          // (query, head) rows per workgroup: 4 waves x 32
constexpr int kKeys = 64;           // keys per block
constexpr float kLazy = 8.0f;       // a row's shift is set 2^8 above its largest score and moves when one passes it: few
                                    // rescales, and no weight above 1, so n rows of values below 2^128 / n have finite sums
constexpr int kPart = 132;          // m, l, two unused words (16-byte aligned rows), the 128 unnormalised outputs
constexpr int kMaxSplits = 16;

struct RangePrefillArgs {
    const uint16_t* q;      // [BG, h, T, 128]
    const void* K;          // [BG, C, 128] bf16 or codes
    const void* V;
    const uint8_t* ke;      // [BG, nb] scale bytes (8-bit cache)
    const uint8_t* ve;
    uint16_t* out;          // [BG, h, T, 128]
    int h, T, q_pos0, legal, C, shift, nb;
    int window, sinks;      // window 0: none
    int bq, qtiles;         // queries per workgroup, ceil(T / bq)
    float scale_log2;
    int splits;             // workgroups that share a tile's key blocks, their partials in `part` (splits > 1)
    float* part;            // [BG, h, T, splits, 132]
};

// NaN and infinity among two packed bf16: the pair with those elements zeroed, and a pair of flags (1.0 or 0).
__device__ __forceinline__ uint32_t bf16x2_finite(uint32_t w, uint32_t& flags) {
    const uint32_t lo = (w & 0x00007f80u) == 0x00007f80u ? 0x0000ffffu : 0u;
    const uint32_t hi = (w & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u;
    flags = (lo & 0x3f80u) | (hi & 0x3f800000u);
    return w & ~(lo | hi);
}

// K and V blocks in LDS: 64 rows in 16-byte chunks, permuted within the row so that the reads meet no bank twice.
// bf16, 16 chunks: K's chunk c of row j at slot c ^ (j & 15) (a read takes 16 rows, one chunk), V's at c ^ (4 (j & 3)) (a
// transposing read takes 4 chunks of 4 consecutive rows). 8-bit, 8 chunks: K's at c ^ (j / 2 % 8) (16 rows, one chunk),
// V's at c ^ (2 (j / 2 % 4)) (half a wave takes two chunks of 8 consecutive rows).
// Key 16 z + 8 g + 4 a + b of a 32-key tile is row 16 z + 8 a + 4 g + b of its product, so that a lane's weights are those
// of eight consecutive keys, the ones whose V its operand holds.
template <bool SPLIT, bool Q8>
__global__ __launch_bounds__(256, 2) void range_prefill(RangePrefillArgs a) {
    constexpr int kRow = Q8 ? kDim : 2 * kDim;   // bytes of a row
    __shared__ __attribute__((aligned(1024))) char kt0[kKeys * kRow], vt0[kKeys * kRow];
    __shared__ __attribute__((aligned(1024))) char kt1[kKeys * kRow], vt1[kKeys * kRow];
    __shared__ int again;
    const int lin = xcd_contiguous_block();
    // the query tiles of a (b, g) in reverse: without a window the later ones read more keys, so they start first
    const int nsp = SPLIT ? a.splits : 1;
    const int per_bg = a.qtiles * nsp;
    const int bg = __builtin_amdgcn_readfirstlane(lin / per_bg), rem = lin - bg * per_bg;
    const int rq = __builtin_amdgcn_readfirstlane(rem / nsp);
    const int qt = a.qtiles - 1 - rq, sp = rem - rq * nsp;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, g = lane >> 5;
    const int t0 = qt * a.bq;
    const int tend = min(t0 + a.bq, a.T);        // the workgroup's queries are [t0, tend)
    const int R = 32 * wave + n;                 // this lane's row: query t0 + R / h, head R % h
    const int t = t0 + R / a.h, head = R % a.h;
    const int tc = min(t, tend - 1);             // rows past the last query repeat it and are not written
    const int pos = a.q_pos0 + tc;
    // B operand of S^T: row R, in step kk dims 16 kk + 8 g .. + 7 (8-bit: 32 (kk / 2) + 16 g + 8 (kk % 2) .., two steps to
    // a 16-byte read of K)
    bf16x8_t qb[8];
    {
        const uint16_t* qr = a.q + (((size_t)bg * a.h + head) * a.T + tc) * kDim;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
            const int d = Q8 ? 32 * (kk >> 1) + 16 * g + 8 * (kk & 1) : 16 * kk + 8 * g;
            qb[kk] = __builtin_bit_cast(bf16x8_t, *reinterpret_cast<const u32x4_t*>(qr + d));
        }
    }
    // the tile's keys: blocks [0, na) for the sinks, then [bw, ceil(kend / 64)) from the first query's window on
    const int kend = min(a.legal, a.q_pos0 + tend);
    int na = 0, bw = 0;
    if (a.window > 0) {
        na = (min(a.sinks, kend) + kKeys - 1) / kKeys;
        bw = max(na, max(a.q_pos0 + t0 + 1 - a.window, 0) / kKeys);
    }
    const int nblocks = na + max((kend + kKeys - 1) / kKeys - bw, 0);
    const int share = SPLIT ? (nblocks + nsp - 1) / nsp : nblocks;
    const int i0 = SPLIT ? min(sp * share, nblocks) : 0, i1 = SPLIT ? min(i0 + share, nblocks) : nblocks;
    auto first_key = [&](int i) { return kKeys * (i < na ? i : i - na + bw); };
    // positions of the wave's first and last row
    const int wfirst = a.q_pos0 + min(t0 + __builtin_amdgcn_readfirstlane((32 * wave) / a.h), tend - 1);
    const int wlast = a.q_pos0 + min(t0 + __builtin_amdgcn_readfirstlane((32 * wave + 31) / a.h), tend - 1);
    const int kend_wave = min(a.legal, wlast + 1);

    // staging: a load of a wave fills 1 KB of a tile, kPer rows, lane l slot l % kSlots of row l / kSlots of them, from a
    // buffer of the block's rows (those past kend give zeros)
    constexpr int kSlots = kRow / 16, kPer = 64 / kSlots, kLoads = kKeys / kPer / 4;
    const int srow = lane / kSlots, slot = lane % kSlots;
    const int kswz = Q8 ? 4 * (wave & 1) + (srow >> 1) : 4 * wave + srow, vswz = Q8 ? 2 * (srow >> 1) : 4 * srow;
    const uint32_t koff = 1024 * wave + kRow * srow + 16 * (slot ^ kswz), voff = 1024 * wave + kRow * srow + 16 * (slot ^ vswz);
    const char* Kb = reinterpret_cast<const char*>(a.K) + (size_t)bg * a.C * kRow;
    const char* Vb = reinterpret_cast<const char*>(a.V) + (size_t)bg * a.C * kRow;
    const uint8_t* keb = Q8 ? a.ke + (size_t)bg * a.nb : nullptr;
    const uint8_t* veb = Q8 ? a.ve + (size_t)bg * a.nb : nullptr;
    const __amdgpu_buffer_rsrc_t ker = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(keb), 0, a.nb, 0x00020000);
    const __amdgpu_buffer_rsrc_t ver = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(veb), 0, a.nb, 0x00020000);
    uint32_t kx[2], vx;   // the next block's scale bytes: K, of this lane's rows; V, of 16 keys in each of lanes 0 .. 3
    auto copy = [&](int kb, char* kt, char* vt) {
        const uint32_t bytes = kRow * (uint32_t)min(kend - kb, kKeys);
        const char* Kt = Kb + (size_t)kb * kRow;
        const char* Vt = Vb + (size_t)kb * kRow;
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
            const int at = 4096 * u;
            load_lds16_buf(reinterpret_cast<const uint16_t*>(Kt), bytes, koff + at,
                           reinterpret_cast<uint16_t*>(kt + 1024 * wave + at));
            load_lds16_buf(reinterpret_cast<const uint16_t*>(Vt), bytes, voff + at,
                           reinterpret_cast<uint16_t*>(vt + 1024 * wave + at));
        }
        if constexpr (Q8) {   // past the last byte: zero, of rows that are zeros
#pragma unroll
            for (int x = 0; x < 2; ++x)
                kx[x] = __builtin_amdgcn_raw_buffer_load_b8(ker, (kb + 32 * x + (n & 16)) >> a.shift, 0, 0);
            vx = __builtin_amdgcn_raw_buffer_load_b8(ver, (kb + 16 * (lane & 3)) >> a.shift, 0, 0);
        }
    };
    // operand reads, as byte offsets into a tile. K: this lane's key of a 32-key tile, bf16 chunk 2 kk + g (8-bit: chunk
    // 2 (kk / 2) + g). V: bf16 rows 16 ks + 8 g + 4 hf + e, dims 32 dt + 16 (lane / 16 % 2) + 4 j .. + 3, e = lane % 16 / 4,
    // j = lane % 4; 8-bit rows 16 ks + 8 g + e, bytes 32 dt + 16 (lane / 16 % 2) + 8 j .. + 7, e = lane % 16 / 2,
    // j = lane % 2. `pin` keeps the compiler from holding a copy of each per tile.
    const int key = (n & 16) + 8 * ((n >> 2) & 1) + 4 * ((n >> 3) & 1) + (n & 3);
    constexpr int kKof = Q8 ? 4 : 8;
    uint32_t kof[kKof], vof[4];
#pragma unroll
    for (int kk = 0; kk < kKof; ++kk) kof[kk] = kRow * key + 16 * ((2 * kk + g) ^ (Q8 ? (key >> 1) & 7 : key & 15));
    const int ve = Q8 ? (lane & 15) >> 1 : (lane & 15) >> 2;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
        vof[dt] = Q8 ? kRow * (8 * g + ve) + 16 * ((2 * dt + ((lane >> 4) & 1)) ^ (2 * (ve >> 1))) + 8 * (lane & 1)
                     : kRow * (8 * g + ve) + 64 * (dt ^ ve) + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
    auto pin = [&]() {
#pragma unroll
        for (int kk = 0; kk < kKof; ++kk) asm volatile("" : "+v"(kof[kk]));
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) asm volatile("" : "+v"(vof[dt]));
    };
    auto widen = [&](uint32_t w0, uint32_t w1, float scale) {   // eight codes as a bf16 operand
        return __builtin_bit_cast(bf16x8_t, u32x4_t{e4m3_to_bf16x2<false>(w0, scale), e4m3_to_bf16x2<true>(w0, scale),
                                                    e4m3_to_bf16x2<false>(w1, scale), e4m3_to_bf16x2<true>(w1, scale)});
    };

    float m_run = -INFINITY, l_run = 0.0f;
    // the scale (log2 domain), made positive: a negative one flips the sign of q instead (exact), and zero becomes the
    // smallest normal float, which gives the same weights while a masked key's -inf * scale stays -inf
    const float sc = a.scale_log2 == 0.0f ? FLT_MIN : fabsf(a.scale_log2);
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

    auto block = [&](auto careful, int kb, const char* ks, const char* vs, const float (&ksc)[2], const float (&vsc)[4])
                     __attribute__((always_inline)) {
        // no key of the block is visible to a row of this wave
        if (kb >= kend_wave || (a.window > 0 && kb >= a.sinks && kb + kKeys - 1 <= wfirst - a.window)) return;
        // whether a key is masked for some row of the wave: past its position or the legal keys, or ahead of its window
        const bool ahead = kb + kKeys - 1 > wfirst || kb + kKeys > a.legal;
        const bool behind = a.window > 0 && kb <= wlast - a.window && kb + kKeys > a.sinks;
        auto value = [&](int ks2, int dt) -> bf16x8_t {   // V^T's operand of 16-key step ks2, dims 32 dt ..
            const char* vp = vs + 16 * kRow * ks2 + vof[dt];
            if constexpr (Q8) {
                const u32x2v_t w = read_tr8(vp);
                return widen(w.x, w.y, vsc[ks2]);
            } else {
                const u32x2v_t lo4 = read_tr16(vp), hi4 = read_tr16(vp + 4 * kRow);
                return __builtin_bit_cast(bf16x8_t, u32x4_t{lo4.x, lo4.y, hi4.x, hi4.y});
            }
        };
        bool spoilt = false;   // some V of a block with masked keys is NaN or infinite
        if (careful && (ahead || behind)) {
            float chk = 0.0f;  // 0 times it, which is NaN
#pragma unroll
            for (int ks2 = 0; ks2 < 4; ++ks2)
#pragma unroll
                for (int dt = 0; dt < 4; ++dt) {
                    const u32x4_t w = __builtin_bit_cast(u32x4_t, value(ks2, dt));
                    chk = dot2_bf16(w.x, 0u, chk);
                    chk = dot2_bf16(w.y, 0u, chk);
                    chk = dot2_bf16(w.z, 0u, chk);
                    chk = dot2_bf16(w.w, 0u, chk);
                    __builtin_amdgcn_sched_barrier(0);   // an operand at a time: registers
                }
            spoilt = __any(chk != 0.0f);
        }
        f32x16_t s[2];
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[x][i] = 0.0f;
        // K's reads stay kAhead steps ahead of their products (left to the compiler, one read: an 8K prompt 519 us, 511 so;
        // the same for V, or V's ahead of the softmax, gave nothing more)
        constexpr int kAhead = 3;
        u32x4_t kw[kKof][2];
        auto read_k = [&](int kk) __attribute__((always_inline)) {
#pragma unroll
            for (int x = 0; x < 2; ++x) kw[kk][x] = *reinterpret_cast<const u32x4_t*>(ks + 32 * kRow * x + kof[kk]);
        };
#pragma unroll
        for (int kk = 0; kk < kAhead; ++kk) read_k(kk);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kk = 0; kk < kKof; ++kk) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const u32x4_t w = kw[kk][x];
                if constexpr (Q8) {
                    s[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(widen(w.x, w.y, ksc[x]), qb[2 * kk], s[x], 0, 0, 0);
                    s[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(widen(w.z, w.w, ksc[x]), qb[2 * kk + 1], s[x], 0, 0, 0);
                } else {
                    s[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, w), qb[kk], s[x], 0, 0, 0);
                }
            }
            if (kk + kAhead < kKof) {
                read_k(kk + kAhead);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        // this lane's scores: row R, keys kb + 8 g + c, c = 32 x + 16 (i / 8) + i % 8. The bounds that a block needs are
        // applied apart, each a compare with a constant and a select
        const int at = kb + 8 * g;
        if (ahead) {
            const int most = min(pos, a.legal - 1) - at;
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[x][i] = 32 * x + 16 * (i >> 3) + (i & 7) <= most ? s[x][i] : -INFINITY;
        }
        if (behind) {
            const int from = pos - a.window - at;   // visible: c > from, or c < sink
            if (kb >= a.sinks) {
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[x][i] = 32 * x + 16 * (i >> 3) + (i & 7) > from ? s[x][i] : -INFINITY;
            } else {
                const int sink = a.sinks - at;
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int c = 32 * x + 16 * (i >> 3) + (i & 7);
                        s[x][i] = (c > from) | (c < sink) ? s[x][i] : -INFINITY;
                    }
            }
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
        // P^T (bf16: the matrix core's operand; the sum l is of the unrounded weights) as the B operand of
        // O^T += V^T P^T, one per 16-key step ks2: tile ks2 / 2, accumulators 8 (ks2 % 2) .. + 7
        bf16x8_t pb[4];
        // no score above -inf in the row yet: weights 0, or NaN for a NaN score
        const float nm = m_run == -INFINITY ? 0.0f : -m_run;
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
    // Two tile pairs: the next block's copies are issued when every wave has left the tiles they overwrite, the barrier that
    // also publishes the current block, and land while it is computed. The pairs are separate arrays, so that the
    // compiler knows a block's reads apart from the copies in flight.
    float ksc[2] = {1.0f, 1.0f}, vsc[4] = {1.0f, 1.0f, 1.0f, 1.0f};
    auto publish = [&]() {
        __builtin_amdgcn_s_waitcnt(0x0070);   // vmcnt(0) lgkmcnt(0): this wave's copies have landed, its reads are done
        asm volatile("s_barrier" ::: "memory");
        pin();
        if constexpr (Q8) {
#pragma unroll
            for (int x = 0; x < 2; ++x) ksc[x] = scale_of(kx[x]);
#pragma unroll
            for (int x = 0; x < 4; ++x) vsc[x] = scale_of((uint32_t)__builtin_amdgcn_readlane((int)vx, x));
        }
    };
    if (tid == 0) again = 0;   // published by the first block's barrier
    if (i0 < i1) copy(first_key(i0), kt0, vt0);
    for (int i = i0; i < i1; i += 2) {
        publish();
        if (i + 1 < i1) copy(first_key(i + 1), kt1, vt1);
        block(std::false_type{}, first_key(i), kt0, vt0, ksc, vsc);
        if (i + 1 >= i1) break;
        publish();
        if (i + 2 < i1) copy(first_key(i + 2), kt0, vt0);
        block(std::false_type{}, first_key(i + 1), kt1, vt1, ksc, vsc);
    }
    // A result that is not finite: a visible key's doing, or zero weights times a masked one's values. All rows again, with
    // the blocks that have masked keys looked over (two to three times the time, where there are such values).
    float finite = 0.0f * l_run;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) finite = fmaf(0.0f, o[dt][i], finite);
    if (__any(finite != 0.0f) && lane == 0) again = 1;
    __syncthreads();
    if (again) {
        m_run = -INFINITY;
        l_run = 0.0f;
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[dt][i] = 0.0f;
        for (int i = i0; i < i1; ++i) {
            copy(first_key(i), kt0, vt0);
            publish();
            block(std::true_type{}, first_key(i), kt0, vt0, ksc, vsc);
            __syncthreads();
        }
    }
    const float l_tot = l_run + shfl_xor_f32(l_run, 32);
    if (t >= tend) return;
    if constexpr (SPLIT) {   // this split's partial: m (log2 domain, scaled), l and the unnormalised outputs
        float* pp = a.part + ((((size_t)bg * a.h + head) * a.T + t) * a.splits + sp) * kPart;
        if (g == 0) {
            pp[0] = m_run;
            pp[1] = l_tot;
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
    uint16_t* orow = a.out + (((size_t)bg * a.h + head) * a.T + t) * kDim;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {   // dims 32 dt + 8 i4 + 4 g + 0..3
            const f32x16_t& od = o[dt];
            *reinterpret_cast<u32x2v_t*>(orow + 32 * dt + 8 * i4 + 4 * g) =
                u32x2v_t{pack_bf16x2(od[4 * i4] * inv, od[4 * i4 + 1] * inv),
                         pack_bf16x2(od[4 * i4 + 2] * inv, od[4 * i4 + 3] * inv)};
        }
}

// The key splits' partials of every row merged into out: thread -> (row, four dims), in split order.
__global__ __launch_bounds__(256) void range_prefill_combine(const float* part, uint16_t* out, int splits, int64_t rows) {
    const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (item >= rows * 32) return;
    const int64_t row = item >> 5;
    const int d4 = 4 * (int)(item & 31);
    const float* pp = part + row * splits * kPart;
    float mx = -INFINITY;
    for (int sp = 0; sp < splits; ++sp) mx = fmaxf(mx, pp[sp * kPart]);
    float l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int sp = 0; sp < splits; ++sp) {
        const float m = pp[sp * kPart], ls = pp[sp * kPart + 1];
        // no finite score in the split: nothing, unless its scores were NaN
        const float w = m == -INFINITY ? (ls == 0.0f ? 0.0f : 1.0f) : fast_exp2(m - mx);
        const float4 v = *reinterpret_cast<const float4*>(pp + sp * kPart + 4 + d4);
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

extern "C" int64_t attnlab_range_prefill_part_bytes(int B, int G, int h, int T, int splits) {
    if (B < 1 || G < 1 || h < 1 || T < 0 || splits < 1) return -1;
    return splits > 1 ? (int64_t)B * G * h * T * splits * kPart * 4 : 0;
}

extern "C" int attnlab_range_prefill(const uint16_t* q, const void* K, const void* V, const uint8_t* k_exp,
                                     const uint8_t* v_exp, int block, uint16_t* out, int B, int G, int h, int T,
                                     int q_pos0, int legal, int C, int window, int sinks, float scale, int splits,
                                     float* part, int64_t part_bytes, void* stream) {
    if (k_exp || v_exp) {
        const int rc = check_quant_cache(K, V, k_exp, v_exp, B, G, C, block);
        if (rc) return rc;
    }
    ATTNLAB_REQUIRE(B >= 1 && G >= 1 && T >= 0, "B, G must be positive and T >= 0 (B=%d G=%d T=%d)", B, G, T);
    ATTNLAB_REQUIRE(1 <= h && h <= 16, "query heads per group h=%d outside [1, 16]", h);
    ATTNLAB_REQUIRE(q_pos0 >= 0 && 0 <= legal && legal <= C, "need q_pos0 >= 0 and 0 <= legal <= C (q_pos0=%d "
                    "legal=%d C=%d)", q_pos0, legal, C);
    ATTNLAB_REQUIRE((int64_t)q_pos0 + T < INT32_MAX, "query positions past 2^31");
    ATTNLAB_REQUIRE(window >= 0 && sinks >= 0, "window=%d and sinks=%d must not be negative", window, sinks);
    ATTNLAB_REQUIRE(1 <= splits && splits <= kMaxSplits, "key splits %d outside [1, %d]", splits, kMaxSplits);
    if (T == 0) return ATTNLAB_OK;
    ATTNLAB_REQUIRE(q && K && V && out, "q, K, V and out are required");
    ATTNLAB_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(K) | reinterpret_cast<uintptr_t>(V) |
                      reinterpret_cast<uintptr_t>(out)) & 15) == 0, "q, K, V and out must be 16-byte aligned");
    const int64_t need = attnlab_range_prefill_part_bytes(B, G, h, T, splits);
    ATTNLAB_REQUIRE(splits == 1 || (part != nullptr && (reinterpret_cast<uintptr_t>(part) & 15) == 0 && part_bytes >= need),
                    "%d key splits need a 16-byte aligned part buffer of %lld bytes", splits, (long long)need);
    const bool q8 = k_exp != nullptr;
    const int bq = kRows / h;
    RangePrefillArgs a{q, K, V, k_exp, v_exp, out, h, T, q_pos0, legal, C, block == 16 ? 4 : block == 32 ? 5 : 6,
                       q8 ? (C + block - 1) / block : 0, window, sinks, bq, (T + bq - 1) / bq, scale * kLog2e, splits,
                       part};
    const int64_t blocks = (int64_t)B * G * a.qtiles * splits, rows = (int64_t)B * G * h * T;
    ATTNLAB_REQUIRE(blocks < (int64_t)1 << 31 && rows * 32 / 256 < (int64_t)1 << 31,
                    "grid of %lld workgroups is too large", (long long)blocks);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)blocks), wg(256);
    if (splits > 1) {
        if (q8) hipLaunchKernelGGL((range_prefill<true, true>), grid, wg, 0, s, a);
        else hipLaunchKernelGGL((range_prefill<true, false>), grid, wg, 0, s, a);
        hipLaunchKernelGGL(range_prefill_combine, dim3((unsigned)((rows * 32 + 255) / 256)), wg, 0, s, part, out, splits,
                           rows);
    } else if (q8) {
        hipLaunchKernelGGL((range_prefill<false, true>), grid, wg, 0, s, a);
    } else {
        hipLaunchKernelGGL((range_prefill<false, false>), grid, wg, 0, s, a);
    }
    return check_launch("range_prefill");
}
