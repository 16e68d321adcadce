// Causal attention of a chunk of queries over a cache whose visible positions end in a sliding window and a few first
// tokens (sinks), or are all the legal ones; over a bf16 cache or an 8-bit one (quant.h). Query t sits at p = q_pos0 + t:
//   out[b,g,i,t] = sum_j softmax_j(scale q[b,g,i,t] . k_j) v_j    over j <= p, j < legal, (j > p - window or j < sinks)
//
// A workgroup owns 128 (query, head) rows, 128 / h consecutive queries with all h heads, and walks blocks of 64 keys: the
// blocks of the sinks, then those from the first query's window on. Per block S^T = K Q^T, the softmax on its
// accumulators, O^T += V^T P^T (v_mfma_f32_32x32x16_bf16; a row's softmax state and outputs stay in lanes n and n + 32),
// with K and V as bf16 tiles in LDS, a block ahead, one barrier a block. The bf16 cache is copied into LDS directly; an
// 8-bit one passes through registers, 32 codes a thread and tensor, each converted once for all four waves (exactly, its
// scale included), while the block before it is computed.
//
// A masked key has weight zero, but zero times a V row that holds NaN or infinity is NaN. Rows past the visible range are
// written as zeros; inside it a key can be masked for one row and visible to the next, so a row whose result is not
// finite is computed again key by key, over its visible keys alone (row_again).
#include <cfloat>

#include "mfma_attend.h"
#include "quant.h"

namespace attnlab {

int check_quant_cache(const void* k_codes, const void* v_codes, const void* k_exp, const void* v_exp, int B, int G,
                      int C, int block);

namespace {

constexpr int kDim = 128;
constexpr int kRows = 128;          // (query, head) rows per workgroup: 4 waves x 32
constexpr int kKeys = 64;           // keys per block
constexpr float kLazy = 8.0f;       // rescale O only when the running max grows by more than 2^8
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

// A row's outputs from the formula over the block's visible keys, one at a time, by one wave: lane l holds dims 2 l and
// 2 l + 1.
template <bool Q8>
__device__ __forceinline__ void row_again(const RangePrefillArgs& a, int bg, int pos, int kb, float q0, float q1,
                                          float& m, float& l, float& a0, float& a1) {
    const int lane = threadIdx.x & 63;
    for (int j = 0; j < kKeys; ++j) {
        const int key = kb + j;
        if (key > pos || key >= a.legal) break;
        if (a.window > 0 && key <= pos - a.window && key >= a.sinks) continue;
        float k0, k1, v0, v1;
        const size_t at = ((size_t)bg * a.C + key) * kDim + 2 * lane;
        if constexpr (Q8) {
            const float ks = scale_of(a.ke[(size_t)bg * a.nb + (key >> a.shift)]);
            const float vs = scale_of(a.ve[(size_t)bg * a.nb + (key >> a.shift)]);
            const qf32x2_t kk = e4m3_to_f32x2<false>(*reinterpret_cast<const uint16_t*>((const uint8_t*)a.K + at));
            const qf32x2_t vv = e4m3_to_f32x2<false>(*reinterpret_cast<const uint16_t*>((const uint8_t*)a.V + at));
            k0 = kk.x * ks;
            k1 = kk.y * ks;
            v0 = vv.x * vs;
            v1 = vv.y * vs;
        } else {
            const uint32_t kk = *reinterpret_cast<const uint32_t*>((const uint16_t*)a.K + at);
            const uint32_t vv = *reinterpret_cast<const uint32_t*>((const uint16_t*)a.V + at);
            k0 = bf16_lo(kk);
            k1 = bf16_hi(kk);
            v0 = bf16_lo(vv);
            v1 = bf16_hi(vv);
        }
        float x = q0 * k0 + q1 * k1;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d, 64);
        x *= a.scale_log2;
        if (x > m) {
            const float al = fast_exp2(m - x);
            l *= al;
            a0 *= al;
            a1 *= al;
            m = x;
        }
        const float p = fast_exp2(x - (m == -INFINITY ? 0.0f : m));
        l += p;
        a0 += p * v0;
        a1 += p * v1;
    }
}

// K and V blocks in LDS: 64 rows of 256 bytes, sixteen 16-byte chunks each, permuted within the row so that the operand
// reads meet no bank twice. K: chunk c of row j at slot c ^ (j & 15) (16 rows, one chunk). V: chunk c of row j at slot
// c ^ (4 (j & 3)) (a transposing read takes 4 chunks of 4 consecutive rows).
template <bool SPLIT, bool Q8>
__global__ __launch_bounds__(256, 2) void range_prefill(RangePrefillArgs a) {
    __shared__ __attribute__((aligned(1024))) uint16_t kt0[kKeys * kDim], vt0[kKeys * kDim];
    __shared__ __attribute__((aligned(1024))) uint16_t kt1[kKeys * kDim], vt1[kKeys * kDim];
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
    bf16x8_t qb[8];                              // B operand of S^T: row R, dims 16 kk + 8 g .. + 7
    {
        const uint16_t* qr = a.q + (((size_t)bg * a.h + head) * a.T + tc) * kDim + 8 * g;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) qb[kk] = __builtin_bit_cast(bf16x8_t, *reinterpret_cast<const u32x4_t*>(qr + 16 * kk));
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

    // staging. bf16: load u of wave w fills rows 16 u + 4 w .. + 3 of a tile, lane l slot l % 16 of row l / 16 of them, from
    // a buffer of those 4 rows (rows past kend give zeros)
    const int srow = 4 * wave + (lane >> 4);
    const uint32_t koff = 256u * (lane >> 4) + 16u * ((lane & 15) ^ srow);
    const uint32_t voff = 256u * (lane >> 4) + 16u * ((lane & 15) ^ ((lane >> 4) << 2));
    const uint16_t* Kb = reinterpret_cast<const uint16_t*>(a.K) + (size_t)bg * a.C * kDim;
    const uint16_t* Vb = reinterpret_cast<const uint16_t*>(a.V) + (size_t)bg * a.C * kDim;
    auto copy = [&](int kb, uint16_t* kt, uint16_t* vt) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int row = kb + 16 * u + 4 * wave;
            const uint32_t bytes = 256u * (uint32_t)__builtin_amdgcn_readfirstlane(max(min(kend - row, 4), 0));
            load_lds16_buf(Kb + (size_t)row * kDim, bytes, koff, kt + (16 * u + 4 * wave) * kDim);
            load_lds16_buf(Vb + (size_t)row * kDim, bytes, voff, vt + (16 * u + 4 * wave) * kDim);
        }
    };
    // 8-bit: 16 codes of rows tid / 8 and 32 + tid / 8 of each tensor through registers
    const uint8_t* K8 = reinterpret_cast<const uint8_t*>(a.K) + (size_t)bg * a.C * kDim;
    const uint8_t* V8 = reinterpret_cast<const uint8_t*>(a.V) + (size_t)bg * a.C * kDim;
    const uint8_t* keb = Q8 ? a.ke + (size_t)bg * a.nb : nullptr;
    const uint8_t* veb = Q8 ? a.ve + (size_t)bg * a.nb : nullptr;
    u32x4_t rk[2], rv[2];
    uint32_t xk[2], xv[2];
    auto fetch = [&](int kb) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int row = kb + 32 * u + (tid >> 3);
            const int rc = min(row, kend - 1);
            rk[u] = *reinterpret_cast<const u32x4_t*>(K8 + (size_t)rc * kDim + 16 * (tid & 7));
            rv[u] = *reinterpret_cast<const u32x4_t*>(V8 + (size_t)rc * kDim + 16 * (tid & 7));
            xk[u] = keb[rc >> a.shift];
            xv[u] = veb[rc >> a.shift];
            if (row >= kend) rk[u] = rv[u] = u32x4_t{0, 0, 0, 0};
        }
    };
    auto expand = [&](uint16_t* kt, uint16_t* vt) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int row = 32 * u + (tid >> 3), c = 2 * (tid & 7);
            auto put = [&](uint16_t* tile, int swz, const u32x4_t& w, float s) {
                u32x4_t* dst = reinterpret_cast<u32x4_t*>(tile + row * kDim);
                dst[c ^ swz] = u32x4_t{e4m3_to_bf16x2<false>(w.x, s), e4m3_to_bf16x2<true>(w.x, s),
                                       e4m3_to_bf16x2<false>(w.y, s), e4m3_to_bf16x2<true>(w.y, s)};
                dst[(c + 1) ^ swz] = u32x4_t{e4m3_to_bf16x2<false>(w.z, s), e4m3_to_bf16x2<true>(w.z, s),
                                             e4m3_to_bf16x2<false>(w.w, s), e4m3_to_bf16x2<true>(w.w, s)};
            };
            put(kt, row & 15, rk[u], scale_of(xk[u]));
            put(vt, 4 * (row & 3), rv[u], scale_of(xv[u]));
        }
    };
    // operand reads, as byte offsets into a tile: K row 32 kt + n, chunk 2 kk + g; V rows 16 ks + 8 hf + 4 g + e, dims
    // 32 dt + 16 (lane / 16 % 2) + 4 j .. + 3, e = lane % 16 / 4, j = lane % 4. `pin` keeps the compiler from holding a
    // copy of each per tile.
    uint32_t kof[8], vof[4];
    const int ve = (lane >> 2) & 3;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) kof[kk] = 256 * n + 16 * ((2 * kk) ^ g ^ (n & 15));
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) vof[dt] = 256 * (4 * g + ve) + 64 * (dt ^ ve) + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
    auto pin = [&]() {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) asm volatile("" : "+v"(kof[kk]));
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) asm volatile("" : "+v"(vof[dt]));
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

    auto block = [&](int kb, const uint16_t* kt, const uint16_t* vt) {
        // no key of the block is visible to a row of this wave
        if (kb >= kend_wave || (a.window > 0 && kb >= a.sinks && kb + kKeys - 1 <= wfirst - a.window)) return;
        const char* ks = reinterpret_cast<const char*>(kt);
        const char* vs = reinterpret_cast<const char*>(vt);
        f32x16_t s[2];
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[x][i] = 0.0f;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const bf16x8_t ka = __builtin_bit_cast(bf16x8_t, *reinterpret_cast<const u32x4_t*>(ks + 8192 * x + kof[kk]));
                s[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka, qb[kk], s[x], 0, 0, 0);
            }
        // this lane's scores: row R, keys kb + 4 g + c, c = 32 x + 8 (i / 4) + i % 4. The bounds that a block needs are
        // applied apart, each a compare with a constant and a select
        const int at = kb + 4 * g;
        if (kb + kKeys - 1 > wfirst || kb + kKeys > a.legal) {
            const int most = min(pos, a.legal - 1) - at;
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[x][i] = 32 * x + 8 * (i >> 2) + (i & 3) <= most ? s[x][i] : -INFINITY;
        }
        if (a.window > 0 && kb <= wlast - a.window && kb + kKeys > a.sinks) {
            const int from = pos - a.window - at;   // visible: c > from, or c < sink
            if (kb >= a.sinks) {
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[x][i] = 32 * x + 8 * (i >> 2) + (i & 3) > from ? s[x][i] : -INFINITY;
            } else {
                const int sink = a.sinks - at;
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int c = 32 * x + 8 * (i >> 2) + (i & 3);
                        s[x][i] = (c > from) | (c < sink) ? s[x][i] : -INFINITY;
                    }
            }
        }
        float bm = -INFINITY;
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int i = 0; i < 16; ++i) bm = fmaxf(bm, s[x][i]);
        bm = max_xor32(bm) * sc;
        if (bm > m_run + kLazy) {   // also the first keys of the row (m_run = -inf)
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
#pragma unroll
        for (int ks2 = 0; ks2 < 4; ++ks2) {
#pragma unroll
            for (int dt = 0; dt < 4; ++dt) {
                const char* vp = vs + 4096 * ks2 + vof[dt];
                const u32x2v_t lo4 = read_tr16(vp), hi4 = read_tr16(vp + 8 * 256);
                const bf16x8_t va = __builtin_bit_cast(bf16x8_t, u32x4_t{lo4.x, lo4.y, hi4.x, hi4.y});
                o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va, pb[ks2], o[dt], 0, 0, 0);
            }
        }
    };
    // Two tile pairs: the next block's copies (or its loads into registers) are issued when every wave has left the tiles
    // they overwrite, the barrier that also publishes the current block, and land while it is computed.
    if constexpr (Q8) {
        auto publish = [&]() {
            __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0): this wave's LDS stores and reads are done
            asm volatile("s_barrier" ::: "memory");
            pin();
        };
        if (i0 < i1) {
            fetch(first_key(i0));
            expand(kt0, vt0);
        }
        for (int i = i0; i < i1; i += 2) {
            publish();
            if (i + 1 < i1) fetch(first_key(i + 1));
            block(first_key(i), kt0, vt0);
            if (i + 1 >= i1) break;
            expand(kt1, vt1);
            publish();
            if (i + 2 < i1) fetch(first_key(i + 2));
            block(first_key(i + 1), kt1, vt1);
            if (i + 2 < i1) expand(kt0, vt0);
        }
    } else {
        auto publish = [&]() {
            __builtin_amdgcn_s_waitcnt(0x0070);   // vmcnt(0) lgkmcnt(0): this wave's copies have landed, its reads are done
            asm volatile("s_barrier" ::: "memory");
            pin();
        };
        if (i0 < i1) copy(first_key(i0), kt0, vt0);
        for (int i = i0; i < i1; i += 2) {
            publish();
            if (i + 1 < i1) copy(first_key(i + 1), kt1, vt1);
            block(first_key(i), kt0, vt0);
            if (i + 1 >= i1) break;
            publish();
            if (i + 2 < i1) copy(first_key(i + 2), kt0, vt0);
            block(first_key(i + 1), kt1, vt1);
        }
    }
    const float l_tot = l_run + shfl_xor_f32(l_run, 32);
    const bool row = t < tend;
    // a row whose result is not finite: from its visible keys alone
    float finite = 0.0f * l_tot;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) finite = fmaf(0.0f, o[dt][i], finite);
    const uint64_t bad2 = __ballot(row && finite != 0.0f);
    const uint32_t bad = (uint32_t)bad2 | (uint32_t)(bad2 >> 32);
    for (uint32_t left = bad; left; left &= left - 1) {
        const int r = 32 * wave + __builtin_ctz(left);
        const int rt = t0 + r / a.h, rh = r % a.h;
        const uint16_t* qr = a.q + (((size_t)bg * a.h + rh) * a.T + rt) * kDim;
        const uint32_t qw = *reinterpret_cast<const uint32_t*>(qr + 2 * lane);
        float m = -INFINITY, l = 0.0f, a0 = 0.0f, a1 = 0.0f;
        for (int i = i0; i < i1; ++i)
            row_again<Q8>(a, bg, a.q_pos0 + rt, first_key(i), bf16_lo(qw), bf16_hi(qw), m, l, a0, a1);
        if constexpr (SPLIT) {
            float* pp = a.part + ((((size_t)bg * a.h + rh) * a.T + rt) * a.splits + sp) * kPart;
            if (lane == 0) {
                pp[0] = m;
                pp[1] = l;
            }
            *reinterpret_cast<float2*>(pp + 4 + 2 * lane) = make_float2(a0, a1);
        } else {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            *reinterpret_cast<uint32_t*>(a.out + (((size_t)bg * a.h + rh) * a.T + rt) * kDim + 2 * lane) =
                pack_bf16x2(a0 * inv, a1 * inv);
        }
    }
    if (!row || (bad >> n & 1)) return;
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
