// One query's attention over part of a cache, on the matrix cores: the positions of a sliding window and a few first
// tokens (sinks), every legal position, or a listed set of rows; over a bf16 cache or an 8-bit one (quant.h).
//   out[b,g,i] = sum_j softmax_j(scale q[b,g,i] . k_j) v_j    over j in [0, s) U [lo, n), or over the listed rows
//
// A wave takes 32 rows at a time: S^T[keys, heads] = K Q^T, two 16-key tiles of v_mfma_f32_16x16x32_bf16, then
// O^T[dims, heads] += V^T P^T, eight 16-dim tiles. K's rows are read from memory in the operand's order (16 keys over
// the lanes, a row's bytes over the four lane groups), so K goes from the load to the matrix core; V's rows are written
// to the wave's own 8 KB of LDS and read transposed (ds_read_b64_tr_b16). Both are loaded a tile ahead, and a wave waits
// for no other until the end. An 8-bit code becomes a bf16 exactly, its block's scale included, in the one conversion
// (v_cvt_scalef32_pk_bf16_fp8).
//
// The 16 columns of a tile are 8 heads twice: columns 0..7 multiply V by P rounded to bf16, columns 8..15 by what that
// rounding left, and the two are added at the end, so the weights keep 16 bits without a second product. Softmax is
// online in the log2 domain with a lazy rescale; sums and outputs are fp32. The waves of a workgroup merge through LDS,
// the P workgroups of a (b, g) through partials and a second small launch: no state outlives the call, so two graphs, or
// two streams, share nothing.
//
// Masked rows: their scores are replaced, and their V rows written as zeros, so whatever they hold (NaN, infinity) leaves
// the output alone. A query with no row to read, or whose scores are all -inf, gets zeros.
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
constexpr float kLazy = 8.0f;       // the running max grows only by more than 2^8
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
    int G, h, C, P, shift, nb;
    int n;                    // keys [0, n); the number of listed rows
    int64_t qend;             // the query's position + 1, where the window ends
    int window, sinks;        // window 0: none
    float scale_log2;
    void* out;
    int out_bf16;
    float* part;              // [B * G, P, h, 130]: m, l, the unnormalised outputs (P > 1)
};

// One tile of a wave in flight. 8-bit: K two 16-byte loads a row (bytes 16 g .. and 64 + 16 g ..), V eight lanes a row;
// bf16: twice as many. `ex`: lane l holds the scale byte of row l % 32, of K (l < 32) or V.
template <bool Q8>
struct Tile {
    u32x4_t k[2][Q8 ? 2 : 4];
    u32x4_t v[Q8 ? 4 : 8];
    uint32_t ex;
};

template <bool Q8, bool LIST>
__global__ __launch_bounds__(256, 2) void range_attend(RangeArgs a) {
    constexpr int kRow = Q8 ? kDim : 2 * kDim;          // bytes of a row
    constexpr int kLanes = kRow / 16;                   // lanes of a V row
    __shared__ __attribute__((aligned(1024))) uint16_t v_sh[kWaves][kTile * kDim];   // a wave's V tile; then the merge
    __shared__ float ml_sh[kWaves][16][2];
    __shared__ int list_sh[LIST ? kListChunk : 1];
    const int lin = xcd_contiguous_block();
    const int bg = lin / a.P, p = lin - bg * a.P;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n16 = lane & 15, g4 = lane >> 4;

    // the entries 0 .. count - 1 of this (b, g): positions [0, s) and [lo, n), or the list
    int s = 0, lo = 0, count = a.n;
    if constexpr (!LIST) {
        int n = a.n;
        int64_t qend = a.qend;
        if (a.lengths) {
            n = min(max(a.lengths[bg / a.G], 0), a.C);
            qend = n;
        }
        if (a.window > 0) {
            s = min(a.sinks, n);
            const int64_t from = qend - a.window;
            lo = (int)min((int64_t)n, max(from, (int64_t)s));
        }
        count = s + n - lo;
    }
    // partitions of whole tiles
    const int tiles = (count + kTile - 1) / kTile;
    const int per = ((tiles + a.P - 1) / a.P) * kTile;
    const int e0 = (int)min((int64_t)p * per, (int64_t)count), e1 = min(e0 + per, count);

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
    const uint8_t* Kb = a.K + (size_t)bg * a.C * kRow;
    const uint8_t* Vb = a.V + (size_t)bg * a.C * kRow;
    const uint8_t* keb = Q8 ? a.ke + (size_t)bg * a.nb : nullptr;
    const uint8_t* veb = Q8 ? a.ve + (size_t)bg * a.nb : nullptr;

    float m = -INFINITY, l = 0.0f;
    f32x4_t o[8];
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) o[dt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    uint16_t* vt = v_sh[wave];

    for (int c0 = e0; c0 < e1; c0 += LIST ? kListChunk : max(e1 - e0, 1)) {
        const int clen = LIST ? min(kListChunk, e1 - c0) : e1 - c0;
        if constexpr (LIST) {
            if (c0 != e0) __syncthreads();
            const int32_t* src = a.rows + (size_t)bg * a.rows_stride + c0;
            for (int i = tid; i < clen; i += 256) {
                const int pos = src[i];
                list_sh[i] = (unsigned)pos < (unsigned)a.C ? pos : -1;
            }
            __syncthreads();
        }
        const int nt = (clen + kTile - 1) / kTile;
        // entry e of the chunk -> its position, or -1: past the chunk, or a listed position outside [0, C)
        auto position = [&](int e) -> int {
            if constexpr (LIST) return e < clen ? list_sh[e] : -1;
            const int x = c0 + e;
            return e < clen ? (x < s ? x : x - s + lo) : -1;
        };
        auto issue = [&](int t, Tile<Q8>& f) {
            const int e = kTile * t;
#pragma unroll
            for (int t2 = 0; t2 < 2; ++t2) {
                const uint8_t* r = Kb + (size_t)max(position(e + 16 * t2 + n16), 0) * kRow + 16 * g4;
#pragma unroll
                for (int c = 0; c < (Q8 ? 2 : 4); ++c)
                    f.k[t2][c] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(r + 64 * c));
            }
#pragma unroll
            for (int u = 0; u < (Q8 ? 4 : 8); ++u) {
                const int row = u * (64 / kLanes) + lane / kLanes;
                const uint8_t* r = Vb + (size_t)max(position(e + row), 0) * kRow + 16 * (lane % kLanes);
                f.v[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(r));
            }
            if constexpr (Q8) f.ex = (lane < 32 ? keb : veb)[max(position(e + (lane & 31)), 0) >> a.shift];
        };
        auto compute = [&](int t, const Tile<Q8>& f) {
            const int e = kTile * t;
            const uint32_t ok = (uint32_t)__ballot(position(e + (lane & 31)) >= 0);   // rows of the tile to read
            f32x4_t sc[2];
#pragma unroll
            for (int t2 = 0; t2 < 2; ++t2) {
                sc[t2] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
                float ks = 1.0f;
                if constexpr (Q8) ks = scale_of(__shfl(f.ex, 16 * t2 + n16, 64));
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
                    sc[t2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, w), qb[kk], sc[t2], 0,
                                                                     0, 0);
                }
            }
            // this lane's scores: column n16, rows 16 t2 + 4 g4 + i
            float bm = -INFINITY;
#pragma unroll
            for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float x = sc[t2][i] * a.scale_log2;
                    if (ok != 0xffffffffu && !(ok >> (16 * t2 + 4 * g4 + i) & 1)) x = -INFINITY;
                    sc[t2][i] = x;
                    bm = fmaxf(bm, x);
                }
            bm = fmaxf(bm, shfl_xor_f32(bm, 16));
            bm = fmaxf(bm, shfl_xor_f32(bm, 32));
            if (__any(bm > m + kLazy)) {
                if (bm > m + kLazy) {   // also a column's first rows (m = -inf)
                    const float al = fast_exp2(m - bm);
                    l *= al;
#pragma unroll
                    for (int dt = 0; dt < 8; ++dt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[dt][i] *= al;
                    m = bm;
                }
            }
            const float mb = m == -INFINITY ? 0.0f : m;   // no score above -inf yet: every weight 0
            uint32_t w4[4];
#pragma unroll
            for (int t2 = 0; t2 < 2; ++t2) {
                float pr[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    pr[i] = fast_exp2(sc[t2][i] - mb);
                    l += pr[i];
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t hi = pack_bf16x2(pr[2 * i], pr[2 * i + 1]);
                    const uint32_t rest = pack_bf16x2(pr[2 * i] - bf16_lo(hi), pr[2 * i + 1] - bf16_hi(hi));
                    w4[2 * t2 + i] = n16 < 8 ? hi : rest;
                }
            }
            const bf16x8_t pb = __builtin_bit_cast(bf16x8_t, u32x4_t{w4[0], w4[1], w4[2], w4[3]});
            // V into LDS as bf16 rows of 16 chunks of 8; chunk c of row r at c ^ (4 (r & 3)), so that a transposing
            // read's four rows lie in four different quarters of the banks
#pragma unroll
            for (int u = 0; u < (Q8 ? 4 : 8); ++u) {
                const int row = u * (64 / kLanes) + lane / kLanes, c = lane % kLanes;
                u32x4_t x = f.v[u];
                if (ok != 0xffffffffu && !(ok >> row & 1)) x = u32x4_t{0, 0, 0, 0};
                u32x4_t* dst = reinterpret_cast<u32x4_t*>(vt + row * kDim);
                const int swz = 4 * (row & 3);
                if constexpr (Q8) {
                    const float vs = scale_of(__shfl(f.ex, 32 + row, 64));
                    dst[(2 * c) ^ swz] = u32x4_t{e4m3_to_bf16x2<false>(x.x, vs), e4m3_to_bf16x2<true>(x.x, vs),
                                                 e4m3_to_bf16x2<false>(x.y, vs), e4m3_to_bf16x2<true>(x.y, vs)};
                    dst[(2 * c + 1) ^ swz] = u32x4_t{e4m3_to_bf16x2<false>(x.z, vs), e4m3_to_bf16x2<true>(x.z, vs),
                                                     e4m3_to_bf16x2<false>(x.w, vs), e4m3_to_bf16x2<true>(x.w, vs)};
                } else {
                    dst[c ^ swz] = x;
                }
            }
            // a wave's LDS operations take effect in order; these keep the compiler from moving them past each other
            asm volatile("" ::: "memory");
            const int j = n16 >> 2;   // row of the four this lane reads from, elements 4 (n16 % 4) ..
#pragma unroll
            for (int dt = 0; dt < 8; ++dt) {
                u32x2v_t w[2];
#pragma unroll
                for (int t2 = 0; t2 < 2; ++t2) {
                    const int row = 16 * t2 + 4 * g4 + j;
                    const int slot = (2 * dt + ((n16 >> 1) & 1)) ^ (4 * (row & 3));
                    w[t2] = read_tr16(reinterpret_cast<const char*>(vt) + 256 * row + 16 * slot + 8 * (n16 & 1));
                }
                const bf16x8_t va = __builtin_bit_cast(bf16x8_t, u32x4_t{w[0].x, w[0].y, w[1].x, w[1].y});
                o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, pb, o[dt], 0, 0, 0);
            }
            asm volatile("" ::: "memory");
        };
        // tile t of the chunk belongs to wave t % kWaves; the next one is in flight while one is computed
        Tile<Q8> f[2];
        int t = wave;
        if (t < nt) issue(t, f[0]);
        while (t < nt) {
            if (t + kWaves < nt) issue(t + kWaves, f[1]);
            compute(t, f[0]);
            t += kWaves;
            if (t >= nt) break;
            if (t + kWaves < nt) issue(t + kWaves, f[0]);
            compute(t, f[1]);
            t += kWaves;
        }
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
    for (int idx = tid; idx < a.h * kDim; idx += 256) {
        const int i = idx / kDim, d = idx - i * kDim;
        float ms = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) ms = fmaxf(ms, ml_sh[w][i][0]);
        float ls = 0.0f, as = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float mw = ml_sh[w][i][0], lw = ml_sh[w][i][1];
            // a wave without a finite score has m = -inf: nothing to add, unless its scores were NaN
            const float ww = mw == -INFINITY ? (lw == 0.0f ? 0.0f : 1.0f) : fast_exp2(mw - ms);
            ls += ww * lw;
            as += ww * (red[(w * 16 + i) * kDim + d] + red[(w * 16 + 8 + i) * kDim + d]);
        }
        if (a.P == 1) {
            const float r = ls == 0.0f ? 0.0f : as / ls;
            const size_t at = ((size_t)bg * a.h + i) * kDim + d;
            if (a.out_bf16) reinterpret_cast<uint16_t*>(a.out)[at] = f32_to_bf16_rne(r);
            else reinterpret_cast<float*>(a.out)[at] = r;
        } else {
            float* pp = a.part + (((size_t)bg * a.P + p) * a.h + i) * kPartWords;
            if (d == 0) {
                pp[0] = ms;
                pp[1] = ls;
            }
            pp[2 + d] = as;
        }
    }
}

// The partials of every (b, g, head) merged in partition order: thread -> (head, dim).
__global__ __launch_bounds__(128) void range_combine(RangeArgs a) {
    const int lin = xcd_contiguous_block();
    const int bg = lin / a.h, i = lin - bg * a.h, d = threadIdx.x;
    const float* pb = a.part + ((size_t)bg * a.P * a.h + i) * kPartWords;
    const size_t step = (size_t)a.h * kPartWords;
    float ms = -INFINITY, ls = 0.0f, as = 0.0f;
    constexpr int kGroup = 8;   // partials in flight
    for (int p0 = 0; p0 < a.P; p0 += kGroup) {
        float mv[kGroup], lv[kGroup], av[kGroup];
#pragma unroll
        for (int u = 0; u < kGroup; ++u) {
            mv[u] = -INFINITY;
            lv[u] = av[u] = 0.0f;
            if (p0 + u < a.P) {
                const float* pp = pb + (p0 + u) * step;
                mv[u] = pp[0];
                lv[u] = pp[1];
                av[u] = pp[2 + d];
            }
        }
        float mn = ms;
#pragma unroll
        for (int u = 0; u < kGroup; ++u) mn = fmaxf(mn, mv[u]);
        const float w0 = ms == -INFINITY ? 1.0f : fast_exp2(ms - mn);
        ls *= w0;
        as *= w0;
#pragma unroll
        for (int u = 0; u < kGroup; ++u) {
            const float w = mv[u] == -INFINITY ? (lv[u] == 0.0f ? 0.0f : 1.0f) : fast_exp2(mv[u] - mn);
            ls += w * lv[u];
            as += w * av[u];
        }
        ms = mn;
    }
    const float r = ls == 0.0f ? 0.0f : as / ls;
    const size_t at = ((size_t)bg * a.h + i) * kDim + d;
    if (a.out_bf16) reinterpret_cast<uint16_t*>(a.out)[at] = f32_to_bf16_rne(r);
    else reinterpret_cast<float*>(a.out)[at] = r;
}

template <bool LIST>
int launch_range(const RangeArgs& a, int B, hipStream_t s) {
    const int64_t blocks = (int64_t)B * a.G * a.P;
    ATTNLAB_REQUIRE(blocks < (int64_t)1 << 31, "grid of %lld workgroups is too large", (long long)blocks);
    const dim3 grid((unsigned)blocks), wg(256);
    if constexpr (LIST) hipLaunchKernelGGL((range_attend<true, true>), grid, wg, 0, s, a);
    else if (a.ke) hipLaunchKernelGGL((range_attend<true, false>), grid, wg, 0, s, a);
    else hipLaunchKernelGGL((range_attend<false, false>), grid, wg, 0, s, a);
    if (a.P > 1) hipLaunchKernelGGL(range_combine, dim3((unsigned)(B * a.G * a.h)), dim3(kDim), 0, s, a);
    return check_launch(LIST ? "range_attend (rows)" : "range_attend");
}

int check_range(const void* K, const void* V, const uint8_t* k_exp, const uint8_t* v_exp, int block, const uint16_t* q,
                int B, int G, int h, int C, int P, const void* out, const float* part) {
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
    ATTNLAB_REQUIRE(P == 1 || part != nullptr, "P > 1 needs the partial buffer");
    return ATTNLAB_OK;
}

RangeArgs range_args(const void* K, const void* V, const uint8_t* k_exp, const uint8_t* v_exp, int block,
                     const uint16_t* q, int G, int h, int C, int P, float scale, void* out, int out_bf16, float* part) {
    RangeArgs a{};
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
    return a;
}

}  // namespace
}  // namespace attnlab

using namespace attnlab;

extern "C" int attnlab_range_decode(const void* K, const void* V, const uint8_t* k_exp, const uint8_t* v_exp, int block,
                                    const uint16_t* q, const int32_t* lengths, int length, int64_t q_pos, int window,
                                    int sinks, int B, int G, int h, int C, int P, float scale, void* out, int out_bf16,
                                    float* part, void* stream) {
    const int rc = check_range(K, V, k_exp, v_exp, block, q, B, G, h, C, P, out, part);
    if (rc) return rc;
    ATTNLAB_REQUIRE(lengths != nullptr || (0 <= length && length <= C), "valid length %d outside [0, C=%d]", length, C);
    ATTNLAB_REQUIRE(lengths != nullptr || q_pos >= 0, "the query's position %lld must not be negative",
                    (long long)q_pos);
    ATTNLAB_REQUIRE(window >= 0 && sinks >= 0, "window=%d and sinks=%d must not be negative", window, sinks);
    RangeArgs a = range_args(K, V, k_exp, v_exp, block, q, G, h, C, P, scale, out, out_bf16, part);
    a.lengths = lengths;
    a.n = lengths ? 0 : (int)(q_pos + 1 < length ? q_pos + 1 : length);   // causal: no key past the query
    a.qend = q_pos + 1;
    a.window = window;
    a.sinks = sinks;
    return launch_range<false>(a, B, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int attnlab_quant_attend(const uint8_t* k_codes, const uint8_t* v_codes, const uint8_t* k_exp,
                                    const uint8_t* v_exp, int block, const uint16_t* q, const int32_t* rows,
                                    int64_t rows_stride, int B, int G, int h, int S, int C, int P, float scale,
                                    void* out, int out_bf16, float* part, void* stream) {
    ATTNLAB_REQUIRE(k_exp && v_exp, "the scale bytes must be device pointers");
    const int rc = check_range(k_codes, v_codes, k_exp, v_exp, block, q, B, G, h, C, P, out, part);
    if (rc) return rc;
    ATTNLAB_REQUIRE(S >= 1, "at least one row must be selected (S=%d)", S);
    ATTNLAB_REQUIRE(rows != nullptr && rows_stride >= S, "rows must hold S=%d positions per (b, g)", S);
    RangeArgs a = range_args(k_codes, v_codes, k_exp, v_exp, block, q, G, h, C, P, scale, out, out_bf16, part);
    a.rows = rows;
    a.rows_stride = rows_stride;
    a.n = S;
    return launch_range<true>(a, B, reinterpret_cast<hipStream_t>(stream));
}
