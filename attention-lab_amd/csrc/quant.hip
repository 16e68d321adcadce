// Writing rows into the 8-bit K/V cache, and reading them back.
//
// The write of T rows at [start, start + T), for every block of `block` positions, KV head and tensor (K, V): N the new
// rows in the block, O the rows of the block before start,
//   need = the smallest scale with max |finite x in N| <= 448 * scale      scale = O empty ? need : max(old scale, need)
//   code(x) = RNE_e4m3(x / scale), non-finite x -> NaN                     O's codes move to the new scale if it grew
// so a block's scale grows only when a louder row arrives, by a power of two, and a row in it is converted once more.
// Rows of the block from start + T on keep their bytes. A caller that will take rows back keeps the last ones as they came
// (KEEP): a block's state follows from its rows and where each write began, so writing them again restores it.
//
// One workgroup of four waves owns 64 aligned positions of one (b, g) and one tensor, hence whole blocks of 16, 32 or
// 64: no block is shared, nothing is atomic. Each wave holds its 16 rows in registers (16 bytes a lane and load, a row
// over 16 lanes) from the maximum to the store, so a row is read once. Bound by its bytes: 3 per value from bf16. Four
// prompts of 32K (8 KV heads): 142 us, 5.7 TB/s, where a kernel that only reads two bytes for each that it writes reaches 6.3;
// the rows pass the caches (non-temporal loads and stores: 149 us without). One token of 16 requests: 3.9 us, the latency of
// a load, two barriers' worth of exchange and a store.
#include "quant.h"

namespace attnlab {
namespace {

constexpr int kSpan = 64;    // positions of one workgroup
constexpr int kDim = 128;

struct AppendArgs {
    const void* x[2];                 // K and V rows: element (b, g, t, e) at x + b sb + g sg + t st + e
    int64_t sb[2], sg[2], st[2];
    uint8_t* codes[2];                // [B, G, C, 128]
    uint8_t* exps[2];                 // [B, G, nb]
    const int32_t* starts;            // one per sequence, or null: `start`
    int start, G, T, C, shift, nb, spans;
    uint16_t* keep[2];                // [B, G, ring, 128] bf16: the rows as they came, position p in slot p % ring (KEEP)
    int ring;
};

// Eight elements of a row as floats.
template <int DT>
__device__ __forceinline__ void load8(const void* base, int64_t off, float (&v)[8]) {
    if constexpr (DT == ATTNLAB_DT_F32) {
        const u32x4_t* p = reinterpret_cast<const u32x4_t*>(reinterpret_cast<const float*>(base) + off);
        const u32x4_t a = p[0], b = p[1];   // the second load finds its half of the lines in the cache
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = __uint_as_float(a[i]);
            v[4 + i] = __uint_as_float(b[i]);
        }
    } else {
        const u32x4_t w = __builtin_nontemporal_load(
            reinterpret_cast<const u32x4_t*>(reinterpret_cast<const uint16_t*>(base) + off));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == ATTNLAB_DT_BF16) {
                v[2 * i] = bf16_lo(w[i]);
                v[2 * i + 1] = bf16_hi(w[i]);
            } else {
                v[2 * i] = f16_to_f32((uint16_t)w[i]);
                v[2 * i + 1] = f16_to_f32((uint16_t)(w[i] >> 16));
            }
        }
    }
}

// Two floats that are bf16 numbers as a packed pair.
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
    return __float_as_uint(lo) >> 16 | (__float_as_uint(hi) & 0xffff0000u);
}

template <int DT, bool KEEP>
__global__ __launch_bounds__(256) void quant_append(AppendArgs a) {
    __shared__ float top_sh[4];
    const int side = blockIdx.x & 1;                   // K, V
    const int lin = blockIdx.x >> 1;
    const int bg = lin / a.spans, sp = lin - bg * a.spans;
    const int b = bg / a.G, g = bg - b * a.G;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t start = a.starts ? a.starts[b] : a.start;
    const int64_t end = min(start + a.T, (int64_t)a.C);
    const int64_t span0 = ((start >> 6) + sp) * kSpan;          // >> rounds down for a negative start too
    if (start >= end || span0 >= end || span0 + kSpan <= 0) return;   // no new row inside [0, C) in this span
    const int chunk = lane & 15;
    float v[4][8];
    bool fresh[4];
    float top = 0.0f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int64_t pos = span0 + 16 * wave + 4 * u + (lane >> 4);
        fresh[u] = pos >= start && pos < end && pos >= 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[u][i] = 0.0f;
        if (fresh[u])
            load8<DT>(a.x[side], b * a.sb[side] + g * a.sg[side] + (pos - start) * a.st[side] + 8 * chunk, v[u]);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = fminf(fabsf(v[u][i]), kQuantLargest);
            top = fmaxf(top, __builtin_isfinite(v[u][i]) ? x : 0.0f);
        }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
    if (lane == 0) top_sh[wave] = top;
    // the wave's block: 1, 2 or 4 waves of the workgroup share one
    const int64_t blo = (span0 + 16 * wave) >> a.shift << a.shift;
    const int64_t bhi = blo + (1 << a.shift);
    const bool touched = blo < end && bhi > start && bhi > 0;    // a new row lies in the block
    const bool held = start > blo && start > 0;                  // rows before start lie in it (where touched)
    uint8_t* ep = a.exps[side] + (int64_t)bg * a.nb + (blo >> a.shift);
    const uint32_t was = touched && held ? *ep : 0;              // read by every wave of the block before one writes
    __syncthreads();
    if (!touched) return;
    const int per = 1 << (a.shift - 4);                          // waves to a block
    const int w0 = wave & ~(per - 1);
    for (int w = w0; w < w0 + per; ++w) top = fmaxf(top, top_sh[w]);
    const uint32_t need = scale_for(top);
    const uint32_t now = held ? max(was, need) : need;
    if (wave == w0 && lane == 0) *ep = (uint8_t)now;
    const float inv = scale_of(254 - now);                       // 2^(127 - now), exact
    uint8_t* rows = a.codes[side] + (int64_t)bg * a.C * kDim + 8 * chunk;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        if (!fresh[u]) continue;
        const int64_t pos = span0 + 16 * wave + 4 * u + (lane >> 4);
        if constexpr (KEEP) {   // of rows that share a slot, the last
            if (pos >= end - a.ring)
                *reinterpret_cast<u32x4_t*>(a.keep[side] + ((int64_t)bg * a.ring + pos % a.ring) * kDim + 8 * chunk) =
                    u32x4_t{bf16_pair(v[u][0], v[u][1]), bf16_pair(v[u][2], v[u][3]), bf16_pair(v[u][4], v[u][5]),
                            bf16_pair(v[u][6], v[u][7])};
        }
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {   // an infinity stays one (it becomes a NaN code), a finite value saturates
            const float x = v[u][i];
            y[i] = __builtin_isfinite(x) ? fminf(fmaxf(x, -kQuantLargest), kQuantLargest) * inv : x;
        }
        __builtin_nontemporal_store(
            u32x2_t{f32_to_e4m3x4(y[0], y[1], y[2], y[3]), f32_to_e4m3x4(y[4], y[5], y[6], y[7])},
            reinterpret_cast<u32x2_t*>(rows + pos * kDim));
    }
    if (!held || now == was) return;
    // the rows before start move to the larger scale: code * 2^(was - now), 0 where that is below fp32's range
    const int shift = (int)was - (int)now;
    const float move = shift < -126 ? 0.0f : scale_of(127 + shift);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int64_t pos = span0 + 16 * wave + 4 * u + (lane >> 4);
        if (pos >= start || pos < 0) continue;
        uint2* p = reinterpret_cast<uint2*>(rows + pos * kDim);
        const uint2 w = *p;
        const qf32x2_t a0 = e4m3_to_f32x2<false>(w.x), a1 = e4m3_to_f32x2<true>(w.x);
        const qf32x2_t a2 = e4m3_to_f32x2<false>(w.y), a3 = e4m3_to_f32x2<true>(w.y);
        *p = make_uint2(f32_to_e4m3x4(a0.x * move, a0.y * move, a1.x * move, a1.y * move),
                        f32_to_e4m3x4(a2.x * move, a2.y * move, a3.x * move, a3.y * move));
    }
}

struct ReadArgs {
    const uint8_t* codes[2];
    const uint8_t* exps[2];
    void* out[2];                     // [B, G, T, 128]
    const int32_t* starts;
    int start, G, T, C, shift, nb, tiles;
};

constexpr int kReadRows = 32;   // rows of a workgroup: 8 lanes of 16 codes each

// Positions outside [0, C) read as zeros.
template <int DT>
__global__ __launch_bounds__(256) void quant_read(ReadArgs a) {
    const int side = blockIdx.x & 1;
    const int lin = blockIdx.x >> 1;
    const int bg = lin / a.tiles, tile = lin - bg * a.tiles;
    const int t = tile * kReadRows + (threadIdx.x >> 3);
    if (t >= a.T) return;
    const int64_t pos = (int64_t)(a.starts ? a.starts[bg / a.G] : a.start) + t;
    const int e0 = 16 * (threadIdx.x & 7);
    u32x4_t w = {0, 0, 0, 0};
    float s = 1.0f;
    if (pos >= 0 && pos < a.C) {
        w = *reinterpret_cast<const u32x4_t*>(a.codes[side] + ((int64_t)bg * a.C + pos) * kDim + e0);
        s = scale_of(a.exps[side][(int64_t)bg * a.nb + (pos >> a.shift)]);
    }
    const int64_t off = ((int64_t)bg * a.T + t) * kDim + e0;
    if constexpr (DT == ATTNLAB_DT_BF16) {
        u32x4_t* o = reinterpret_cast<u32x4_t*>(reinterpret_cast<uint16_t*>(a.out[side]) + off);
        o[0] = u32x4_t{e4m3_to_bf16x2<false>(w.x, s), e4m3_to_bf16x2<true>(w.x, s), e4m3_to_bf16x2<false>(w.y, s),
                       e4m3_to_bf16x2<true>(w.y, s)};
        o[1] = u32x4_t{e4m3_to_bf16x2<false>(w.z, s), e4m3_to_bf16x2<true>(w.z, s), e4m3_to_bf16x2<false>(w.w, s),
                       e4m3_to_bf16x2<true>(w.w, s)};
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const qf32x2_t x = e4m3_to_f32x2<false>(w[i]), y = e4m3_to_f32x2<true>(w[i]);
            const float4 f = make_float4(x.x * s, x.y * s, y.x * s, y.y * s);
            if constexpr (DT == ATTNLAB_DT_F32) {
                reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out[side]) + off)[i] = f;
            } else {   // fp16: the one output type that rounds, to nearest even
                const uint32_t lo = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f.x) |
                                    (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f.y) << 16;
                const uint32_t hi = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f.z) |
                                    (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f.w) << 16;
                reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.out[side]) + off)[i] = make_uint2(lo, hi);
            }
        }
    }
}

int block_shift(int block) { return block == 16 ? 4 : block == 32 ? 5 : 6; }

bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }

}  // namespace

int check_quant_cache(const void* k_codes, const void* v_codes, const void* k_exp, const void* v_exp, int B, int G,
                      int C, int block) {
    ATTNLAB_REQUIRE(B >= 1 && G >= 1 && C >= 1, "B=%d G=%d C=%d must be positive", B, G, C);
    ATTNLAB_REQUIRE(block == 16 || block == 32 || block == 64, "block=%d must be 16, 32 or 64 positions", block);
    ATTNLAB_REQUIRE(k_codes && v_codes && k_exp && v_exp, "the codes and scale bytes must be device pointers");
    ATTNLAB_REQUIRE(aligned(k_codes, 16) && aligned(v_codes, 16), "the codes must be 16-byte aligned");
    return ATTNLAB_OK;
}

}  // namespace attnlab

using namespace attnlab;

namespace {

// keep_rows 0: no rows are kept.
int run_append(const void* k, int64_t k_b_stride, int64_t k_g_stride, int64_t k_t_stride, const void* v,
               int64_t v_b_stride, int64_t v_g_stride, int64_t v_t_stride, int dtype, uint8_t* k_codes, uint8_t* v_codes,
               uint8_t* k_exp, uint8_t* v_exp, const int32_t* starts, int start, int B, int G, int T, int C, int block,
               uint16_t* k_keep, uint16_t* v_keep, int keep_rows, void* stream) {
    const int rc = check_quant_cache(k_codes, v_codes, k_exp, v_exp, B, G, C, block);
    if (rc) return rc;
    ATTNLAB_REQUIRE(dtype == ATTNLAB_DT_BF16 || dtype == ATTNLAB_DT_F16 || dtype == ATTNLAB_DT_F32,
                    "rows must be bf16, fp16 or fp32 (dtype %d)", dtype);
    ATTNLAB_REQUIRE(T >= 0, "T=%d must not be negative", T);
    ATTNLAB_REQUIRE(starts != nullptr || (start >= 0 && (int64_t)start + T <= C), "rows [%d, %lld) outside the cache of "
                    "C=%d", start, (long long)start + T, C);
    if (T == 0) return ATTNLAB_OK;
    const int64_t step = dtype == ATTNLAB_DT_F32 ? 4 : 8;   // elements in 16 bytes
    ATTNLAB_REQUIRE(k && v, "k and v must be device pointers");
    ATTNLAB_REQUIRE(aligned(k, 16) && aligned(v, 16) && (k_b_stride | k_g_stride | k_t_stride | v_b_stride |
                                                         v_g_stride | v_t_stride) % step == 0,
                    "the rows of k and v must be 16-byte aligned");
    AppendArgs a{{k, v}, {k_b_stride, v_b_stride}, {k_g_stride, v_g_stride}, {k_t_stride, v_t_stride},
                 {k_codes, v_codes}, {k_exp, v_exp}, starts, start, G, T, C, block_shift(block), 0, 0,
                 {k_keep, v_keep}, keep_rows};
    a.nb = (C + block - 1) / block;
    // aligned spans that T rows touch: at any start, or at the one given
    a.spans = starts ? (int)(((int64_t)T + 62) / kSpan + 1) : (start + T - 1) / kSpan - start / kSpan + 1;
    const int64_t blocks = 2 * (int64_t)B * G * a.spans;
    ATTNLAB_REQUIRE(blocks < (int64_t)1 << 31, "grid of %lld workgroups is too large", (long long)blocks);
    const dim3 grid((unsigned)blocks), wg(256);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (keep_rows) hipLaunchKernelGGL((quant_append<ATTNLAB_DT_BF16, true>), grid, wg, 0, s, a);
    else if (dtype == ATTNLAB_DT_BF16) hipLaunchKernelGGL((quant_append<ATTNLAB_DT_BF16, false>), grid, wg, 0, s, a);
    else if (dtype == ATTNLAB_DT_F16) hipLaunchKernelGGL((quant_append<ATTNLAB_DT_F16, false>), grid, wg, 0, s, a);
    else hipLaunchKernelGGL((quant_append<ATTNLAB_DT_F32, false>), grid, wg, 0, s, a);
    return check_launch("quant_append");
}

}  // namespace

extern "C" int attnlab_quant_append(const void* k, int64_t k_b_stride, int64_t k_g_stride, int64_t k_t_stride,
                                    const void* v, int64_t v_b_stride, int64_t v_g_stride, int64_t v_t_stride,
                                    int dtype, uint8_t* k_codes, uint8_t* v_codes, uint8_t* k_exp, uint8_t* v_exp,
                                    const int32_t* starts, int start, int B, int G, int T, int C, int block,
                                    void* stream) {
    return run_append(k, k_b_stride, k_g_stride, k_t_stride, v, v_b_stride, v_g_stride, v_t_stride, dtype, k_codes, v_codes,
                      k_exp, v_exp, starts, start, B, G, T, C, block, nullptr, nullptr, 0, stream);
}

extern "C" int attnlab_quant_append_kept(const uint16_t* k, int64_t k_b_stride, int64_t k_g_stride, int64_t k_t_stride,
                                         const uint16_t* v, int64_t v_b_stride, int64_t v_g_stride, int64_t v_t_stride,
                                         uint8_t* k_codes, uint8_t* v_codes, uint8_t* k_exp, uint8_t* v_exp, int start,
                                         int B, int G, int T, int C, int block, uint16_t* k_keep, uint16_t* v_keep,
                                         int keep_rows, void* stream) {
    ATTNLAB_REQUIRE(keep_rows >= 1 && k_keep && v_keep && aligned(k_keep, 16) && aligned(v_keep, 16),
                    "the kept rows (%d) must be 16-byte aligned device buffers of at least one row", keep_rows);
    return run_append(k, k_b_stride, k_g_stride, k_t_stride, v, v_b_stride, v_g_stride, v_t_stride, ATTNLAB_DT_BF16, k_codes,
                      v_codes, k_exp, v_exp, nullptr, start, B, G, T, C, block, k_keep, v_keep, keep_rows, stream);
}

extern "C" int attnlab_quant_read(const uint8_t* k_codes, const uint8_t* v_codes, const uint8_t* k_exp,
                                  const uint8_t* v_exp, void* k_out, void* v_out, int dtype, const int32_t* starts,
                                  int start, int B, int G, int T, int C, int block, void* stream) {
    const int rc = check_quant_cache(k_codes, v_codes, k_exp, v_exp, B, G, C, block);
    if (rc) return rc;
    ATTNLAB_REQUIRE(dtype == ATTNLAB_DT_BF16 || dtype == ATTNLAB_DT_F16 || dtype == ATTNLAB_DT_F32,
                    "rows are read back as bf16, fp16 or fp32 (dtype %d)", dtype);
    ATTNLAB_REQUIRE(T >= 0, "T=%d must not be negative", T);
    ATTNLAB_REQUIRE(starts != nullptr || (start >= 0 && (int64_t)start + T <= C), "rows [%d, %lld) outside the cache of "
                    "C=%d", start, (long long)start + T, C);
    if (T == 0) return ATTNLAB_OK;
    ATTNLAB_REQUIRE(k_out && v_out && aligned(k_out, 16) && aligned(v_out, 16),
                    "k_out and v_out must be 16-byte aligned device pointers");
    ReadArgs a{{k_codes, v_codes}, {k_exp, v_exp}, {k_out, v_out}, starts, start, G, T, C, block_shift(block),
               (C + block - 1) / block, (T + kReadRows - 1) / kReadRows};
    const int64_t blocks = 2 * (int64_t)B * G * a.tiles;
    ATTNLAB_REQUIRE(blocks < (int64_t)1 << 31, "grid of %lld workgroups is too large", (long long)blocks);
    const dim3 grid((unsigned)blocks), wg(256);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (dtype == ATTNLAB_DT_BF16) hipLaunchKernelGGL(quant_read<ATTNLAB_DT_BF16>, grid, wg, 0, s, a);
    else if (dtype == ATTNLAB_DT_F16) hipLaunchKernelGGL(quant_read<ATTNLAB_DT_F16>, grid, wg, 0, s, a);
    else hipLaunchKernelGGL(quant_read<ATTNLAB_DT_F32>, grid, wg, 0, s, a);
    return check_launch("quant_read");
}
