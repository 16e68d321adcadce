// Log probabilities of given tokens, the entropy and the most likely alternatives, of rows of logits x[0 .. V):
//   lse = m + log sum_j e^(x_j - m)      logprob = x_token - lse      H = log l - sum_j e^(x_j - m) (x_j - m) / l,  l = e^(lse - m)
//   top: the k largest x, equal ones by the lower token (NaN last, -0 equal to +0), as logprobs
//
// A row is cut into up to 64 segments, a workgroup each. A thread holds up to 64 logits in registers, so each is read once:
// its own maximum m, l and s = sum p (x - m) come from them, merge over the wave and the workgroup, and leave as a partial
// (m, l, s). A second launch merges a row's partials. Sums are fp32 in the log2 domain.
//
// The top k without a second look at the memory: the k-th largest of a wave's 64 thread maxima is a lower bound of the k-th
// largest logit, found by a search over the order-preserving key's bits with one ballot a bit; the largest of the four waves'
// bounds is the workgroup's. What lies above it (k and few more, in any distribution that does not crowd its largest logits into
// a few threads) goes to LDS, of those that equal it the first k of each wave, and is ranked there by counting. More than LDS
// takes: k rounds of a maximum over the workgroup, with the same result. The second launch does the same to the segments' lists.
//
// What bounds it: the bytes for float32, for 16-bit logits as much the vector units (9 operations for two bytes, of them an
// exponential at a quarter of the rate).
#include <cfloat>

#include "select.h"

namespace attnlab {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxTop = 64;
constexpr int kMaxSegments = 64;
constexpr int kCandidates = 1024;        // what a segment's workgroup ranks in LDS
constexpr int kPartWords = 4;            // m, l, s and the largest logit (16 bytes)
// x log2 e - m cancels what m's rounding left, up to where that is no longer small. A row whose largest logit is past kFar is
// summed again by differences; a thread whose own is below -2 kFar weighs nothing in any other row (e^-65536 is 0).
constexpr float kFar = 65536.0f;
constexpr float kLn2 = 0.69314718055994531f;

struct LogprobArgs {
    const void* x;                       // row r at x + r stride (elements)
    int64_t stride;
    int V, segments, words, top;         // words: 16-byte words of a segment
    float* part;                         // [N, segments, 4]
    uint64_t* best;                      // [N, segments, top] keys, largest first; 0 past a segment's last logit
    const void* tokens;                  // [N] int32 or int64, or null
    int tokens64;
    float* logprob;                      // [N]
    float* entropy;                      // [N] or null
    float* top_logprob;                  // [N, top]
    int64_t* top_token;                  // [N, top]
};

// Larger logit -> larger key, then lower token -> larger key. Never 0 for a token below 2^31.
__device__ __forceinline__ uint64_t key_of(float x, int token) {
    return (uint64_t)score_key(x) << 32 | (uint32_t)~token;
}
__device__ __forceinline__ float logit_of(uint32_t key) {   // of score_key's; NaN for 0
    return key == 0 ? __builtin_nanf("") : __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// The k-th largest of the wave's 64 keys (k <= 64): the largest t with k keys of at least t. The upper half of t by its bits,
// then the least key from there on.
__device__ __forceinline__ uint32_t wave_kth(uint32_t key, int k) {
    uint32_t t = 0;
#pragma unroll
    for (int bit = 31; bit >= 16; --bit) {
        const uint32_t with = t | 1u << bit;
        if (__popcll(__ballot(key >= with)) >= k) t = with;
    }
    uint32_t least = key >= t ? key : 0xffffffffu;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) least = min(least, (uint32_t)__shfl_xor((int)least, d, 64));
    return least;
}

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) x = fmaxf(x, shfl_xor_f32(x, d));
    return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) x += shfl_xor_f32(x, d);
    return x;
}

// (m, l, s) against a common maximum mt; m = -inf: nothing but, where they were NaN, its l and s.
__device__ __forceinline__ void rescale(float m, float mt, float& l, float& s) {
    if (m == -INFINITY) return;
    const float d = m - mt, w = fast_exp2(d);     // mt = inf: w is 0, or NaN where m is infinite too
    s = w == 0.0f && l == l ? 0.0f : w * (s + l * d);
    l *= w;
}

// One 16-byte word of a row as floats.
template <int DT>
__device__ __forceinline__ void unpack(u32x4_t w, float* v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == ATTNLAB_DT_F32) {
            v[i] = __uint_as_float(w[i]);
        } else if constexpr (DT == ATTNLAB_DT_BF16) {
            v[2 * i] = bf16_lo(w[i]);
            v[2 * i + 1] = bf16_hi(w[i]);
        } else {
            v[2 * i] = f16_to_f32((uint16_t)w[i]);
            v[2 * i + 1] = f16_to_f32((uint16_t)(w[i] >> 16));
        }
    }
}

// `count` keys in `sh` ranked by counting the larger ones; the first `top` of them to `take(rank, key)`.
template <typename Take>
__device__ __forceinline__ void rank_keys(const uint64_t* sh, int count, int top, Take take) {
    for (int i = threadIdx.x; i < count; i += kThreads) {
        const uint64_t own = sh[i];
        int rank = 0;
        for (int j = 0; j < count; ++j) rank += sh[j] > own;
        if (rank < top) take(rank, own);
    }
}

template <int DT, int U>
__global__ __launch_bounds__(kThreads) void logprob_segment(LogprobArgs a) {
    constexpr int kPer = DT == ATTNLAB_DT_F32 ? 4 : 8, kBytes = 16 / kPer;
    __shared__ uint64_t cand_sh[kCandidates];
    __shared__ float part_sh[kWaves][4];
    __shared__ uint32_t bound_sh[kWaves];
    __shared__ uint32_t count_sh;
    const int seg = blockIdx.x % a.segments;
    const int64_t row = blockIdx.x / a.segments;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // the row in aligned words: word w holds tokens kPer w - head .. (an aligned word with a byte of the row lies in its memory)
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.x) + (uintptr_t)row * a.stride * kBytes;
    const int head = (int)(at & 15) / kBytes;
    const u32x4_t* words = reinterpret_cast<const u32x4_t*>(at & ~(uintptr_t)15);
    const int first = seg * a.words, end = min(first + a.words, (head + a.V + kPer - 1) / kPer);
    u32x4_t raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int w = first + kThreads * u + tid;
        if (w < end) raw[u] = __builtin_nontemporal_load(words + w);
    }
    float x[U][kPer];
    bool whole = true;                   // every element of this thread is a logit
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int w = first + kThreads * u + tid, t = kPer * w - head;
        if (w < end) unpack<DT>(raw[u], x[u]);
        const bool in = w < end && t >= 0 && t + kPer <= a.V;
        if (!in) {
            whole = false;
#pragma unroll
            for (int j = 0; j < kPer; ++j) x[u][j] = w < end && t + j >= 0 && t + j < a.V ? x[u][j] : -INFINITY;
        }
    }
    float m = x[0][0];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < kPer; ++j) m = fmaxf(m, x[u][j]);
    const float top = m;                 // NaN where all are
    m = m > -2.0f * kFar ? m * kLog2e : -INFINITY;
    float l = 0.0f, s = 0.0f;
    const float nm = m == -INFINITY ? 0.0f : -m;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const float d = fmaf(x[u][j], kLog2e, nm), p = fast_exp2(d);
            l += p;
            s = fmaf(p, d, s);
        }
    if (l == l && s != s) {              // some logit is -inf: a weight of zero, and no term
        s = 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                const float d = fmaxf(fmaf(x[u][j], kLog2e, nm), -1000.0f);
                s = fmaf(fast_exp2(d), d, s);
            }
    }
    const float mw = wave_max(m), largest = wave_max(top);
    rescale(m, mw, l, s);
    l = wave_sum(l);
    s = wave_sum(s);
    if (lane == 0) {
        part_sh[wave][0] = mw;
        part_sh[wave][1] = l;
        part_sh[wave][2] = s;
        part_sh[wave][3] = largest;
    }
    // a thread without logits of its own, or with nothing above -inf among elements that are none: no bound
    const uint32_t mine = !whole && !(top > -INFINITY) ? 0u : score_key(top);
    uint32_t bound = 0;
    if (a.top) {
        bound = wave_kth(mine, a.top);
        if (lane == 0) bound_sh[wave] = bound;
    }
    if (tid == 0) count_sh = 0;
    __syncthreads();
    if (tid == 0) {
        float ms = part_sh[0][0], ls = 0.0f, ss = 0.0f, xs = part_sh[0][3];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) {
            ms = fmaxf(ms, part_sh[w][0]);
            xs = fmaxf(xs, part_sh[w][3]);
        }
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            float lw = part_sh[w][1], sw = part_sh[w][2];
            rescale(part_sh[w][0], ms, lw, sw);
            ls += lw;
            ss += sw;
        }
        *reinterpret_cast<float4*>(a.part + (row * a.segments + seg) * kPartWords) = make_float4(ms, ls, ss, xs);
    }
    if (!a.top) return;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) bound = max(bound, bound_sh[w]);
    if (__any(mine >= bound || mine == 0)) {
        int equal = 0;                   // of this wave so far, in the order of their tokens
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int w = first + kThreads * u + tid, t = kPer * w - head;
            uint32_t own = 0;            // elements that equal the bound
            bool some = false;
#pragma unroll
            for (int j = 0; j < kPer; ++j) some |= !(x[u][j] < logit_of(bound));   // NaN too
            if (!__any(some)) continue;
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                const uint32_t k = score_key(x[u][j]);
                const bool in = w < end && t + j >= 0 && t + j < a.V;
                if (in && k > bound) {
                    const uint32_t i = atomicAdd(&count_sh, 1u);
                    if (i < kCandidates) cand_sh[i] = (uint64_t)k << 32 | (uint32_t)~(t + j);
                }
                own |= in && k == bound ? 1u << j : 0u;
            }
            if (equal < a.top && __any(own != 0)) {
                const uint32_t mine_here = (uint32_t)__popc(own);
                const uint32_t upto = wave_incl_scan(mine_here);
                int at_rank = equal + (int)(upto - mine_here);
                equal += __builtin_amdgcn_readlane((int)upto, 63);
#pragma unroll
                for (int j = 0; j < kPer; ++j)
                    if (own >> j & 1 && at_rank++ < a.top) {
                        const uint32_t i = atomicAdd(&count_sh, 1u);
                        if (i < kCandidates) cand_sh[i] = (uint64_t)bound << 32 | (uint32_t)~(t + j);
                    }
            }
        }
    }
    __syncthreads();
    const uint32_t count = count_sh;
    uint64_t* best = a.best + (row * a.segments + seg) * a.top;
    if (count <= kCandidates) {
        rank_keys(cand_sh, (int)count, a.top, [&](int r, uint64_t k) { best[r] = k; });
        for (int r = (int)count + tid; r < a.top; r += kThreads) best[r] = 0;
        return;
    }
    uint64_t last = ~0ull;               // the largest key below the last one taken, `top` times
    for (int r = 0; r < a.top; ++r) {
        uint64_t k = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int w = first + kThreads * u + tid, t = kPer * w - head;
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                const uint64_t y = key_of(x[u][j], t + j);
                if (w < end && t + j >= 0 && t + j < a.V && y < last && y > k) k = y;
            }
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint64_t y = (uint64_t)(uint32_t)__shfl_xor((int)(k >> 32), d, 64) << 32 | (uint32_t)__shfl_xor((int)(uint32_t)k, d, 64);
            k = y > k ? y : k;
        }
        __syncthreads();
        if (lane == 0) cand_sh[wave] = k;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) k = cand_sh[w] > k ? cand_sh[w] : k;
        if (tid == 0) best[r] = k;
        last = k;
    }
}

// A row's partials: lane s of every wave holds segment s.
template <int DT>
__global__ __launch_bounds__(kThreads) void logprob_merge(LogprobArgs a) {
    constexpr int kMost = kMaxSegments * kMaxTop, kHold = kMost / kThreads;
    __shared__ uint64_t cand_sh[kMost];
    __shared__ uint32_t bound_sh[kWaves];
    __shared__ float far_sh[kWaves][2];
    __shared__ uint32_t count_sh;
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    float4 p = make_float4(-INFINITY, 0.0f, 0.0f, -INFINITY);
    if (lane < a.segments) p = *reinterpret_cast<const float4*>(a.part + (row * a.segments + lane) * kPartWords);
    const float m = wave_max(p.x), largest = wave_max(p.w);
    rescale(p.x, m, p.y, p.z);
    float l = wave_sum(p.y), s = wave_sum(p.z);
    auto at = [&](int64_t t) -> float {
        if constexpr (DT == ATTNLAB_DT_F32) return static_cast<const float*>(a.x)[row * a.stride + t];
        const uint16_t w = static_cast<const uint16_t*>(a.x)[row * a.stride + t];
        return DT == ATTNLAB_DT_BF16 ? bf16_to_f32(w) : f16_to_f32(w);
    };
    // a row whose largest logit is far from 0 (one that a mask of the type's lowest value has covered whole)
    const bool far = fabsf(largest) >= kFar && fabsf(largest) < INFINITY;
    if (far) {
        l = s = 0.0f;
        for (int t = tid; t < a.V; t += kThreads) {
            const float d = (at(t) - largest) * kLog2e, e = fast_exp2(d);
            l += e;
            s += d < -1000.0f ? 0.0f : e * d;
        }
        l = wave_sum(l);
        s = wave_sum(s);
        if (lane == 0) {
            far_sh[wave][0] = l;
            far_sh[wave][1] = s;
        }
        __syncthreads();
        l = s = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            l += far_sh[w][0];
            s += far_sh[w][1];
        }
    }
    // no logit above -inf: no distribution
    const float log2l = largest > -INFINITY ? log2f(l) : __builtin_nanf("");
    // l is relative to m, largest log2 e rounded: what that rounding left goes back
    const float lnl = (log2l - (far ? 0.0f : fmaf(largest, kLog2e, -m))) * kLn2;
    auto logprob = [&](float x) { return (x - largest) - lnl; };
    if (tid == 0) {
        if (a.entropy) a.entropy[row] = (log2l - s / l) * kLn2;
        if (a.logprob) {
            const int64_t t = a.tokens64 ? static_cast<const int64_t*>(a.tokens)[row] : static_cast<const int32_t*>(a.tokens)[row];
            a.logprob[row] = t < 0 ? 0.0f : t < a.V ? logprob(at(t)) : __builtin_nanf("");
        }
    }
    if (!a.top) return;
    const int most = a.segments * a.top;
    const uint64_t* best = a.best + row * most;
    auto take = [&](int r, uint64_t k) {
        a.top_logprob[row * a.top + r] = logprob(logit_of((uint32_t)(k >> 32)));
        a.top_token[row * a.top + r] = (int64_t)(uint32_t)~(uint32_t)k;
    };
    uint64_t k[kHold];
    uint32_t mine = 0, bound = 0;
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
        k[i] = kThreads * i + tid < most ? best[kThreads * i + tid] : 0;
        mine = max(mine, (uint32_t)(k[i] >> 32));
    }
    bound = wave_kth(mine, a.top);
    if (lane == 0) bound_sh[wave] = bound;
    if (tid == 0) count_sh = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) bound = max(bound, bound_sh[w]);
#pragma unroll
    for (int i = 0; i < kHold; ++i)
        if (k[i] && (uint32_t)(k[i] >> 32) >= bound) cand_sh[atomicAdd(&count_sh, 1u)] = k[i];
    __syncthreads();
    rank_keys(cand_sh, (int)count_sh, a.top, take);
}

int per_word(int dtype) { return dtype == ATTNLAB_DT_F32 ? 4 : 8; }

// Words of a thread (1, 2, 4, 8, 16) and segments of a row: as many segments as give about two workgroups per CU, of 2048 logits
// or more and at most 64; a thread holds at most 64 logits.
int plan(int64_t N, int V, int dtype, int& segments, int& words) {
    const int per = per_word(dtype), total = (V + 2 * (per - 1)) / per;   // a row that begins inside a word has one more
    const int most = 64 / per;
    int u = 1;
    while (u < most && (N * ((total + kThreads * u - 1) / (kThreads * u)) >= 1024 ||
                        (total + kThreads * u - 1) / (kThreads * u) > kMaxSegments || kThreads * u * per < 2048))
        u *= 2;
    segments = (total + kThreads * u - 1) / (kThreads * u);
    words = (total + segments - 1) / segments;
    return u;
}

constexpr int kMaxVocab = 1 << 20;      // 64 segments of 16384 logits, one word of them lost to a row's alignment

template <int DT>
int launch(const LogprobArgs& a, int u, int64_t N, hipStream_t s) {
    const dim3 grid((unsigned)(N * a.segments)), wg(kThreads);
    if (u == 1) hipLaunchKernelGGL((logprob_segment<DT, 1>), grid, wg, 0, s, a);
    else if (u == 2) hipLaunchKernelGGL((logprob_segment<DT, 2>), grid, wg, 0, s, a);
    else if (u == 4) hipLaunchKernelGGL((logprob_segment<DT, 4>), grid, wg, 0, s, a);
    else if (u == 8) hipLaunchKernelGGL((logprob_segment<DT, 8>), grid, wg, 0, s, a);
    else if constexpr (DT == ATTNLAB_DT_F32) hipLaunchKernelGGL((logprob_segment<DT, 16>), grid, wg, 0, s, a);
    hipLaunchKernelGGL(logprob_merge<DT>, dim3((unsigned)N), wg, 0, s, a);
    return check_launch("token_logprobs");
}

}  // namespace
}  // namespace attnlab

using namespace attnlab;

extern "C" int64_t attnlab_logprob_part_bytes(int64_t N, int V, int dtype, int top) {
    if (N < 0 || V < 1 || V > kMaxVocab - 16 || dtype < ATTNLAB_DT_BF16 || dtype > ATTNLAB_DT_F32 || top < 0 || top > kMaxTop) return -1;
    int segments, words;
    plan(N, V, dtype, segments, words);
    return N * segments * (kPartWords * 4 + 8 * (int64_t)top);
}

extern "C" int attnlab_token_logprobs(const void* logits, int dtype, int64_t stride, int64_t N, int V, const void* tokens,
                                      int tokens64, int top, float* logprobs, float* entropy, float* top_logprobs,
                                      int64_t* top_tokens, void* part, int64_t part_bytes, void* stream) {
    ATTNLAB_REQUIRE(dtype == ATTNLAB_DT_BF16 || dtype == ATTNLAB_DT_F16 || dtype == ATTNLAB_DT_F32,
                    "logits must be bf16, fp16 or fp32 (dtype %d)", dtype);
    ATTNLAB_REQUIRE(N >= 0 && 1 <= V && V <= kMaxVocab - 16, "rows N=%lld must not be negative and V=%d be in [1, %d]", (long long)N, V,
                    kMaxVocab - 16);
    ATTNLAB_REQUIRE(0 <= top && top <= kMaxTop && top <= V, "top=%d outside [0, min(%d, V=%d)]", top, kMaxTop, V);
    ATTNLAB_REQUIRE((tokens == nullptr) == (logprobs == nullptr), "tokens and logprobs go together");
    ATTNLAB_REQUIRE(top == 0 || (top_logprobs && top_tokens), "top=%d needs top_logprobs and top_tokens", top);
    if (N == 0) return ATTNLAB_OK;
    ATTNLAB_REQUIRE(logits, "logits must be a device pointer");
    const int bytes = dtype == ATTNLAB_DT_F32 ? 4 : 2;
    ATTNLAB_REQUIRE(reinterpret_cast<uintptr_t>(logits) % bytes == 0, "logits must be aligned to their type");
    LogprobArgs a{logits, stride, V, 0, 0, top, static_cast<float*>(part), nullptr, tokens, tokens64, logprobs, entropy, top_logprobs,
                  top_tokens};
    const int u = plan(N, V, dtype, a.segments, a.words);
    ATTNLAB_REQUIRE(N * a.segments < (int64_t)1 << 31, "%lld rows of %d segments are too many", (long long)N, a.segments);
    const int64_t need = attnlab_logprob_part_bytes(N, V, dtype, top);
    ATTNLAB_REQUIRE(part && reinterpret_cast<uintptr_t>(part) % 16 == 0 && part_bytes >= need,
                    "part must be a 16-byte aligned device buffer of %lld bytes", (long long)need);
    a.best = reinterpret_cast<uint64_t*>(a.part + N * a.segments * kPartWords);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (dtype == ATTNLAB_DT_BF16) return launch<ATTNLAB_DT_BF16>(a, u, N, s);
    if (dtype == ATTNLAB_DT_F16) return launch<ATTNLAB_DT_F16>(a, u, N, s);
    return launch<ATTNLAB_DT_F32>(a, u, N, s);
}
