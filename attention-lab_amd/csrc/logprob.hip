// Log probabilities of given tokens, the entropy and the most likely alternatives, of rows of logits x[0 .. V):
//   lse = m + log sum_j e^(x_j - m)      logprob = x_token - lse      H = log l - sum_j e^(x_j - m) (x_j - m) / l,  l = e^(lse - m)
//   top: the k largest x, equal ones by the lower token (NaN last, -0 equal to +0), as logprobs
//
// A row is cut into up to 64 segments, a workgroup each. A thread holds up to 64 logits in registers, as they came, so each is read
// once: the waves sum l and s = sum p (x - m) relative to an m of their own, and a segment's leave as a partial (m, l, s,
// largest). The last of a row's workgroups to arrive merges its partials, where there are few rows; else a second launch does.
// Sums are fp32 in the log2 domain.
//
// The top k without a second look at every logit: the k-th largest of a wave's 64 thread maxima (or one near it) is a lower
// bound of the k-th largest logit, found by a search over the order-preserving key's bits with one ballot a bit; so are the
// largest of the four waves' bounds, and, nearer where the waves' logits are alike, the least of the waves' k / 4-th largest.
// The few 16-byte words that reach the bound (k and some more, in any distribution that does not crowd its largest logits into
// a few threads) go to LDS, and one wave looks them over again and ranks what it finds by counting. More words than that holds,
// which takes logits that are equal in their type: k rounds of a maximum over the workgroup, with the same result (64 bf16 rows
// of 30000 + N(0, 2.5), which are all the same, top 20: 150 us, of N(0, 2.5) 13). The merge does the same to the segments'
// lists.
//
// What bounds it, vocabulary of 151936. 4096 bf16 rows, top 5: 204 to 219 us, 1.24 GB at 5.7 to 6.1 TB/s (reads alone go at
// 7.1); as much as the bytes it is the vector units (11 operations a logit, half of them in the sums, an exponential among
// them). 64 float32 rows, top 20: 16 us, of which the 39 MB take 6 (all workgroups at once), the bounds 1, the lists 2.5,
// arrivals 1 and the merge 2.5: latencies.
#include <cfloat>

#include "select.h"

namespace attnlab {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxTop = 64;
constexpr int kMaxSegments = 64;
constexpr int kWords = 256;              // words of a segment that are looked over again
// Up to kFew, the k / 4-th largest of the waves are not asked for: few words reach the first bound anyway, and a second search
// costs more than it saves (4096 rows, top 5: 207 and 217 us; 64 rows, top 20: 18.0 without it and 16.2 with).
constexpr int kFew = 8;
constexpr int kPartWords = 4;            // m, l, s and the largest logit (16 bytes)
// x log2 e - m cancels what m's rounding left, up to where that is no longer small. A row whose largest logit is past kFar is
// summed again by differences; a thread whose own is below -2 kFar weighs nothing in any other row (e^-65536 is 0).
constexpr float kFar = 65536.0f;
constexpr float kNear = 16.0f;           // log2 of what a weight may be above 1: the entropy is off by some 2^-23 of it
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
    uint32_t* arrive;                    // [N] arrival counters, zero on entry and left zero: the last segment's workgroup of a
                                         // row to arrive merges it (segments * top <= kWaveKeys); null: a second launch does
};

// Larger logit -> larger key, then lower token -> larger key. Never 0 for a token below 2^31.
__device__ __forceinline__ uint64_t key_of(float x, int token) {
    return (uint64_t)score_key(x) << 32 | (uint32_t)~token;
}
__device__ __forceinline__ float logit_of(uint32_t key) {   // of score_key's; NaN for 0
    return key == 0 ? __builtin_nanf("") : __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// Over the wave's lanes: a scan along each row of 16, then the rows' ends; the last lane's value, for all.
template <int CTRL, int ROWS>
__device__ __forceinline__ float moved(float x, float none) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(none), __float_as_int(x), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float last_lane(float x) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63)); }
__device__ __forceinline__ float wave_max(float x) {   // NaN where all are
    x = fmaxf(x, moved<0x111, 0xf>(x, x));
    x = fmaxf(x, moved<0x112, 0xf>(x, x));
    x = fmaxf(x, moved<0x114, 0xf>(x, x));
    x = fmaxf(x, moved<0x118, 0xf>(x, x));
    x = fmaxf(x, moved<0x142, 0xa>(x, x));
    x = fmaxf(x, moved<0x143, 0xc>(x, x));
    return last_lane(x);
}
__device__ __forceinline__ float wave_sum(float x) {
    x += moved<0x111, 0xf>(x, 0.0f);
    x += moved<0x112, 0xf>(x, 0.0f);
    x += moved<0x114, 0xf>(x, 0.0f);
    x += moved<0x118, 0xf>(x, 0.0f);
    x += moved<0x142, 0xa>(x, 0.0f);
    x += moved<0x143, 0xc>(x, 0.0f);
    return last_lane(x);
}

__device__ __forceinline__ uint32_t wave_min(uint32_t x) {
    auto with = [&](float y) { x = min(x, (uint32_t)__float_as_int(y)); };
    auto own = [&]() { return __uint_as_float(x); };
    with(moved<0x111, 0xf>(own(), own()));
    with(moved<0x112, 0xf>(own(), own()));
    with(moved<0x114, 0xf>(own(), own()));
    with(moved<0x118, 0xf>(own(), own()));
    with(moved<0x142, 0xa>(own(), own()));
    with(moved<0x143, 0xc>(own(), own()));
    return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}
// This lane's place among those of `hit`.
__device__ __forceinline__ uint32_t before_me(uint64_t hit) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(hit >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)hit, 0));
}

// A key that k of the wave's 64 keys reach, and few more (k <= 64): the upper half of the largest such bound by its bits, then
// the least key from there on. A bf16 logit's key has no more bits, so that is the k-th largest. Another's upper half is a
// range of 2^-7 of its size, where logits far from 0 (or with a common part, which changes no probability) lie together: the
// other bits follow where the range holds more than kClose keys too many. 64 float32 rows of 1000 + N(0, 2.5), top 20: 15.5 us,
// without them 172; of N(0, 2.5) 14.8 and 14.7.
constexpr int kClose = 8;
template <int DT>
__device__ __forceinline__ uint32_t wave_kth(uint32_t key, int k) {
    uint32_t t = 0;
    int reach = 64;
    auto search = [&](int bit) {
        const uint32_t with = t | 1u << bit;
        const int n = __popcll(__ballot(key >= with));
        if (n >= k) {
            t = with;
            reach = n;
        }
    };
#pragma unroll
    for (int bit = 31; bit >= 16; --bit) search(bit);
    constexpr int kLast = DT == ATTNLAB_DT_F32 ? 0 : DT == ATTNLAB_DT_F16 ? 13 : 16;   // the last bit that is not the same in all
    if (kLast < 16 && reach > k + kClose)
        for (int bit = 15; bit >= kLast; --bit) search(bit);
    return wave_min(key >= t ? key : 0xffffffffu);
}

// (m, l, s) against a common maximum mt; m = -inf: nothing but, where they were NaN, its l and s.
__device__ __forceinline__ void rescale(float m, float mt, float& l, float& s) {
    if (m == -INFINITY) return;
    const float d = m - mt, w = fast_exp2(d);     // mt = inf: w is 0, or NaN where m is infinite too
    s = w == 0.0f && l == l ? 0.0f : w * (s + l * d);
    l *= w;
}

// Element j of a 16-byte word of a row as a float.
template <int DT>
__device__ __forceinline__ float element(const u32x4_t& w, int j) {
    if constexpr (DT == ATTNLAB_DT_F32) return __uint_as_float(w[j]);
    else if constexpr (DT == ATTNLAB_DT_BF16) return j & 1 ? bf16_hi(w[j >> 1]) : bf16_lo(w[j >> 1]);
    else return f16_to_f32((uint16_t)(w[j >> 1] >> (16 * (j & 1))));
}
// The word's elements outside [0, V) as -inf; t: the first one's token.
template <int DT>
__device__ __forceinline__ void only_logits(u32x4_t& w, int t, int V) {
    constexpr uint32_t kNone = DT == ATTNLAB_DT_F32 ? 0xff800000u : DT == ATTNLAB_DT_BF16 ? 0xff80u : 0xfc00u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == ATTNLAB_DT_F32) {
            if (t + i < 0 || t + i >= V) w[i] = kNone;
        } else {
            if (t + 2 * i < 0 || t + 2 * i >= V) w[i] = (w[i] & 0xffff0000u) | kNone;
            if (t + 2 * i + 1 < 0 || t + 2 * i + 1 >= V) w[i] = (w[i] & 0xffffu) | kNone << 16;
        }
    }
}

// `count` keys in `sh` ranked by counting the larger ones; the first `top` of them to `take(rank, key)`. Eight at a time:
// zeros, which are larger than none, fill the last ones up (`sync`: they are there for all).
constexpr int kAtOnce = 8;
template <int THREADS, typename Sync, typename Take>
__device__ __forceinline__ void rank_keys(uint64_t* sh, int count, int top, Sync sync, Take take) {
    const int tid = threadIdx.x & (THREADS - 1), padded = (count + kAtOnce - 1) / kAtOnce * kAtOnce;
    if (count + tid < padded) sh[count + tid] = 0;
    sync();
    for (int i = tid; i < count; i += THREADS) {
        const uint64_t own = sh[i];
        int rank = 0;
        for (int j = 0; j < padded; j += kAtOnce) {
            ulonglong2 k[kAtOnce / 2];
#pragma unroll
            for (int u = 0; u < kAtOnce / 2; ++u) k[u] = *reinterpret_cast<const ulonglong2*>(sh + j + 2 * u);
#pragma unroll
            for (int u = 0; u < kAtOnce / 2; ++u) rank += (k[u].x > own) + (k[u].y > own);
        }
        if (rank < top) take(rank, own);
    }
}

// What threads of a merge exchange.
struct MergeShared {
    uint32_t bound[kWaves], count;
    float far[kWaves][2];
};
constexpr int kWaveKeys = 256;

// A row's partials merged by THREADS threads (a wave, or the workgroup): lane s of every wave holds segment s. COHERENT: written by
// workgroups of this launch, read past the caches of this XCD. cand: room for the segments' keys.
template <int DT, int THREADS, bool COHERENT>
__device__ __forceinline__ void merge_row(const LogprobArgs& a, int64_t row, uint64_t* cand, MergeShared& sh) {
    constexpr int kMost = THREADS == 64 ? kWaveKeys : kMaxSegments * kMaxTop, kHold = kMost / THREADS;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tid = THREADS == 64 ? lane : (int)threadIdx.x;
    auto sync = [&]() {   // a wave's LDS operations take effect in order
        if constexpr (THREADS == 64) asm volatile("" ::: "memory");
        else __syncthreads();
    };
    const float* part = a.part + row * a.segments * kPartWords;
    const int most = a.segments * a.top;
    const uint64_t* best = a.best + row * most;
    int64_t token = -1;                      // on its way first, and its logit behind the partials
    if (tid == 0 && a.logprob)
        token = a.tokens64 ? static_cast<const int64_t*>(a.tokens)[row] : static_cast<const int32_t*>(a.tokens)[row];
    float4 p = make_float4(-INFINITY, 0.0f, 0.0f, -INFINITY);
    if (lane < a.segments) {
        if constexpr (COHERENT) {
            const float* q = part + lane * kPartWords;
            p = make_float4(load_coherent(q), load_coherent(q + 1), load_coherent(q + 2), load_coherent(q + 3));
        } else {
            p = *reinterpret_cast<const float4*>(part + lane * kPartWords);
        }
    }
    uint64_t k[kHold];
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
        k[i] = 0;
        if (THREADS * i + tid < most) {
            const uint64_t* q = best + THREADS * i + tid;
            k[i] = COHERENT ? __hip_atomic_load(q, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM) : *q;
        }
    }
    auto at = [&](int64_t t) -> float {
        if constexpr (DT == ATTNLAB_DT_F32) return static_cast<const float*>(a.x)[row * a.stride + t];
        const uint16_t w = static_cast<const uint16_t*>(a.x)[row * a.stride + t];
        return DT == ATTNLAB_DT_BF16 ? bf16_to_f32(w) : f16_to_f32(w);
    };
    const float given = token >= 0 && token < a.V ? at(token) : __builtin_nanf("");
    const float m = wave_max(p.x), largest = wave_max(p.w);
    rescale(p.x, m, p.y, p.z);
    float l = wave_sum(p.y), s = wave_sum(p.z);
    // a row whose largest logit is far from 0 (one that a mask of the type's lowest value has covered whole)
    const bool far = fabsf(largest) >= kFar && fabsf(largest) < INFINITY;
    if (far) {
        l = s = 0.0f;
        for (int t = tid; t < a.V; t += THREADS) {
            const float d = (at(t) - largest) * kLog2e, e = fast_exp2(d);
            l += e;
            s += d < -1000.0f ? 0.0f : e * d;
        }
        l = wave_sum(l);
        s = wave_sum(s);
        if constexpr (THREADS > 64) {
            if (lane == 0) {
                sh.far[wave][0] = l;
                sh.far[wave][1] = s;
            }
            __syncthreads();
            l = s = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                l += sh.far[w][0];
                s += sh.far[w][1];
            }
        }
    }
    // no logit above -inf: no distribution
    const float log2l = largest > -INFINITY ? log2f(l) : __builtin_nanf("");
    // l is relative to m, not the largest logit
    const float lnl = (log2l - (far ? 0.0f : fmaf(largest, kLog2e, -m))) * kLn2;
    auto logprob = [&](float x) { return (x - largest) - lnl; };
    if (tid == 0) {
        if (a.entropy) a.entropy[row] = (log2l - s / l) * kLn2;
        if (a.logprob) a.logprob[row] = token < 0 ? 0.0f : logprob(given);   // NaN past the last token
        sh.count = 0;
    }
    if (!a.top) return;
#pragma unroll
    for (int i = 0; i < kHold; ++i) mine = max(mine, (uint32_t)(k[i] >> 32));
    uint32_t bound = wave_kth<DT>(mine, a.top);
    if constexpr (THREADS > 64) {
        if (lane == 0) sh.bound[wave] = bound;
    }
    sync();
    if constexpr (THREADS > 64) {
#pragma unroll
        for (int w = 0; w < kWaves; ++w) bound = max(bound, sh.bound[w]);
    }
    uint32_t count = 0;
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
        const bool in = k[i] && (uint32_t)(k[i] >> 32) >= bound;
        const uint64_t hit = __ballot(in);
        if (!hit) continue;
        uint32_t first = count;
        if constexpr (THREADS == 64) {
            count += (uint32_t)__popcll(hit);
        } else {
            if (lane == 0) first = atomicAdd(&sh.count, (uint32_t)__popcll(hit));
            first = (uint32_t)__builtin_amdgcn_readfirstlane((int)first);
        }
        if (in) cand[first + before_me(hit)] = k[i];
    }
    if constexpr (THREADS > 64) {
        __syncthreads();
        count = sh.count;
    }
    rank_keys<THREADS>(cand, (int)count, a.top, sync, [&](int i, uint64_t y) {
        a.top_logprob[row * a.top + i] = logprob(logit_of((uint32_t)(y >> 32)));
        a.top_token[row * a.top + i] = (int64_t)(uint32_t)~(uint32_t)y;
    });
}

template <int DT, int U, bool MERGE>
__global__ __launch_bounds__(kThreads) void logprob_segment(LogprobArgs a) {
    constexpr int kPer = DT == ATTNLAB_DT_F32 ? 4 : 8, kBytes = 16 / kPer;
    __shared__ __attribute__((aligned(16))) uint64_t cand_sh[kWords * kPer];
    __shared__ uint16_t word_sh[kWords];
    __shared__ u32x4_t data_sh[kWords];
    __shared__ float part_sh[kWaves][4];
    __shared__ uint2 bound_sh[kWaves];
    __shared__ uint32_t words_sh, last_sh;
    __shared__ MergeShared merge_sh;
    const int seg = blockIdx.x % a.segments;
    const int64_t row = blockIdx.x / a.segments;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // the row in aligned words: word w holds tokens kPer w - head .. (an aligned word with a byte of the row lies in its memory)
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.x) + (uintptr_t)row * a.stride * kBytes;
    const int head = (int)(at & 15) / kBytes;
    const u32x4_t* words = reinterpret_cast<const u32x4_t*>(at & ~(uintptr_t)15);
    const int row_words = (head + a.V + kPer - 1) / kPer;   // the last segment can begin behind them
    const int first = seg * a.words, end = min(first + a.words, row_words);
    // the wave's word u: 64 in line, a segment's end between waves (but for the row's end)
    auto there = [&](int u) { return first + kThreads * u + 64 * wave < end; };
    u32x4_t x[U];
    {   // as a buffer that ends with the segment: zeros behind it. All of the offset is the vector one: a scalar offset need
        // not count where it is compared with the end
        constexpr int kNt = 2;   // non-temporal
        const __amdgpu_buffer_rsrc_t r =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<u32x4_t*>(words + first), 0, 16 * max(end - first, 0), 0x00020000);
#pragma unroll
        for (int u = 0; u < U; ++u)
            x[u] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(r, 16 * tid + 16 * kThreads * u, 0, kNt));
    }
    if (tid == 0) words_sh = 0;
    // -inf for what is not the row's, in its first and last word and behind it (the waves behind a segment's end between waves skip
    // their words); `whole`: every element of this thread is a logit
    bool whole = first + kThreads * (U - 1) + tid < end;
    if (seg == 0 || first + a.words >= row_words) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int t = kPer * (first + kThreads * u + tid) - head;
            if (t < 0 || t + kPer > a.V) {
                only_logits<DT>(x[u], t, a.V);
                whole = false;
            }
        }
    }
    auto word_max = [&](const u32x4_t& w) {   // NaN where all are
        float y = element<DT>(w, 0);
#pragma unroll
        for (int j = 1; j < kPer; ++j) y = fmaxf(y, element<DT>(w, j));
        return y;
    };
    // One pass: each word's maximum, and the sums relative to the largest of the wave's first words, near enough to the largest of
    // all, as soon as a word is there.
    float m = wave_max(word_max(x[0]));
    bool near = there(0) && m > -2.0f * kFar && m < INFINITY;
    m *= kLog2e;
    float most[U], l = 0.0f, s = 0.0f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        most[u] = -INFINITY;
        if (!there(u)) continue;
        most[u] = word_max(x[u]);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const float d = fmaf(element<DT>(x[u], j), kLog2e, -m), p = fast_exp2(d);
            l += p;
            s = fmaf(p, d, s);
        }
    }
    float top = most[0];
#pragma unroll
    for (int u = 1; u < U; ++u) top = fmaxf(top, most[u]);
    const float largest = wave_max(top);
    // Not near enough (the sum's logarithm and the entropy's quotient would cancel), or some logit is -inf (a weight of zero,
    // and no term), or none is a number: again, by the wave's own maximum
    near = near && fmaf(top, kLog2e, -m) <= kNear && l < FLT_MAX && fabsf(s) < FLT_MAX;
    if (!__all(near)) {
        m = largest > -2.0f * kFar ? largest * kLog2e : -INFINITY;
        const float nm = m == -INFINITY ? 0.0f : -m;
        l = s = 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!there(u)) continue;
            asm volatile("" : "+v"(x[u].x), "+v"(x[u].y), "+v"(x[u].z), "+v"(x[u].w));   // unpacked again, not kept
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                const float d = fmaf(element<DT>(x[u], j), kLog2e, nm), p = fast_exp2(d);
                l += p;
                s = fmaf(p, fmaxf(d, -1000.0f), s);
            }
        }
    }
    l = wave_sum(l);
    s = wave_sum(s);
    if (lane == 0) {
        part_sh[wave][0] = m;
        part_sh[wave][1] = l;
        part_sh[wave][2] = s;
        part_sh[wave][3] = largest;
    }
    // a thread with nothing above -inf among elements that are no logits: no bound
    if (a.top) {
        const uint32_t key = !whole && !(top > -INFINITY) ? 0u : score_key(top);
        const uint32_t all = wave_kth<DT>(key, a.top), part = a.top > kFew ? wave_kth<DT>(key, (a.top + kWaves - 1) / kWaves) : 0u;
        if (lane == 0) bound_sh[wave] = make_uint2(all, part);
    }
    __syncthreads();
    if (tid == kThreads - 1) {
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
        float* part = a.part + (row * a.segments + seg) * kPartWords;
        if constexpr (MERGE) {           // written through to memory, so the merging workgroup reads them on any XCD
            store_coherent(part, ms);
            store_coherent(part + 1, ls);
            store_coherent(part + 2, ss);
            store_coherent(part + 3, xs);
        } else {
            *reinterpret_cast<float4*>(part) = make_float4(ms, ls, ss, xs);
        }
    }
    if (a.top) {
        // k of one wave's logits reach its k-th largest maximum, and k / 4 of each wave's the least of the k / 4-th largest
        uint32_t bound = bound_sh[0].y;
#pragma unroll
        for (int w = 1; w < kWaves; ++w) bound = min(bound, bound_sh[w].y);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) bound = max(bound, bound_sh[w].x);
        const float least = logit_of(bound);   // NaN: every word
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool reaches = !(most[u] < least) && first + kThreads * u + tid < end;
            if (reaches) {
                const uint32_t i = atomicAdd(&words_sh, 1u);
                if (i < kWords) {
                    word_sh[i] = (uint16_t)(kThreads * u + tid);
                    data_sh[i] = x[u];
                }
            }
        }
        __syncthreads();
        const uint32_t listed = words_sh;
        uint64_t* best = a.best + (row * a.segments + seg) * a.top;
        auto take = [&](int r, uint64_t k) {
            if constexpr (MERGE) __hip_atomic_store(best + r, k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
            else best[r] = k;
        };
        if (listed <= kWords) {
            if (wave == 0) {
                int count = 0;
                for (uint32_t i0 = 0; i0 < listed; i0 += 64) {
                    const uint32_t i = min(i0 + lane, listed - 1);
                    const int t = i0 + lane < listed ? kPer * (first + word_sh[i]) - head : a.V;   // past the last: no logits
                    const u32x4_t v = data_sh[i];
#pragma unroll
                    for (int j = 0; j < kPer; ++j) {
                        const uint32_t k = score_key(element<DT>(v, j));
                        const bool in = k >= bound && t + j >= 0 && t + j < a.V;
                        const uint64_t found = __ballot(in);
                        if (in) cand_sh[count + before_me(found)] = (uint64_t)k << 32 | (uint32_t)~(t + j);
                        count += __popcll(found);
                    }
                }
                // a wave's LDS operations take effect in order
                rank_keys<64>(cand_sh, count, a.top, [] { asm volatile("" ::: "memory"); }, take);
                for (int r = count + lane; r < a.top; r += 64) take(r, 0);
            }
        } else {
            uint64_t last = ~0ull;           // the largest key below the last one taken, `top` times
            for (int r = 0; r < a.top; ++r) {
                uint64_t k = 0;
                for (int w = first + tid; w < end; w += kThreads) {
                    const int t = kPer * w - head;
                    const u32x4_t v = words[w];
#pragma unroll
                    for (int j = 0; j < kPer; ++j) {
                        const uint64_t y = key_of(element<DT>(v, j), t + j);
                        if (t + j >= 0 && t + j < a.V && y < last && y > k) k = y;
                    }
                }
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) {
                    const uint64_t y = (uint64_t)(uint32_t)__shfl_xor((int)(k >> 32), d, 64) << 32 |
                                       (uint32_t)__shfl_xor((int)(uint32_t)k, d, 64);
                    k = y > k ? y : k;
                }
                __syncthreads();
                if (lane == 0) cand_sh[wave] = k;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < kWaves; ++w) k = cand_sh[w] > k ? cand_sh[w] : k;
                if (tid == 0) take(r, k);
                last = k;
            }
        }
    }
    if constexpr (MERGE) {
        // Every store of this workgroup has completed before its count (the wait and the barrier), so the one that counts all
        // others before itself finds every partial in memory. It leaves the counter zero.
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (tid == 0)
            last_sh = __hip_atomic_fetch_add(a.arrive + row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                      (uint32_t)(a.segments - 1);
        __syncthreads();
        if (!last_sh || wave != 0) return;
        static_assert(kWords * kPer >= kWaveKeys, "the merge's keys lie in the segment's");
        merge_row<DT, 64, true>(a, row, cand_sh, merge_sh);
        if (lane == 0) __hip_atomic_store(a.arrive + row, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}

// The rows' partials in a launch of their own: a wave a row where the segments' lists hold kWaveKeys keys or fewer, else a
// workgroup.
template <int DT, int THREADS>
__global__ __launch_bounds__(kThreads) void logprob_merge(LogprobArgs a, int64_t N) {
    constexpr int kRows = kThreads / THREADS;
    __shared__ __attribute__((aligned(16))) uint64_t cand_sh[kRows][THREADS == 64 ? kWaveKeys : kMaxSegments * kMaxTop];
    __shared__ MergeShared sh[kRows];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = THREADS == 64 ? wave : 0;
    const int64_t row = (int64_t)blockIdx.x * kRows + r;
    if (row < N) merge_row<DT, THREADS, false>(a, row, cand_sh[r], sh[r]);
}

int per_word(int dtype) { return dtype == ATTNLAB_DT_F32 ? 4 : 8; }

// Words of a thread (1, 2, 4, 8, 16) and segments of a row: as many segments as give about two workgroups per CU, of 2048 logits
// or more and at most 64.
int plan(int64_t N, int V, int dtype, int& segments, int& words) {
    const int per = per_word(dtype), total = (V + 2 * (per - 1)) / per;   // a row that begins inside a word has one more
    // 64 logits; 16-bit ones of 4, 8 and 16 words: 260, 218, 220 us (4096 rows)
    const int most = dtype == ATTNLAB_DT_F32 ? 16 : 8;
    int u = 1;
    while (u < most && (N * ((total + kThreads * u - 1) / (kThreads * u)) >= 1024 ||
                        (total + kThreads * u - 1) / (kThreads * u) > kMaxSegments || kThreads * u * per < 2048))
        u *= 2;
    segments = (total + kThreads * u - 1) / (kThreads * u);
    words = ((total + segments - 1) / segments + 63) / 64 * 64;   // whole waves of them
    segments = (total + words - 1) / words;
    return u;
}

constexpr int kMaxVocab = 1 << 20;      // 64 segments of 16384 logits, one word of them lost to a row's alignment

template <int DT, bool MERGE>
void launch_segments(const LogprobArgs& a, int u, int64_t N, hipStream_t s) {
    const dim3 grid((unsigned)(N * a.segments)), wg(kThreads);
    if (u == 1) hipLaunchKernelGGL((logprob_segment<DT, 1, MERGE>), grid, wg, 0, s, a);
    else if (u == 2) hipLaunchKernelGGL((logprob_segment<DT, 2, MERGE>), grid, wg, 0, s, a);
    else if (u == 4) hipLaunchKernelGGL((logprob_segment<DT, 4, MERGE>), grid, wg, 0, s, a);
    else if (u == 8 || DT != ATTNLAB_DT_F32) hipLaunchKernelGGL((logprob_segment<DT, 8, MERGE>), grid, wg, 0, s, a);
    else if constexpr (DT == ATTNLAB_DT_F32) hipLaunchKernelGGL((logprob_segment<DT, 16, MERGE>), grid, wg, 0, s, a);
}

template <int DT>
int launch(const LogprobArgs& a, int u, int64_t N, hipStream_t s) {
    if (a.arrive) {
        launch_segments<DT, true>(a, u, N, s);
        return check_launch("token_logprobs");
    }
    launch_segments<DT, false>(a, u, N, s);
    const dim3 wg(kThreads);
    if (a.segments * a.top <= kWaveKeys) hipLaunchKernelGGL((logprob_merge<DT, 64>), dim3((unsigned)((N + 3) / 4)), wg, 0, s, a, N);
    else hipLaunchKernelGGL((logprob_merge<DT, kThreads>), dim3((unsigned)N), wg, 0, s, a, N);
    return check_launch("token_logprobs");
}

}  // namespace
}  // namespace attnlab

using namespace attnlab;

extern "C" int64_t attnlab_logprob_part_bytes(int64_t N, int V, int dtype, int top) {
    if (N < 0 || V < 1 || V > kMaxVocab - 16 || dtype < ATTNLAB_DT_BF16 || dtype > ATTNLAB_DT_F32 || top < 0 || top > kMaxTop)
        return -1;
    int segments, words;
    plan(N, V, dtype, segments, words);
    return N * segments * (kPartWords * 4 + 8 * (int64_t)top);
}

extern "C" int attnlab_token_logprobs(const void* logits, int dtype, int64_t stride, int64_t N, int V, const void* tokens,
                                      int tokens64, int top, float* logprobs, float* entropy, float* top_logprobs,
                                      int64_t* top_tokens, void* part, int64_t part_bytes, uint32_t* arrive, void* stream) {
    ATTNLAB_REQUIRE(dtype == ATTNLAB_DT_BF16 || dtype == ATTNLAB_DT_F16 || dtype == ATTNLAB_DT_F32,
                    "logits must be bf16, fp16 or fp32 (dtype %d)", dtype);
    ATTNLAB_REQUIRE(N >= 0 && 1 <= V && V <= kMaxVocab - 16, "rows N=%lld must not be negative and V=%d be in [1, %d]",
                    (long long)N, V, kMaxVocab - 16);
    ATTNLAB_REQUIRE(0 <= top && top <= kMaxTop && top <= V, "top=%d outside [0, min(%d, V=%d)]", top, kMaxTop, V);
    ATTNLAB_REQUIRE((tokens == nullptr) == (logprobs == nullptr), "tokens and logprobs go together");
    ATTNLAB_REQUIRE(top == 0 || (top_logprobs && top_tokens), "top=%d needs top_logprobs and top_tokens", top);
    if (N == 0) return ATTNLAB_OK;
    ATTNLAB_REQUIRE(logits, "logits must be a device pointer");
    const int bytes = dtype == ATTNLAB_DT_F32 ? 4 : 2;
    ATTNLAB_REQUIRE(reinterpret_cast<uintptr_t>(logits) % bytes == 0, "logits must be aligned to their type");
    LogprobArgs a{logits, stride, V, 0, 0, top, static_cast<float*>(part), nullptr, tokens, tokens64, logprobs, entropy,
                  top_logprobs, top_tokens, nullptr};
    const int u = plan(N, V, dtype, a.segments, a.words);
    ATTNLAB_REQUIRE(N * a.segments < (int64_t)1 << 31, "%lld rows of %d segments are too many", (long long)N, a.segments);
    const int64_t need = attnlab_logprob_part_bytes(N, V, dtype, top);
    ATTNLAB_REQUIRE(part && reinterpret_cast<uintptr_t>(part) % 16 == 0 && part_bytes >= need,
                    "part must be a 16-byte aligned device buffer of %lld bytes", (long long)need);
    a.best = reinterpret_cast<uint64_t*>(a.part + N * a.segments * kPartWords);
    a.arrive = a.segments * top <= kWaveKeys ? arrive : nullptr;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (dtype == ATTNLAB_DT_BF16) return launch<ATTNLAB_DT_BF16>(a, u, N, s);
    if (dtype == ATTNLAB_DT_F16) return launch<ATTNLAB_DT_F16>(a, u, N, s);
    return launch<ATTNLAB_DT_F32>(a, u, N, s);
}
