// Beam search: the choice of the next beams over beams and vocabulary, and the beams' rows of fixed
// size (recurrent states, last pages of a cache) put in the order of that choice.
//
//   de_beam_select   total[b, v] = score[b] + logit[b, v] - log(sum_w exp(logit[b, w])); the `take`
//                    largest totals of a group of beams, with their beams and tokens
//   de_beam_reorder  x[:, slots[g, b]] <- x[:, slots[g, parent[g, b]]], for all beams at once
//
// The reference decodes greedily (src/layers/sampler.py:5-8) and has neither.

#include "common.cuh"

DE_DEFINE_PDL_SWITCH

namespace {

constexpr int MAX_BEAMS = 32;
constexpr int MAX_TAKE = 64;
constexpr int MAX_VOCAB = 1 << 27;

// ------------------------------------------------------------------------------------------
// Selection.  Two launches: `slices` takes a slice of a row of logits to a block, which leaves the
// slice's maximum, its sum of exponentials and its `take` best logits; `join` takes a group of
// beams to a block, which forms the rows' normalisers and picks the best of what the slices left
// (within a row the order of the totals is the order of the logits, so the best of a row are among
// the best of its slices).
//
// Candidates are compared as integers: a float's bits mapped to an unsigned number of the same
// order, and below it the complement of the token, so that no two are equal and the lower token is
// the larger key.  0 is no candidate: NaN, and minus infinity, whose totals could never be taken.
//
// Which of two beams' candidates comes first depends on both rows' sums, and sums of float32
// exponentials are off by some 1e-7: `slices` forms them so (a 64-bit sum of groups of 16), and
// `join` compares with them only what is further apart than such sums can be wrong.  Where two
// neighbours in its order are nearer than that, or the last one taken and any candidate of another
// beam (one selection of a thousand, or beams with equal rows), it forms the sums of their rows again,
// as whole numbers of 2^-68 in two words, so that the order of a row's tokens does not matter and the
// smallest terms count (2^27 of them are off by 2^-42 together), and orders again.
// That is enough: a row's own candidates are in their order whatever its sum; whoever is in its wrong
// place against the last one taken is of another beam and near it; and between two of those taken
// that are the wrong way round all neighbours are near, and some of other beams.
//
// How far a fast sum may be off, relative to itself: ex2.approx 2^-22; its argument, a number of up to
// 25 below the largest, rounded to half a step of 2^-20 for the smallest terms, which can have half of
// the sum: 3.3e-7; four levels of float32 additions 2^-22; log2(e) as a float32, 1.3e-8 of up to 17:
// 2.3e-7.  In all 1.05e-6, and twice that between two rows.
// ------------------------------------------------------------------------------------------
typedef unsigned long long u64;

constexpr int SLICE_THREADS = 512;
constexpr int FOUND = 512;             // keys that a block keeps of its slice, to pick the best from
constexpr int QUADS = 4;               // 16-byte loads of a thread under way at once
constexpr int SEGMENTS = 2048;
constexpr int WINNERS = 320;           // segments that are looked at again
constexpr int JOIN_THREADS = 512;
constexpr int PICKS = 256;             // candidates of which the best are picked
constexpr double UNSURE = 2.2e-6;      // totals of two beams nearer than this are formed again
constexpr float COARSE = 1048576.0f;   // rows with a larger maximum: formed in 64 bits at once
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ unsigned ordered(float v) {    // of a number that is not NaN
    const unsigned u = __float_as_uint(v);
    return u ^ (unsigned)((int)u >> 31 | 0x80000000);
}
__device__ __forceinline__ u64 logit_key(float v, int token) {
    if (!(v > -INFINITY)) return 0;                       // NaN and minus infinity
    return (u64)ordered(v + 0.0f) << 32 | (unsigned)~token;        // (minus zero is as large as zero)
}
__device__ __forceinline__ float key_logit(u64 key) {
    const unsigned u = (unsigned)(key >> 32);
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ int key_token(u64 key) { return (int)~(unsigned)key; }

__device__ __forceinline__ u64 warp_largest(u64 v) {      // upper halves first, then the lower ones of those
    const unsigned high = __reduce_max_sync(0xffffffffu, (unsigned)(v >> 32));
    const unsigned low = (unsigned)(v >> 32) == high ? (unsigned)v : 0;
    return (u64)high << 32 | __reduce_max_sync(0xffffffffu, low);
}
__device__ __forceinline__ double shfl_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
// 2^n for an n of up to 1000 either way
__device__ __forceinline__ double power_of_two(float n) {
    return __hiloint2double((1023 + (int)fminf(fmaxf(n, -1000.0f), 1000.0f)) << 20, 0);
}
// The exponent that a row's, slice's or thread's terms are divided by 2 to the power of: a whole
// number, so that changing it is exact.
__device__ __forceinline__ float exponent_of(float top) {
    return rintf(fminf(fmaxf(top, -COARSE), COARSE) * LOG2E);
}

// A threshold with which `count(t)`, the number of keys of at least t over the block, lies between
// `want` and `most`, or all keys but 0 where there are at most `most`.  `low` is a guess from below
// (1: none), `top` the largest key; the range between is halved until it is met, which distinct keys
// guarantee for most >= want (keys that are the same end with the largest threshold that has `want`).
// `count` is called by all threads.
template <typename Count>
__device__ __forceinline__ u64 threshold(u64 low, u64 top, int want, int most, Count count) {
    u64 high = top;
    if (low > 1) {
        const int n = count(low);
        if (n >= want && n <= most) return low;
        if (n < want) { high = low - 1; low = 1; }
    }
    if (low <= 1) {
        if (top == 0 || count(1) <= most) return 1;
        low = 1;
    }
    while (low < high) {                                  // count(low) > most
        const u64 mid = low + ((high - low + 1) >> 1);
        const int n = count(mid);
        if (n >= want) {
            low = mid;
            if (n <= most) break;
        } else {
            high = mid - 1;
        }
    }
    return low;
}

// For each of n things, how many come before it: eight threads count for one.  `before(c, j)`, then
// `place(c, rank)` by one thread.
template <int THREADS, typename Before, typename Place>
__device__ __forceinline__ void rank_all(int n, Before before, Place place) {
    const int sub = threadIdx.x & 7;
    for (int first = 0; first < n; first += THREADS / 8) {
        const int c = first + (threadIdx.x >> 3);
        int rank = 0;
        if (c < n)
            for (int j = sub; j < n; j += 8) rank += before(c, j) ? 1 : 0;
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
        if (sub == 0 && c < n) place(c, rank);
    }
}

// A slice goes by in quads (four logits, a 16-byte load); up to three logits before the first 16-byte
// boundary and up to three behind the last quad are for themselves.  For the search of the best, runs
// of 2^shift quads form segments; segment 0 is the head, the last one the rest.
struct Quads {
    const float* x;          // the slice
    int n, head, count;      // logits; those before the boundary; whole quads
    int shift;               // the smallest segments of which there are not too many
    __device__ __forceinline__ Quads(const float* p, int logits) : x(p), n(logits) {
        head = min(n, (int)((16 - ((uintptr_t)p & 15)) & 15) >> 2);
        count = (n - head) >> 2;
        shift = 0;
        while ((count - 1) >> shift > SEGMENTS - 3) shift += shift == 0 ? 3 : shift == 3 ? 2 : 1;
    }
    __device__ __forceinline__ float4 quad(int i) const {
        return *(reinterpret_cast<const float4*>(x + head) + i);
    }
    __device__ __forceinline__ int segments() const { return ((count - 1) >> shift) + 3; }
    // logits of the head (0) or the rest (1), minus infinity where there is none
    __device__ __forceinline__ float4 edge(int which) const {
        const int first = edge_start(which), most = which ? n - first : head;
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = j < most ? x[first + j] : -INFINITY;
        return make_float4(v[0], v[1], v[2], v[3]);
    }
    __device__ __forceinline__ int edge_start(int which) const { return which ? head + 4 * count : 0; }
};
// (never NaN: the largest number, or minus infinity)
__device__ __forceinline__ float largest(const float4& v) {
    return fmaxf(fmaxf(fmaxf(v.x, v.y), v.z), fmaxf(v.w, -INFINITY));
}
constexpr unsigned NOTHING = 0x007fffffu;                 // ordered(-INFINITY)

template <int N> struct Int {
    static constexpr int value = N;
};

// One pass over the slice: the sum, and the maximum of every segment.  A segment whose maximum is not
// among the `take` largest holds none of the `take` best, so only as many segments are looked at
// again (1.5% of a row of 128,256, still in the L2 for the most part).
__global__ void __launch_bounds__(SLICE_THREADS, 4)
beam_slices_kernel(const float* __restrict__ logits, long long stride, int vocab, int slice,
                   int slices, int take, float* __restrict__ maxima, double* __restrict__ sums,
                   u64* __restrict__ keys) {
    __shared__ u64 found[FOUND];
    __shared__ unsigned segment_s[SEGMENTS];
    __shared__ unsigned part_top[SLICE_THREADS / 8];
    __shared__ double warp_sum_s[SLICE_THREADS / 32];
    __shared__ int winner_s[WINNERS], winners_s, count_s, counts_s[3];
    const int row = blockIdx.x / slices, part = blockIdx.x % slices;
    const int begin = part * slice;
    const Quads quads(logits + (long long)row * stride + begin, min(vocab, begin + slice) - begin);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int shift = quads.shift, segments = quads.segments();
    if (tid == 0) count_s = 0;
    if (tid < 3) counts_s[tid] = 0;
    if (shift > 5) {                                      // several warps' loads form a segment
        for (int i = tid; i < segments; i += SLICE_THREADS) segment_s[i] = 0;
        __syncthreads();
    }
    pdl_wait();
    // the sum of 2^(logit log2(e) - r), with an r near the largest so far
    float top_v = -INFINITY, r = 0.0f;
    double sum = 0.0;
    auto follow = [&](float m) {
        if (!(m > top_v)) return;
        if (top_v == -INFINITY || m * LOG2E > r + 1.0f) {
            const float to = exponent_of(m);
            sum *= power_of_two(r - to);                  // (0 when there was nothing before)
            r = to;
        }
        top_v = m;
    };
    auto terms = [&](const float4& v) {
        return (exp2_fast(fmaf(v.x, LOG2E, -r)) + exp2_fast(fmaf(v.y, LOG2E, -r))) +
               (exp2_fast(fmaf(v.z, LOG2E, -r)) + exp2_fast(fmaf(v.w, LOG2E, -r)));
    };
    // LANES of a warp form a segment; 33: more than a warp
    auto go_through = [&](auto lanes) {
        constexpr int LANES = decltype(lanes)::value;
        const float4* p = reinterpret_cast<const float4*>(quads.x + quads.head) + tid;
        auto step = [&](int base, const float4 (&v)[QUADS], int left) {
            float m[QUADS];
#pragma unroll
            for (int u = 0; u < QUADS; ++u) m[u] = largest(v[u]);
            follow(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])));
#pragma unroll
            for (int u = 0; u < QUADS; ++u) {
                unsigned o = ordered(m[u] + 0.0f);
                if (LANES == 8) {
#pragma unroll
                    for (int d = 1; d < 8; d <<= 1) o = max(o, __shfl_xor_sync(0xffffffffu, o, d));
                } else if (LANES >= 32) {
                    o = __reduce_max_sync(0xffffffffu, o);
                }
                const int i = base + u * SLICE_THREADS + tid;
                if (u * SLICE_THREADS < left && (LANES == 1 || lane % (LANES < 32 ? LANES : 32) == 0)) {
                    if (LANES > 32) atomicMax(&segment_s[1 + (i >> shift)], o);
                    else segment_s[1 + i / LANES] = o;
                }
            }
            sum += (double)((terms(v[0]) + terms(v[1])) + (terms(v[2]) + terms(v[3])));
        };
        int base = 0;
        for (; base + QUADS * SLICE_THREADS <= quads.count; base += QUADS * SLICE_THREADS) {
            float4 v[QUADS];
#pragma unroll
            for (int u = 0; u < QUADS; ++u) v[u] = p[base + u * SLICE_THREADS];
            step(base, v, QUADS * SLICE_THREADS);
        }
        if (base < quads.count) {
            float4 v[QUADS];
#pragma unroll
            for (int u = 0; u < QUADS; ++u)
                v[u] = base + u * SLICE_THREADS + tid < quads.count
                           ? p[base + u * SLICE_THREADS]
                           : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            step(base, v, quads.count - base - tid);
        }
    };
    if (shift == 0) go_through(Int<1>());
    else if (shift == 3) go_through(Int<8>());
    else if (shift == 5) go_through(Int<32>());
    else go_through(Int<33>());
    if (tid < 2) {
        const float4 v = quads.edge(tid);
        const float m = largest(v);
        follow(m);
        segment_s[tid ? segments - 1 : 0] = ordered(m + 0.0f);
        sum += (double)terms(v);
    }
    __syncthreads();
    // The largest; and a guess at the last of the `take` largest segments: where as many parts of the block as
    // are taken hold a number, each has a segment of at least the smallest part's largest.
    // (Part p has every 64th segment from p on, so that few segments are spread over all parts.)
    unsigned mine = 0;
    for (int i = (tid & 7) * (SLICE_THREADS / 8) + (tid >> 3); i < segments; i += SLICE_THREADS)
        mine = max(mine, segment_s[i]);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
    if ((lane & 7) == 0) part_top[tid >> 3] = mine;
    __syncthreads();
    const unsigned x = part_top[2 * lane], y = part_top[2 * lane + 1];
    const unsigned top = __reduce_max_sync(0xffffffffu, max(x, y));
    unsigned guess = max(x, y);
    if (take <= 16) guess = max(guess, __shfl_xor_sync(0xffffffffu, guess, 1));
    int parts = __popc(__ballot_sync(0xffffffffu, guess > NOTHING));
    if (take <= 16) parts >>= 1;
    guess = guess > NOTHING ? guess : 0xffffffffu;
    if (take > 32) {                                      // each of the two for itself
        parts = __popc(__ballot_sync(0xffffffffu, x > NOTHING)) +
                __popc(__ballot_sync(0xffffffffu, y > NOTHING));
        guess = min(x > NOTHING ? x : 0xffffffffu, y > NOTHING ? y : 0xffffffffu);
    }
    guess = __reduce_min_sync(0xffffffffu, guess);
    if (parts < take) guess = 0;
    const float m = top > NOTHING ? key_logit((u64)top << 32) : -INFINITY;

    sum = shfl_sum(sum * power_of_two(r - exponent_of(m)));
    if (lane == 0) warp_sum_s[warp] = sum;

    // Segments with at least the guess's maximum are few enough nearly always.  Where they are not,
    // segments are told apart by their maxima and, equal ones, by their place.
    auto segment_key = [&](int i) {
        const unsigned o = segment_s[i];
        return o > NOTHING ? (u64)o << 32 | (unsigned)~i : 0;
    };
    int turn = 0;                                         // one barrier a count: three counters in turn
    auto segments_from = [&](u64 t) {
        int k = 0;
        for (int i = tid; i < segments; i += SLICE_THREADS) k += segment_key(i) >= t;
        k = __reduce_add_sync(0xffffffffu, k);
        if (lane == 0 && k) atomicAdd(&counts_s[turn], k);
        __syncthreads();
        k = counts_s[turn];
        turn = turn == 2 ? 0 : turn + 1;
        if (tid == 0) counts_s[turn == 2 ? 0 : turn + 1] = 0;
        return k;
    };
    const u64 last = threshold(guess > NOTHING ? (u64)guess << 32 : 1, (u64)top << 32 | 0xffffffffu, take,
                               min(max(6 * take, 96), WINNERS), segments_from);
    if (tid == 0) winners_s = 0;
    __syncthreads();
    for (int i = tid; i < segments; i += SLICE_THREADS)
        if (segment_key(i) >= last) winner_s[atomicAdd(&winners_s, 1)] = i;
    __syncthreads();
    // The keys of at least t in those segments, all their quads side by side; how many there are.
    auto collect = [&](u64 t) {
        float floor_v = key_logit(t);
        if (floor_v != floor_v) floor_v = -INFINITY;      // (a threshold below all numbers)
        auto keep = [&](const float4& v, int first) {
            const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const u64 k = logit_key(e[j], begin + first + j);
                if (k < t || k == 0) continue;
                const int at = atomicAdd(&count_s, 1);
                if (at < FOUND) found[at] = k;
            }
        };
        const int all = winners_s << shift;
        for (int base = tid; base < all; base += QUADS * SLICE_THREADS) {
            float4 v[QUADS];
            int first[QUADS];
#pragma unroll
            for (int u = 0; u < QUADS; ++u) {
                const int at = base + u * SLICE_THREADS;
                first[u] = -1;
                if (at >= all) continue;
                const int s = winner_s[at >> shift], q = at & ((1 << shift) - 1);
                const int i = ((s - 1) << shift) + q;
                if (s == 0 || s == segments - 1) {
                    if (q) continue;
                    v[u] = quads.edge(s != 0);
                    first[u] = quads.edge_start(s != 0);
                } else if (i < quads.count) {
                    v[u] = quads.quad(i);
                    first[u] = quads.head + 4 * i;
                }
            }
#pragma unroll
            for (int u = 0; u < QUADS; ++u)
                if (first[u] >= 0 && largest(v[u]) >= floor_v) keep(v[u], first[u]);
        }
        __syncthreads();
        return count_s;
    };
    u64 low = last >> 32 << 32, high = (u64)top << 32 | 0xffffffffu;
    int n = collect(low);
    if (n > FOUND)                                        // the best are crowded in few segments
        while (low < high) {
            const u64 mid = low + ((high - low + 1) >> 1);
            __syncthreads();
            if (tid == 0) count_s = 0;
            __syncthreads();
            n = collect(mid);
            if (n >= take) {
                low = mid;
                if (n <= FOUND) break;
            } else {
                high = mid - 1;
            }
        }
    pdl_trigger();
    u64* out = keys + (size_t)blockIdx.x * take;
    rank_all<SLICE_THREADS>(n, [&](int c, int j) { return found[j] > found[c]; }, [&](int c, int rank) {
        if (rank < take) out[rank] = found[c];
    });
    for (int c = n + tid; c < take; c += SLICE_THREADS) out[c] = 0;
    if (tid == 0) {
        double all = 0.0;
        for (int w = 0; w < SLICE_THREADS / 32; ++w) all += warp_sum_s[w];
        maxima[blockIdx.x] = m;
        sums[blockIdx.x] = all;                           // NaN where a logit is
    }
}

// a total's bits as an unsigned number of the same order; 0 for one that is no candidate
__device__ __forceinline__ u64 total_key(double t) {
    if (!(t > (double)-INFINITY)) return 0;
    const u64 u = (u64)__double_as_longlong(t);
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ double key_total(u64 k) {
    return __longlong_as_double((long long)(k >> 63 ? k & 0x7fffffffffffffffull : ~k));
}

__global__ void __launch_bounds__(JOIN_THREADS)
beam_join_kernel(const float* __restrict__ logits, long long stride, int vocab,
                 const float* __restrict__ scores, int beams, int slices, int take,
                 const float* __restrict__ maxima, const double* __restrict__ sums,
                 const u64* __restrict__ keys, float* __restrict__ best, int* __restrict__ beam,
                 int* __restrict__ token) {
    extern __shared__ u64 total_s[];                      // [beams x slices x take], twice
    u64* key_s = total_s + beams * slices * take;
    __shared__ double max_s[MAX_BEAMS], log_s[MAX_BEAMS]; // log(sum exp) of a row: max + log
    __shared__ u64 warp_part[2][JOIN_THREADS / 32];
    __shared__ int counts_s[3];
    __shared__ int pick_s[PICKS], order_s[MAX_TAKE];
    __shared__ u64 pick_total_s[PICKS];
    __shared__ float score_s[MAX_BEAMS];
    __shared__ int count_s;
    __shared__ unsigned again_s;                          // rows whose sums are to be formed again
    const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) again_s = 0;
    if (tid < 3) counts_s[tid] = 0;
    __syncthreads();
    const int per_beam = slices * take, n = beams * per_beam;
    const u64* mine = keys + (size_t)g * n;
    pdl_wait();
    pdl_trigger();
    if (tid < beams) score_s[tid] = scores[(size_t)g * beams + tid];
    for (int c = tid; c < n; c += JOIN_THREADS)           // (while the rows' sums are on their way)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8;\n" ::"r"(
                         (unsigned)__cvta_generic_to_shared(key_s + c)), "l"(mine + c) : "memory");
    for (int b = warp; b < beams; b += JOIN_THREADS / 32) {
        const size_t at = ((size_t)g * beams + b) * slices;
        // (a lane's sum refers to the exponent of its own slices' maximum, as the threads' did)
        float m = -INFINITY;
        double sum = 0.0;
        auto shrink = [](float e) { return e < -1000.0f ? 0.0 : power_of_two(e); };
        for (int s = lane; s < slices; s += 32) {
            const float x = maxima[at + s];
            const double y = sums[at + s], top = fmaxf(m, x);
            sum = (sum != 0.0 ? sum * shrink(exponent_of(m) - exponent_of(top)) : 0.0) +
                  (y != 0.0 ? y * shrink(exponent_of(x) - exponent_of(top)) : 0.0);
            m = top;
        }
        const float own = exponent_of(m);
        m = warp_max(m);
        const float r = exponent_of(m);
        sum = shfl_sum(sum != 0.0 ? sum * shrink(own - r) : 0.0);
        if (lane == 0) {
            // (a float32 log2(e) makes the logits larger by a factor, which is taken back for the
            // largest: what is left is the factor on the others' distance from it)
            max_s[b] = (double)m;
            log_s[b] = m < INFINITY ? log(sum) + ((double)r - (double)LOG2E * (double)m) * 0.6931471805599453
                                    : (double)NAN;
            if (sum == sum && (m > COARSE || m < -COARSE) && m > -INFINITY && m < INFINITY)
                atomicOr(&again_s, 1u << b);
        }
    }
    // (the logit less the row's maximum first: both may be the lowest number there is)
    auto total_of = [&](int c) {
        const int b = c / per_beam;
        return (double)score_s[b] +
               (((double)key_logit(key_s[c]) - max_s[b]) - log_s[b]);
    };
    int turn = 0;                             // one barrier a count: three counters in turn
    auto over_block = [&](auto test) {
        int k = 0;
        for (int c = tid; c < n; c += JOIN_THREADS) k += test(c) ? 1 : 0;
        k = __reduce_add_sync(0xffffffffu, k);
        if (lane == 0) atomicAdd(&counts_s[turn], k);
        __syncthreads();
        k = counts_s[turn];
        turn = turn == 2 ? 0 : turn + 1;
        if (tid == 0) counts_s[turn == 2 ? 0 : turn + 1] = 0;
        return k;
    };
    auto place = [&](int c) {                 // of equal totals: beam, larger logit, lower token
        const u64 k = key_s[c];
        return (u64)(c / per_beam) << 59 | (u64)(unsigned)~(unsigned)(k >> 32) << 27 |
               (unsigned)key_token(k);
    };
    asm volatile("cp.async.wait_all;\n" ::: "memory");
    const int most = max(2 * take, 96);
    unsigned formed = 0;                                  // rows whose sums are 64-bit ones
    int found;
    for (;;) {
        if (tid == 0) count_s = 0;
        __syncthreads();
        const unsigned again = again_s & ~formed;
        formed |= again;
        for (int b = 0; b < beams; ++b) {
            if (!(again >> b & 1)) continue;
            // a term, of up to 1, as a whole number of 2^-34 and what is left of it of 2^-68: sums of up to
            // 2^27 of either fit 62 bits
            constexpr double UNIT = 17179869184.0;        // 2^34
            const float* x = logits + ((long long)g * beams + b) * stride;
            const double m = max_s[b];
            u64 high = 0, low = 0;
            for (int i = tid; i < vocab; i += JOIN_THREADS) {
                const double e = exp((double)x[i] - m) * UNIT, whole = floor(e);
                high += (u64)__double2ll_rn(whole);
                low += (u64)__double2ll_rn((e - whole) * UNIT);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                high += __shfl_xor_sync(0xffffffffu, high, o);
                low += __shfl_xor_sync(0xffffffffu, low, o);
            }
            if (lane == 0) { warp_part[0][warp] = high; warp_part[1][warp] = low; }
            __syncthreads();
            if (tid == 0) {
                high = low = 0;
                for (int w = 0; w < JOIN_THREADS / 32; ++w) {
                    high += warp_part[0][w];
                    low += warp_part[1][w];
                }
                log_s[b] = log(((double)high + (double)low / UNIT) / UNIT);
            }
            __syncthreads();
        }
        if (n <= PICKS / 2) {                             // few: all are ranked
            for (int c = tid; c < n; c += JOIN_THREADS) {
                const u64 t = key_s[c] ? total_key(total_of(c)) : 0;
                total_s[c] = t;
                if (t) {
                    const int at = atomicAdd(&count_s, 1);
                    pick_s[at] = c;
                    pick_total_s[at] = t;
                }
            }
        } else {
            // the largest, and a guess at the last one taken: the largest last one of a slice, which has
            // as many as are taken that are no smaller
            u64 top = 0, guess = 0;
            for (int c = tid; c < n; c += JOIN_THREADS) {
                const u64 t = key_s[c] ? total_key(total_of(c)) : 0;
                total_s[c] = t;
                top = max(top, t);
            }
            for (int i = tid; i < beams * slices; i += JOIN_THREADS) {
                const int c = i * take + take - 1;
                if (key_s[c]) guess = max(guess, total_key(total_of(c)));
            }
            top = warp_largest(top);
            guess = warp_largest(guess);
            if (lane == 0) { warp_part[0][warp] = top; warp_part[1][warp] = guess; }
            __syncthreads();
            for (int w = 0; w < JOIN_THREADS / 32; ++w) {
                top = max(top, warp_part[0][w]);
                guess = max(guess, warp_part[1][w]);
            }

            // the best by their totals; of those with the total of the last place the first by `place`
            const u64 t0 = threshold(guess, top, take, most, [&](u64 t) {
                return over_block([&](int c) { return total_s[c] >= t; });
            });
            u64 last = ~0ull;
            if (over_block([&](int c) { return total_s[c] >= t0; }) > most) {
                const int above = over_block([&](int c) { return total_s[c] > t0; });
                u64 low = 0, high = ~0ull;
                while (low < high) {
                    const u64 mid = low + ((high - low) >> 1);
                    const int k = over_block([&](int c) { return total_s[c] == t0 && place(c) <= mid; });
                    if (above + k >= take) high = mid; else low = mid + 1;
                }
                last = high;
            }
            for (int c = tid; c < n; c += JOIN_THREADS) {
                const u64 t = total_s[c];
                if (t > t0 || (t == t0 && t != 0 && place(c) <= last)) {
                    const int at = atomicAdd(&count_s, 1);
                    pick_s[at] = c;
                    pick_total_s[at] = t;
                }
            }
        }
        __syncthreads();
        found = count_s;
        rank_all<JOIN_THREADS>(found, [&](int i, int j) {
            const u64 x = pick_total_s[i], y = pick_total_s[j];
            return y > x || (y == x && place(pick_s[j]) < place(pick_s[i]));
        }, [&](int i, int rank) {
            if (rank < take) order_s[rank] = pick_s[i];
        });
        __syncthreads();
        found = min(found, take);
        // candidates of different beams that are too near each other for the sums that they have
        auto compare = [&](int c, int d) {
            const int b = c / per_beam, e = d / per_beam;
            const unsigned rows = 1u << b | 1u << e;
            const double a = key_total(total_s[c]), z = key_total(total_s[d]);
            if (b != e && (rows & ~formed) && fabs(a) < INFINITY && fabs(a - z) <= UNSURE)
                atomicOr(&again_s, rows);
        };
        if (tid + 1 < found) compare(order_s[tid], order_s[tid + 1]);
        if (found == take)
            for (int c = tid; c < n; c += JOIN_THREADS)
                if (total_s[c]) compare(order_s[take - 1], c);
        __syncthreads();
        if (!(again_s & ~formed)) break;
    }
    for (int i = tid; i < take; i += JOIN_THREADS) {
        const size_t at = (size_t)g * take + i;
        const int c = i < found ? order_s[i] : -1;
        best[at] = c < 0 ? -INFINITY : (float)key_total(total_s[c]);
        beam[at] = c < 0 ? -1 : c / per_beam;
        token[at] = c < 0 ? -1 : key_token(key_s[c]);
    }
}

// Slices that a row is cut into, and their logits.  A block an SM; more, up to the four that an SM holds at
// once, only of 32,768 logits and longer, since a block's end takes some microseconds (us with one and with up
// to four blocks an SM: 64 rows of 32,000 10.7 and 16.8, 35 of 50,021 13.8 and 16.4, 186 of 79,707 28.7 and
// 25.4).  No slice is shorter than 2,048 logits, and the slices of a group leave no more than 1,024 candidates,
// for the block that joins them (eight rows of 128,256, 16 taken, with 512, 1,024, 2,048 and 8,192: 16.2, 14.0,
// 14.2 and 23.9).
struct Slicing {
    int slices, elements;
};
constexpr int JOIN_MOST = 1024;
Slicing slicing(int rows, int beams, int vocab, int take) {
    int slices = rows > 0 ? 148 / rows : 1;
    const int longer = rows > 0 ? 4 * 148 / rows : 1, whole = vocab / 32768;
    if (slices < longer && slices < whole) slices = longer < whole ? longer : whole;
    const int least = vocab / (4 * SLICE_THREADS), most = JOIN_MOST / (beams * take);
    if (slices > least) slices = least;
    if (slices > most) slices = most;
    if (slices < 1) slices = 1;
    Slicing s;
    s.elements = (vocab + slices - 1) / slices;
    s.slices = (vocab + s.elements - 1) / s.elements;
    return s;
}
size_t aligned(size_t bytes) { return (bytes + 15) & ~(size_t)15; }

// ------------------------------------------------------------------------------------------
// Reordering.  x is [layers, pool, width]; a thread owns one piece of a row's width in all rows of a
// group in one layer: it reads the pieces of every row that a moved beam takes, and only then writes,
// so the rows can change places without a buffer.
// ------------------------------------------------------------------------------------------
constexpr int MOVE_THREADS = 256;
// Blocks of a launch for every SM.  (us for 2, 4, 8 and 16: four beams of sixteen groups, pages of 32 x 16 x 128
// bfloat16 in 32 layers, 69, 65, 60 and 58; eight beams of eight groups, states of 16 x 128 x 128 floats in six
// layers, 102, 96, 88 and 85, where a plain copy of the bytes takes 80.)
constexpr int MOVE_BLOCKS = 16;

// pieces of a row that a thread has under way at once: as many as 64 registers hold for all beams
template <typename U, int BEAMS> __host__ __device__ constexpr int pieces_at_once() {
    const int n = 256 / (BEAMS * (int)sizeof(U));
    return n < 1 ? 1 : n > 8 ? 8 : n;
}

template <typename U, int BEAMS>
__global__ void __launch_bounds__(MOVE_THREADS)
beam_reorder_kernel(unsigned char* __restrict__ x, long long row_bytes, int pool,
                    const int* __restrict__ slots, const int* __restrict__ parent, int groups,
                    int beams, int chunks, int units, int* __restrict__ status) {
    constexpr int N = pieces_at_once<U, BEAMS>();
    __shared__ int from_s[BEAMS], to_s[BEAMS], slot_s[BEAMS];
    const int g = blockIdx.y, tid = threadIdx.x;
    pdl_wait();
    pdl_trigger();
    if (tid < BEAMS) slot_s[tid] = tid < beams ? slots[g * beams + tid] : -1;
    __syncthreads();
    // a row that two beams hold cannot be moved: nothing of the group moves then
    bool twice = false;
    for (int i = tid; i < groups * beams; i += MOVE_THREADS) {
        const int s = slots[i];
        for (int b = 0; b < beams; ++b)
            twice |= s >= 0 && s == slot_s[b] && i != g * beams + b;
    }
    twice = __syncthreads_or(twice);
    if (tid < BEAMS) {
        int from = -1, to = -1;
        bool bad = twice;
        if (tid < beams && !twice) {
            const int s = slot_s[tid], p = parent[g * beams + tid];
            bad = s < -1 || s >= pool || p < -1 || p >= beams;
            if (!bad && s >= 0 && p >= 0 && p != tid) {
                const int src = slot_s[p];
                bad = src < 0 || src >= pool;
                if (!bad) { from = src; to = s; }
            }
        }
        if (bad && tid < beams) atomicExch(status, 5);
        from_s[tid] = from;
        to_s[tid] = to;
    }
    __syncthreads();
    // a chunk is N pieces of every thread; layer after layer, the blocks of the group in turn
    for (int unit = blockIdx.x; unit < units; unit += gridDim.x) {
        const long long at = ((long long)(unit % chunks) * N * MOVE_THREADS + tid) * sizeof(U);
        unsigned char* base = x + (long long)(unit / chunks) * pool * row_bytes + at;
        U v[BEAMS][N];
#pragma unroll
        for (int b = 0; b < BEAMS; ++b) {
            if (from_s[b] < 0) continue;
            const unsigned char* src = base + from_s[b] * row_bytes;
#pragma unroll
            for (int n = 0; n < N; ++n)
                if (at + n * MOVE_THREADS * (long long)sizeof(U) < row_bytes)
                    v[b][n] = *reinterpret_cast<const U*>(src + n * MOVE_THREADS * sizeof(U));
        }
#pragma unroll
        for (int b = 0; b < BEAMS; ++b) {
            if (from_s[b] < 0) continue;
            unsigned char* dst = base + to_s[b] * row_bytes;
#pragma unroll
            for (int n = 0; n < N; ++n)
                if (at + n * MOVE_THREADS * (long long)sizeof(U) < row_bytes)
                    *reinterpret_cast<U*>(dst + n * MOVE_THREADS * sizeof(U)) = v[b][n];
        }
    }
}

template <typename U, int BEAMS>
int reorder_with(unsigned char* x, int layers, int pool, long long row_bytes, const int* slots,
                 const int* parent, int groups, int beams, int* status, cudaStream_t stream) {
    const long long per_chunk = pieces_at_once<U, BEAMS>() * MOVE_THREADS * (long long)sizeof(U);
    const long long chunks = (row_bytes + per_chunk - 1) / per_chunk, units = chunks * layers;
    if (units > 0x7fffffffll || groups > 65535) return -4;
    // a block looks the group's moves up once and goes through several chunks
    long long blocks = (MOVE_BLOCKS * 148 + groups - 1) / groups;
    if (blocks > units) blocks = units;
    return de_launch(beam_reorder_kernel<U, BEAMS>, dim3((unsigned)blocks, groups), dim3(MOVE_THREADS),
                     0, stream, x, row_bytes, pool, slots, parent, groups, beams, (int)chunks,
                     (int)units, status);
}
template <typename U>
int reorder_of(unsigned char* x, int layers, int pool, long long row_bytes, const int* slots,
               const int* parent, int groups, int beams, int* status, cudaStream_t stream) {
    if (beams <= 4)
        return reorder_with<U, 4>(x, layers, pool, row_bytes, slots, parent, groups, beams, status, stream);
    if (beams <= 8)
        return reorder_with<U, 8>(x, layers, pool, row_bytes, slots, parent, groups, beams, status, stream);
    if (beams <= 16)
        return reorder_with<U, 16>(x, layers, pool, row_bytes, slots, parent, groups, beams, status, stream);
    return reorder_with<U, 32>(x, layers, pool, row_bytes, slots, parent, groups, beams, status, stream);
}

}  // namespace

DE_EXPORT int de_beam_max_beams() { return MAX_BEAMS; }
DE_EXPORT int de_beam_max_take() { return MAX_TAKE; }

// Bytes of scratch memory that de_beam_select needs for these sizes; negative: sizes it refuses.
DE_EXPORT int de_beam_scratch(int groups, int beams, int vocab, int take) {
    if (groups < 0 || beams < 1 || beams > MAX_BEAMS || take < 1 || take > MAX_TAKE || vocab < 1 ||
        vocab > MAX_VOCAB || (long long)groups * beams > (1 << 20))
        return -2;
    const Slicing s = slicing(groups * beams, beams, vocab, take);
    const size_t n = (size_t)groups * beams * s.slices;
    const size_t bytes = aligned(4 * n) + aligned(8 * n) + 8 * n * take;
    return bytes > 0x7fffffff ? -4 : (int)bytes;
}

DE_EXPORT int de_beam_select(const float* logits, long long stride, const float* scores, int groups,
                             int beams, int vocab, int take, float* best, int* beam, int* token,
                             void* scratch, void* stream) {
    const int bytes = de_beam_scratch(groups, beams, vocab, take);
    if (bytes < 0) return bytes;
    if (groups == 0) return 0;
    const Slicing s = slicing(groups * beams, beams, vocab, take);
    const size_t n = (size_t)groups * beams * s.slices;
    float* maxima = (float*)scratch;
    double* sums = (double*)((char*)scratch + aligned(4 * n));
    u64* keys = (u64*)((char*)sums + aligned(8 * n));
    const int totals = 2 * beams * s.slices * take * 8;   // (up to 32 KB)
    const int code = de_launch(beam_slices_kernel, dim3((unsigned)n), dim3(SLICE_THREADS), 0,
                               (cudaStream_t)stream, logits, stride, vocab, s.elements, s.slices, take,
                               maxima, sums, keys);
    if (code) return code;
    return de_launch(beam_join_kernel, dim3(groups), dim3(JOIN_THREADS), totals,
                     (cudaStream_t)stream, logits, stride, vocab, scores, beams, s.slices, take, maxima,
                     sums, keys, best, beam, token);
}

// x: [layers, pool] rows of row_bytes bytes; slots, parent: int32 [groups, beams].
DE_EXPORT int de_beam_reorder(void* x, int layers, int pool, long long row_bytes, const int* slots,
                              const int* parent, int groups, int beams, int* status, void* stream) {
    if (beams < 1 || beams > MAX_BEAMS || layers < 0 || pool < 0 || groups < 0 || row_bytes < 0)
        return -2;
    if (layers == 0 || groups == 0 || row_bytes == 0) return 0;
    const unsigned long long bits = (unsigned long long)(uintptr_t)x | (unsigned long long)row_bytes;
    unsigned char* p = (unsigned char*)x;
    cudaStream_t s = (cudaStream_t)stream;
    if (bits % 16 == 0) return reorder_of<uint4>(p, layers, pool, row_bytes, slots, parent, groups, beams, status, s);
    if (bits % 8 == 0) return reorder_of<uint2>(p, layers, pool, row_bytes, slots, parent, groups, beams, status, s);
    if (bits % 4 == 0) return reorder_of<unsigned>(p, layers, pool, row_bytes, slots, parent, groups, beams, status, s);
    if (bits % 2 == 0) return reorder_of<unsigned short>(p, layers, pool, row_bytes, slots, parent, groups, beams, status, s);
    return reorder_of<unsigned char>(p, layers, pool, row_bytes, slots, parent, groups, beams, status, s);
}
