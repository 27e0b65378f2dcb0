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
// neighbours in its order are nearer than that (one selection of a thousand, or beams with equal
// rows), it forms the sums of their rows again in 64 bits, as integers, so that the order of a row's
// tokens does not matter, and orders again.
//
// How far a fast sum may be off, relative to itself: ex2.approx 2^-22; its argument, a number of up to
// 25 below the largest, rounded to half a step of 2^-20 for the smallest terms, which can have half of
// the sum: 3.3e-7; four levels of float32 additions 2^-22; log2(e) as a float32, 1.3e-8 of up to 17:
// 2.3e-7.  In all 1.05e-6, and twice that between two rows.
// ------------------------------------------------------------------------------------------
typedef unsigned long long u64;

constexpr int SLICE_THREADS = 512;
constexpr int JOIN_THREADS = 512;
constexpr double UNSURE = 2.2e-6;      // totals of two beams nearer than this are formed again
constexpr float COARSE = 1048576.0f;   // rows with a larger maximum: formed in 64 bits at once
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ u64 logit_key(float v, int token) {
    if (!(v > -INFINITY)) return 0;                       // NaN and minus infinity
    const unsigned u = __float_as_uint(v + 0.0f);         // (minus zero is as large as zero)
    const unsigned ordered = u & 0x80000000u ? ~u : u | 0x80000000u;
    return (u64)ordered << 32 | (unsigned)~token;
}
__device__ __forceinline__ float key_logit(u64 key) {
    const unsigned ordered = (unsigned)(key >> 32);
    return __uint_as_float(ordered & 0x80000000u ? ordered & 0x7fffffffu : ~ordered);
}
__device__ __forceinline__ int key_token(u64 key) { return (int)~(unsigned)key; }

__device__ __forceinline__ u64 shfl_max(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const u64 w = __shfl_xor_sync(0xffffffffu, v, o);
        v = w > v ? w : v;
    }
    return v;
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
// `want` and `most`; 1 if there are at most `most` keys that are not 0 in all.  Halves the range
// of the keys until it is met, which distinct keys guarantee for most >= want.  `count` is called
// by all threads; `top` is the largest key.
template <typename Count>
__device__ __forceinline__ u64 threshold(u64 top, int want, int most, Count count) {
    if (top == 0 || count(1) <= most) return 1;
    u64 low = 1, high = top;                              // count(low) > most, and high not below it
    while (low < high) {
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

// A slice goes by in pieces of four logits (one 16-byte load); up to three logits before the first
// 16-byte boundary and behind the last are pieces of their own.
struct Pieces {
    const float* x;          // the slice
    int n, head, quads;      // logits; those before the boundary; whole pieces
    __device__ __forceinline__ Pieces(const float* p, int count) : x(p), n(count) {
        head = min(n, (int)((16 - ((uintptr_t)p & 15)) & 15) >> 2);
        quads = (n - head) >> 2;
    }
    __device__ __forceinline__ int count() const { return quads + 2; }
    // piece i: 0 .. quads - 1 whole ones, quads the head, quads + 1 the rest; -inf where there is none
    __device__ __forceinline__ float4 get(int i) const {
        if (i < quads) return __ldg(reinterpret_cast<const float4*>(x + head) + i);
        float v[4];
        const int first = start(i), most = i == quads ? head : i == quads + 1 ? n - first : 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = j < most ? x[first + j] : -INFINITY;
        return make_float4(v[0], v[1], v[2], v[3]);
    }
    __device__ __forceinline__ int start(int i) const {
        return i < quads ? head + 4 * i : i == quads ? 0 : head + 4 * quads;
    }
};

__global__ void __launch_bounds__(SLICE_THREADS)
beam_slices_kernel(const float* __restrict__ logits, long long stride, int vocab, int slice,
                   int slices, int take, float* __restrict__ maxima, double* __restrict__ sums,
                   u64* __restrict__ keys) {
    extern __shared__ u64 found[];                        // [2 take x logits of a thread]
    __shared__ u64 warp_top[SLICE_THREADS / 32];
    __shared__ double warp_sum_s[SLICE_THREADS / 32];
    __shared__ int count_s;
    const int row = blockIdx.x / slices, part = blockIdx.x % slices;
    const int begin = part * slice;
    const Pieces pieces(logits + (long long)row * stride + begin, min(vocab, begin + slice) - begin);
    const int count = pieces.count();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) count_s = 0;
    pdl_wait();
    // the largest logit and the first piece that holds it; the sum of 2^(logit log2(e) - r)
    float top_v = -INFINITY, r = 0.0f;
    int top_piece = -1;
    double sum = 0.0;
    for (int i = tid; i < count; i += 4 * SLICE_THREADS) {
        float4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            v[u] = i + u * SLICE_THREADS < count
                       ? pieces.get(i + u * SLICE_THREADS)
                       : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        const float before = top_v;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float m = fmaxf(fmaxf(v[u].x, v[u].y), fmaxf(v[u].z, v[u].w));
            if (m > top_v) { top_v = m; top_piece = i + u * SLICE_THREADS; }
        }
        if (top_v > before && (before == -INFINITY || top_v * LOG2E > r + 1.0f)) {
            const float to = exponent_of(top_v);
            sum *= power_of_two(r - to);                  // (0 when there was nothing before)
            r = to;
        }
        float part_sum[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            part_sum[u] = (exp2_fast(fmaf(v[u].x, LOG2E, -r)) + exp2_fast(fmaf(v[u].y, LOG2E, -r))) +
                          (exp2_fast(fmaf(v[u].z, LOG2E, -r)) + exp2_fast(fmaf(v[u].w, LOG2E, -r)));
        sum += (double)((part_sum[0] + part_sum[1]) + (part_sum[2] + part_sum[3]));
    }
    u64 mine = 0;
    if (top_piece >= 0) {
        const float4 v = pieces.get(top_piece);
        const float e[4] = {v.x, v.y, v.z, v.w};
        int at = 3;
#pragma unroll
        for (int j = 3; j >= 0; --j)
            if (e[j] == top_v) at = j;
        mine = logit_key(top_v, begin + pieces.start(top_piece) + at);
    }
    u64 top = shfl_max(mine);
    if (lane == 0) warp_top[warp] = top;
    __syncthreads();
    top = 0;
    for (int w = 0; w < SLICE_THREADS / 32; ++w) top = max(top, warp_top[w]);
    const float m = top ? key_logit(top) : -INFINITY;
    sum = shfl_sum(sum * power_of_two(r - exponent_of(m)));
    if (lane == 0) warp_sum_s[warp] = sum;

    // the threads whose largest key is below the threshold have none of the best; the others look again
    const u64 floor_key = threshold(top, min(take, SLICE_THREADS), 2 * take, [&](u64 t) {
        return __syncthreads_count(mine >= t);
    });
    if (mine >= floor_key)
        for (int i = tid; i < count; i += SLICE_THREADS) {
            const float4 v = pieces.get(i);
            const float e[4] = {v.x, v.y, v.z, v.w};
            const int first = begin + pieces.start(i);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const u64 k = logit_key(e[j], first + j);
                if (k >= floor_key) found[atomicAdd(&count_s, 1)] = k;
            }
        }
    __syncthreads();
    pdl_trigger();
    const int n = count_s;
    u64* out = keys + (size_t)blockIdx.x * take;
    for (int c = tid; c < n; c += SLICE_THREADS) {
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += found[j] > found[c];
        if (rank < take) out[rank] = found[c];
    }
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
    extern __shared__ u64 total_s[];                      // [beams x slices x take]
    __shared__ double max_s[MAX_BEAMS], log_s[MAX_BEAMS]; // log(sum exp) of a row: max + log
    __shared__ u64 warp_part[JOIN_THREADS / 32];
    __shared__ int warp_count[JOIN_THREADS / 32];
    __shared__ int pick_s[2 * MAX_TAKE + 2], order_s[MAX_TAKE + 1];
    __shared__ int count_s;
    __shared__ unsigned again_s;                          // rows whose sums are to be formed again
    const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) again_s = 0;
    __syncthreads();
    pdl_wait();
    pdl_trigger();
    for (int b = warp; b < beams; b += JOIN_THREADS / 32) {
        const size_t at = ((size_t)g * beams + b) * slices;
        float m = -INFINITY;
        for (int s = lane; s < slices; s += 32) m = fmaxf(m, maxima[at + s]);
        m = warp_max(m);
        const float r = exponent_of(m);
        double sum = 0.0;
        for (int s = lane; s < slices; s += 32) {
            const float e = exponent_of(maxima[at + s]) - r;
            if (sums[at + s] != 0.0) sum += sums[at + s] * (e < -1000.0f ? 0.0 : power_of_two(e));
        }
        sum = shfl_sum(sum);
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
    const int per_beam = slices * take, n = beams * per_beam;
    const u64* mine = keys + (size_t)g * n;
    // (the logit less the row's maximum first: both may be the lowest number there is)
    auto total_of = [&](int c) {
        const int b = c / per_beam;
        return (double)scores[(size_t)g * beams + b] +
               (((double)key_logit(mine[c]) - max_s[b]) - log_s[b]);
    };
    auto over_block = [&](auto test) {
        int k = 0;
        for (int c = tid; c < n; c += JOIN_THREADS) k += test(c) ? 1 : 0;
        k = __reduce_add_sync(0xffffffffu, k);
        __syncthreads();
        if (lane == 0) warp_count[warp] = k;
        __syncthreads();
        k = 0;
        for (int w = 0; w < JOIN_THREADS / 32; ++w) k += warp_count[w];
        return k;
    };
    auto place = [&](int c) {                 // of equal totals: beam, larger logit, lower token
        const u64 k = mine[c];
        return (u64)(c / per_beam) << 59 | (u64)(unsigned)~(unsigned)(k >> 32) << 27 |
               (unsigned)key_token(k);
    };
    // one more than is taken: what the last one taken is compared with
    const int want = take + 1, most = 2 * want;
    unsigned formed = 0;                                  // rows whose sums are 64-bit ones
    int found;
    for (;;) {
        __syncthreads();
        const unsigned again = again_s & ~formed;
        formed |= again;
        for (int b = 0; b < beams; ++b) {
            if (!(again >> b & 1)) continue;
            // terms of up to 1 as whole numbers of 2^-scale, whose sum fits 63 bits
            const int scale = min(46, 62 - (32 - __clz(vocab)));
            const double unit = __hiloint2double((1023 + scale) << 20, 0);
            const float* x = logits + ((long long)g * beams + b) * stride;
            const double m = max_s[b];
            u64 sum = 0;
            for (int i = tid; i < vocab; i += JOIN_THREADS)
                sum += (u64)__double2ll_rn(exp((double)x[i] - m) * unit);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == 0) warp_part[warp] = sum;
            __syncthreads();
            if (tid == 0) {
                sum = 0;
                for (int w = 0; w < JOIN_THREADS / 32; ++w) sum += warp_part[w];
                log_s[b] = log((double)sum / unit);
            }
            __syncthreads();
        }
        u64 top = 0;
        for (int c = tid; c < n; c += JOIN_THREADS) {
            const u64 t = mine[c] ? total_key(total_of(c)) : 0;
            total_s[c] = t;
            top = t > top ? t : top;
        }
        top = shfl_max(top);
        if (lane == 0) warp_part[warp] = top;
        if (tid == 0) count_s = 0;
        __syncthreads();
        top = 0;
        for (int w = 0; w < JOIN_THREADS / 32; ++w) top = max(top, warp_part[w]);

        // the best by their totals; of those with the total of the last place the first by `place`
        const u64 t0 = threshold(top, want, most, [&](u64 t) {
            return over_block([&](int c) { return total_s[c] >= t; });
        });
        u64 last = ~0ull;
        if (over_block([&](int c) { return total_s[c] >= t0; }) > most) {
            const int above = over_block([&](int c) { return total_s[c] > t0; });
            u64 low = 0, high = ~0ull;
            while (low < high) {
                const u64 mid = low + ((high - low) >> 1);
                const int k = over_block([&](int c) { return total_s[c] == t0 && place(c) <= mid; });
                if (above + k >= want) high = mid; else low = mid + 1;
            }
            last = high;
        }
        for (int c = tid; c < n; c += JOIN_THREADS) {
            const u64 t = total_s[c];
            if (t > t0 || (t == t0 && t != 0 && place(c) <= last)) pick_s[atomicAdd(&count_s, 1)] = c;
        }
        __syncthreads();
        found = count_s;
        for (int i = tid; i < found; i += JOIN_THREADS) {
            const int c = pick_s[i];
            int rank = 0;
            for (int j = 0; j < found; ++j) {
                const int d = pick_s[j];
                rank += total_s[d] > total_s[c] || (total_s[d] == total_s[c] && place(d) < place(c));
            }
            if (rank < want) order_s[rank] = c;
        }
        __syncthreads();
        found = min(found, want);
        // neighbours of different beams that are too near each other for the sums that they have
        if (tid + 1 < found) {
            const int c = order_s[tid], d = order_s[tid + 1];
            const unsigned rows = 1u << (c / per_beam) | 1u << (d / per_beam);
            const double a = key_total(total_s[c]), z = key_total(total_s[d]);
            if (c / per_beam != d / per_beam && (rows & ~formed) && a < INFINITY && a - z <= UNSURE)
                atomicOr(&again_s, rows);
        }
        __syncthreads();
        if (!(again_s & ~formed)) break;
    }
    for (int i = tid; i < take; i += JOIN_THREADS) {
        const size_t at = (size_t)g * take + i;
        const int c = i < found ? order_s[i] : -1;
        best[at] = c < 0 ? -INFINITY : (float)key_total(total_s[c]);
        beam[at] = c < 0 ? -1 : c / per_beam;
        token[at] = c < 0 ? -1 : key_token(mine[c]);
    }
}

// slices a row is cut into, and elements of one
struct Slicing {
    int slices, elements, per_thread;
};
constexpr int JOIN_MOST = 8192;                           // candidates of a group in shared memory
Slicing slicing(int rows, int beams, int vocab, int take) {
    const int blocks = 4 * 148;
    int slices = (vocab + 64 * SLICE_THREADS - 1) / (64 * SLICE_THREADS);
    while (rows * slices < blocks && vocab / (slices + 1) >= 4 * SLICE_THREADS) ++slices;
    const int most = JOIN_MOST / (beams * take);
    if (slices > most) slices = most < 1 ? 1 : most;
    Slicing s;
    s.elements = (vocab + slices - 1) / slices;
    s.slices = (vocab + s.elements - 1) / s.elements;
    s.per_thread = 4 * ((s.elements / 4 + 2 + SLICE_THREADS - 1) / SLICE_THREADS);
    return s;
}
size_t aligned(size_t bytes) { return (bytes + 15) & ~(size_t)15; }

// ------------------------------------------------------------------------------------------
// Reordering.  x is [layers, pool, width]; a thread owns one piece of a row's width in all rows of a
// group in one layer: it reads the pieces of every row that a moved beam takes, and only then writes,
// so the rows can change places without a buffer.
// ------------------------------------------------------------------------------------------
constexpr int MOVE_THREADS = 256;

template <typename U, int BEAMS>
__global__ void __launch_bounds__(MOVE_THREADS)
beam_reorder_kernel(unsigned char* __restrict__ x, long long row_bytes, int pool,
                    const int* __restrict__ slots, const int* __restrict__ parent, int groups,
                    int beams, int blocks_per_row, int* __restrict__ status) {
    __shared__ int from_s[BEAMS], to_s[BEAMS], slot_s[BEAMS];
    const int block = blockIdx.x % blocks_per_row;
    const int g = blockIdx.x / blocks_per_row % groups;
    const long long layer = blockIdx.x / blocks_per_row / groups;
    const int tid = threadIdx.x;
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
            bad = s < -1 || s >= pool || p >= beams;
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
    const long long at = ((long long)block * MOVE_THREADS + tid) * sizeof(U);
    if (at >= row_bytes) return;
    unsigned char* base = x + layer * pool * row_bytes + at;
    U v[BEAMS];
#pragma unroll
    for (int b = 0; b < BEAMS; ++b)
        if (from_s[b] >= 0) v[b] = *reinterpret_cast<const U*>(base + from_s[b] * row_bytes);
#pragma unroll
    for (int b = 0; b < BEAMS; ++b)
        if (from_s[b] >= 0) *reinterpret_cast<U*>(base + to_s[b] * row_bytes) = v[b];
}

template <typename U, int BEAMS>
int reorder_with(unsigned char* x, int layers, int pool, long long row_bytes, const int* slots,
                 const int* parent, int groups, int beams, int* status, cudaStream_t stream) {
    const long long per_row = (row_bytes / (long long)sizeof(U) + MOVE_THREADS - 1) / MOVE_THREADS;
    const long long blocks = per_row * groups * layers;
    if (blocks > 0x7fffffffll) return -4;
    return de_launch(beam_reorder_kernel<U, BEAMS>, dim3((unsigned)blocks), dim3(MOVE_THREADS), 0,
                     stream, x, row_bytes, pool, slots, parent, groups, beams, (int)per_row, status);
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
    if ((size_t)2 * take * s.per_thread * 8 > 200 * 1024) return -3;
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
    const int found = 2 * take * s.per_thread * 8, totals = beams * s.slices * take * 8;
    cudaError_t e = cudaSuccess;
    if (found > 32 * 1024)
        e = cudaFuncSetAttribute(beam_slices_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, found);
    if (e == cudaSuccess && totals > 32 * 1024)
        e = cudaFuncSetAttribute(beam_join_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, totals);
    if (e != cudaSuccess) return (int)e;
    const int code = de_launch(beam_slices_kernel, dim3((unsigned)n), dim3(SLICE_THREADS), found,
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
