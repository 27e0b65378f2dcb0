// Attention over the paged cache for steps whose requests share a long prefix: beams of one prompt,
// answers drawn to one document, requests behind one system prompt.
//
//   A request's keys are its group's prefix (positions 0 .. P - 1, in pages that the group's
//   requests share, read through the first one's table) and its own keys behind it.  With
//   s_j = scale q . k_j, a row's result is sum_j exp(s_j) v_j / sum_j exp(s_j) over both.
//
// The prefix is worked through once for all rows of the group: the tokens of its requests are
// consecutive in the step, so the rows (token, query head of a kv head's group) of the whole group
// form tiles that see every key of the prefix.  Each request's own keys are worked through for its
// own rows, causally.  Every tile leaves, for a range of keys, a maximum m, a sum l of exp(s - m)
// and the sum of exp(s - m) v; `merge` joins what belongs to a row:
//   M = max m_i,   out = sum_i exp(m_i - M) acc_i / sum_i exp(m_i - M) l_i.
//
// This file has the kernel for all types and even head sizes, in float32 on the CUDA cores, and the
// merge.  Softmax weights as in src/layers/attention.py:35-71.

#include "shared_prefix.cuh"

DE_DEFINE_PDL_SWITCH

namespace {

using namespace shared_prefix;

constexpr int ROWS = 8;               // query rows of a block
constexpr int KT = 32;                // keys of a tile
constexpr int THREADS = 128;
constexpr int MERGE_MOST = 1024;       // partial results of a row
constexpr int MERGE_FEW = 8;           // of them a warp reads alone

// A block takes eight rows of an item (blockIdx.y: which), a warp two.  Scores: a lane a key;
// results: a lane every 32nd feature.
template <typename T>
__global__ void __launch_bounds__(THREADS)
shared_rows_kernel(const T* __restrict__ q, int q_stride, const T* __restrict__ k_pages,
                   const T* __restrict__ v_pages, const int* __restrict__ block_table,
                   int table_stride, int num_pages, const int* __restrict__ seq_slot,
                   const int* __restrict__ seq_pos0, const Item* __restrict__ items,
                   float* __restrict__ partial_acc, float2* __restrict__ partial_ml, int heads,
                   int kv_heads, int d, int page, float scale, int unit, int order,
                   int* __restrict__ status) {
    extern __shared__ float smem[];
    const int ld = d + 1;
    float* q_s = smem;                                    // [ROWS][d]
    float* k_s = q_s + ROWS * d;                          // [KT][ld]
    float* v_s = k_s + KT * ld;                           // [KT][ld]
    __shared__ long long offset_s[KT];
    const Item it = items[blockIdx.x / kv_heads];
    const int hk = blockIdx.x % kv_heads, g = heads / kv_heads;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int first = blockIdx.y * ROWS;                  // of the tile's rows
    const bool behind = order & BEHIND;
    if (!behind) pdl_wait();
    if (order & FOLLOWED) pdl_trigger();
    if (first >= it.count) {
        if (behind) pdl_wait();
        return;
    }
    const Range range = range_of(it, seq_pos0, g, unit);
    const int slot = seq_slot[it.seq];
    for (int i = tid; i < ROWS * d; i += THREADS) {
        const int r = it.row0 + first + i / d;
        q_s[i] = first + i / d < it.count ? to_float(q[(size_t)(it.tok0 + r / g) * q_stride +
                                          (hk * g + r % g) * d + i % d])
                             : 0.0f;
    }
    const float sl = scale * 1.4426950408889634f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    float acc[2][8];
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[r][i] = 0.0f;
    int hi[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) hi[r] = range.row_end(it, first + 2 * warp + r, g);

    for (int kt = range.begin; kt < range.end; kt += KT) {
        __syncthreads();
        if (tid < KT) {
            const int key = kt + tid;
            long long at = -1;
            if (key < range.end) {
                const int id = page_of(block_table, table_stride, num_pages, slot, key / page, status);
                if (id >= 0) at = (((long long)id * kv_heads + hk) * page + key % page) * d;
            }
            offset_s[tid] = at;
        }
        __syncthreads();
        for (int i = tid; i < KT * d; i += THREADS) {
            const int j = i / d, f = i % d;
            const long long at = offset_s[j];
            k_s[j * ld + f] = at >= 0 ? to_float(k_pages[at + f]) : 0.0f;
            v_s[j * ld + f] = at >= 0 ? to_float(v_pages[at + f]) : 0.0f;
        }
        __syncthreads();
        const bool there = offset_s[lane] >= 0;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const float* qr = q_s + (2 * warp + r) * d;
            float s = 0.0f;
            for (int f = 0; f < d; ++f) s = fmaf(qr[f], k_s[lane * ld + f], s);
            const bool seen = there && kt + lane < hi[r];
            if (!seen) s = -INFINITY;
            const float top = fmaxf(m[r], warp_max(s));
            const float base = top == -INFINITY ? 0.0f : top * sl;
            const float p = seen ? exp2f(s * sl - base) : 0.0f;
            const float corr = exp2f(m[r] * sl - base);
            l[r] = l[r] * corr + warp_sum(p);
            m[r] = top;
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[r][i] *= corr;
            unsigned seen_keys = __ballot_sync(0xffffffffu, seen);
            while (seen_keys) {
                const int j = __ffs(seen_keys) - 1;
                seen_keys &= seen_keys - 1;
                const float w = __shfl_sync(0xffffffffu, p, j);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int f = lane + 32 * i;
                    if (f < d) acc[r][i] = fmaf(w, v_s[j * ld + f], acc[r][i]);
                }
            }
        }
    }
    pdl_trigger();
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int row = first + 2 * warp + r;
        if (row >= it.count) continue;
        const size_t at = (size_t)(it.base + row) * kv_heads + hk;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int f = lane + 32 * i;
            if (f < d) partial_acc[at * d + f] = acc[r][i];
        }
        if (lane == 0) {
            partial_ml[at] = make_float2(m[r] * sl, l[r]);
            if (has_second_place(it))
                partial_ml[at + (size_t)HALF_ROWS * kv_heads] = make_float2(-INFINITY, 0.0f);
        }
    }
    if (behind) pdl_wait();
}

// WARPS warps a (token, query head).  The threads take the partial results' maxima and sums in turn,
// which gives each its weight; then the weighted results are summed, LANES lanes a result (a lane four
// features at a time where VEC) and several results at once.
template <typename T, int WARPS, int LANES, bool VEC>
__global__ void __launch_bounds__(128)
shared_merge_kernel(T* __restrict__ out, int out_stride, const int* __restrict__ token_seq,
                    const Joined* __restrict__ seqs, const float* __restrict__ partial_acc,
                    const float2* __restrict__ partial_ml, int heads, int kv_heads, int d) {
    constexpr int UNITS = 4 / WARPS, GROUP = 32 * WARPS, AT_ONCE = GROUP / LANES;
    constexpr int N = VEC ? 4 : 8, DEEP = VEC ? 4 : 1;
    __shared__ float weight_s[UNITS][WARPS == 1 ? MERGE_FEW : MERGE_MOST];
    __shared__ float top_s[4], total_s[4];
    __shared__ float sum_s[WARPS == 1 ? 1 : 4][WARPS == 1 ? 1 : (VEC ? 4 * LANES : 256)];
    const int unit = threadIdx.x / GROUP, tid = threadIdx.x % GROUP;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int token = blockIdx.x, h = blockIdx.y * UNITS + unit;
    const bool there = h < heads;                         // (with one warp a unit; else all are)
    const int g = heads / kv_heads, hk = (there ? h : 0) / g;
    const Joined s = seqs[token_seq[token]];
    // the results of a row lie a tile's rows apart: the prefix's, then its own keys'
    const int row_p = (token - s.group_tok0) * g + h % g, row_o = (token - s.tok0) * g + h % g;
    const int parts = s.prefix_chunks + s.own_chunks;
    size_t at_p = 0, at_o = 0;
    if (s.prefix_chunks)
        at_p = (size_t)(s.prefix_base + row_p / s.prefix_rows * s.prefix_chunks * s.prefix_rows +
                        row_p % s.prefix_rows) * kv_heads + hk;
    if (s.own_chunks)
        at_o = (size_t)(s.own_base + row_o / s.own_rows * s.own_chunks * s.own_rows +
                        row_o % s.own_rows) * kv_heads + hk;
    auto place = [&](int c) {
        return c < s.prefix_chunks
                   ? at_p + (size_t)c * s.prefix_rows * kv_heads
                   : at_o + (size_t)(c - s.prefix_chunks) * s.own_rows * kv_heads;
    };
    pdl_wait();
    pdl_trigger();
    if (!there) return;
    // (what a thread reads first it keeps: there are seldom more results than threads)
    float2 first = make_float2(-INFINITY, 0.0f);
    if (tid < parts) first = partial_ml[place(tid)];
    float top = first.x;
    for (int c = tid + GROUP; c < parts; c += GROUP) top = fmaxf(top, partial_ml[place(c)].x);
    top = warp_max(top);
    if (WARPS > 1) {
        if (lane == 0) top_s[warp] = top;
        __syncthreads();
        top = fmaxf(fmaxf(top_s[0], top_s[1]), fmaxf(top_s[2], top_s[3]));
    }
    if (top == -INFINITY) top = 0.0f;
    float total = 0.0f;
    for (int c = tid; c < parts; c += GROUP) {
        const float2 ml = c == tid ? first : partial_ml[place(c)];
        // (a range without a key has left no result; one of NaN scores only has a sum that is NaN)
        const bool empty = ml.x == -INFINITY && ml.y == 0.0f;
        const float w = empty ? 0.0f : exp2f(ml.x - top);
        total += empty ? 0.0f : w * ml.y;
        weight_s[unit][c] = empty ? -1.0f : w;
    }
    total = warp_sum(total);
    if (WARPS > 1) {
        if (lane == 0) total_s[warp] = total;
        __syncthreads();
        total = (total_s[0] + total_s[1]) + (total_s[2] + total_s[3]);
    } else {
        __syncwarp();
    }
    const int sub = tid % LANES;
    float acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.0f;
    for (int c0 = tid / LANES; c0 < parts; c0 += AT_ONCE * DEEP) {
        if constexpr (VEC) {
            float4 v[DEEP];
            float w[DEEP];
#pragma unroll
            for (int k = 0; k < DEEP; ++k) {
                const int c = c0 + k * AT_ONCE;
                w[k] = c < parts ? weight_s[unit][c] : -1.0f;
                if (w[k] != -1.0f)
                    v[k] = *reinterpret_cast<const float4*>(partial_acc + place(c) * d + 4 * sub);
            }
#pragma unroll
            for (int k = 0; k < DEEP; ++k) {
                if (w[k] == -1.0f) continue;
                acc[0] = fmaf(w[k], v[k].x, acc[0]);
                acc[1] = fmaf(w[k], v[k].y, acc[1]);
                acc[2] = fmaf(w[k], v[k].z, acc[2]);
                acc[3] = fmaf(w[k], v[k].w, acc[3]);
            }
        } else {
            const float w = weight_s[unit][c0];
            if (w == -1.0f) continue;
            const size_t at = place(c0);
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (sub + LANES * i < d) acc[i] = fmaf(w, partial_acc[at * d + sub + LANES * i], acc[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int o = LANES; o < 32; o <<= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    T* dst = out + (size_t)token * out_stride + h * d;
    if constexpr (WARPS == 1) {
        if (tid >= LANES) return;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int f = VEC ? 4 * sub + i : sub + LANES * i;
            if (f < d) dst[f] = from_float<T>(acc[i] * inv);
        }
    } else {
        if (lane < LANES) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int f = VEC ? 4 * sub + i : sub + LANES * i;
                if (f < d) sum_s[warp][f] = acc[i];
            }
        }
        __syncthreads();
        for (int f = tid; f < d; f += GROUP)
            dst[f] = from_float<T>(((sum_s[0][f] + sum_s[1][f]) + (sum_s[2][f] + sum_s[3][f])) * inv);
    }
}

// A warp alone reads up to MERGE_FEW results a row, four at once or eight; more are shared out over four
// warps.  (us for all launches, a warp and four: 16 requests behind 4,096 keys, 32 heads of 64, 65 results a
// row, 25.2 and 14.4; four beams behind 512 keys, nine results, 7.5 and 7.2; 64 requests behind 16 prompts of
// 1,003 keys, five results, 55.5 and 57.5.)
template <typename T, int WARPS>
int merge_with(void* out, int out_stride, const int* token_seq, const int* seqs, const float* partial_acc,
               const float* partial_ml, int tokens, int heads, int kv_heads, int d, cudaStream_t stream) {
    const auto kernel = d == 128  ? shared_merge_kernel<T, WARPS, 32, true>
                        : d == 64 ? shared_merge_kernel<T, WARPS, 16, true>
                                  : shared_merge_kernel<T, WARPS, 32, false>;
    const int units = 4 / WARPS;
    return de_launch(kernel, dim3((unsigned)tokens, (heads + units - 1) / units), dim3(128), 0, stream,
                     (T*)out, out_stride, token_seq, (const Joined*)seqs, partial_acc,
                     (const float2*)partial_ml, heads, kv_heads, d);
}
template <typename T>
int merge_of(void* out, int out_stride, const int* token_seq, const int* seqs, const float* partial_acc,
             const float* partial_ml, int most, int tokens, int heads, int kv_heads, int d,
             cudaStream_t stream) {
    const auto f = most <= MERGE_FEW ? merge_with<T, 1> : merge_with<T, 4>;
    return f(out, out_stride, token_seq, seqs, partial_acc, partial_ml, tokens, heads, kv_heads, d, stream);
}

template <typename T>
int rows_of(const void* q, int q_stride, const void* k_pages, const void* v_pages,
            const int* block_table, int table_stride, int num_pages, const int* seq_slot,
            const int* seq_pos0, const int* items, int num_items, int tile_rows, int unit,
            int order, float* partial_acc, float* partial_ml, int heads, int kv_heads, int d, int page,
            float scale, int* status, cudaStream_t stream) {
    const int smem = (ROWS * d + 2 * KT * (d + 1)) * 4;
    if (smem > 40 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(
            shared_rows_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return (int)e;
    }
    return de_launch(shared_rows_kernel<T>, dim3((unsigned)num_items * kv_heads, (tile_rows + ROWS - 1) / ROWS),
                     dim3(THREADS), smem, stream, (const T*)q, q_stride, (const T*)k_pages,
                     (const T*)v_pages, block_table, table_stride, num_pages, seq_slot, seq_pos0, (const Item*)items, partial_acc,
                     (float2*)partial_ml, heads, kv_heads, d, page, scale, unit, order, status);
}

}  // namespace

// `tile_rows`: most rows of an item; `unit`: what the ranges of own keys are a multiple of; `order`:
// 1 where the launch before this one is another of the same step's, 2 where the next one is.
DE_EXPORT int de_shared_rows(int dtype, const void* q, int q_stride, const void* k_pages,
                             const void* v_pages, const int* block_table, int table_stride,
                             int num_pages, const int* seq_slot, const int* seq_pos0,
                             const int* items, int num_items, int tile_rows, int unit,
                             int order, float* partial_acc, float* partial_ml, int heads, int kv_heads,
                             int head_dim, int page, float scale, int* status, void* stream) {
    if (num_items <= 0) return 0;
    if (tile_rows < 1 || tile_rows > 1024 || unit < 1) return -3;
    if (head_dim < 2 || head_dim > 256 || head_dim % 2 || kv_heads < 1 || heads % kv_heads || page < 1 ||
        (long long)num_items * kv_heads > 0x7fffffffll)
        return -2;
    const auto f = dtype == DE_F32 ? rows_of<float> : rows_of<__nv_bfloat16>;
    return f(q, q_stride, k_pages, v_pages, block_table, table_stride, num_pages, seq_slot, seq_pos0,
             items, num_items, tile_rows, unit, order, partial_acc, partial_ml, heads, kv_heads,
             head_dim, page, scale, status, (cudaStream_t)stream);
}

// `most`: partial results of a row, at most (up to 1,024).
DE_EXPORT int de_shared_merge(int dtype, void* out, int out_stride, const int* token_seq,
                              const int* seqs, const float* partial_acc, const float* partial_ml,
                              int most, int tokens, int heads, int kv_heads, int head_dim,
                              void* stream) {
    if (tokens <= 0) return 0;
    if (most < 0 || most > MERGE_MOST || heads > 262140) return -3;
    if (head_dim < 2 || head_dim > 256 || head_dim % 2 || kv_heads < 1 || heads % kv_heads) return -2;
    const auto f = dtype == DE_F32 ? merge_of<float> : merge_of<__nv_bfloat16>;
    return f(out, out_stride, token_seq, seqs, partial_acc, partial_ml, most, tokens, heads, kv_heads,
             head_dim, (cudaStream_t)stream);
}
