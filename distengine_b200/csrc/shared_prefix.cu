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

// A block takes eight rows of an item (blockIdx.y: which), a warp two.  Scores: a lane a key;
// results: a lane every 32nd feature.
template <typename T>
__global__ void __launch_bounds__(THREADS)
shared_rows_kernel(const T* __restrict__ q, int q_stride, const T* __restrict__ k_pages,
                   const T* __restrict__ v_pages, const int* __restrict__ block_table,
                   int table_stride, int num_pages, const int* __restrict__ seq_slot,
                   const int* __restrict__ seq_pos0, const Item* __restrict__ items,
                   float* __restrict__ partial_acc, float2* __restrict__ partial_ml, int heads,
                   int kv_heads, int d, int page, float scale, int unit, int behind,
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
    if (!behind) pdl_wait();
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

// A warp a (token, query head): the lanes take the partial results' maxima and sums in turn, then
// all of them the features of one partial result after the other.
template <typename T>
__global__ void __launch_bounds__(128)
shared_merge_kernel(T* __restrict__ out, int out_stride, const int* __restrict__ token_seq,
                    const Joined* __restrict__ seqs, const float* __restrict__ partial_acc,
                    const float2* __restrict__ partial_ml, int tokens, int heads, int kv_heads,
                    int d) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long unit = (long long)blockIdx.x * 4 + warp;
    pdl_wait();
    pdl_trigger();
    if (unit >= (long long)tokens * heads) return;
    const int token = (int)(unit / heads), h = (int)(unit % heads);
    const int g = heads / kv_heads, hk = h / g;
    const Joined s = seqs[token_seq[token]];
    const int parts = s.prefix_chunks + s.own_chunks;
    auto place = [&](int c) {
        const bool shared = c < s.prefix_chunks;
        const int row = (token - (shared ? s.group_tok0 : s.tok0)) * g + h % g;
        const int tile = shared ? s.prefix_rows : s.own_rows;
        const int chunks = shared ? s.prefix_chunks : s.own_chunks;
        const int base = shared ? s.prefix_base : s.own_base;
        const int chunk = shared ? c : c - s.prefix_chunks;
        return (size_t)(base + (row / tile * chunks + chunk) * tile + row % tile) * kv_heads + hk;
    };
    float top = -INFINITY;
    for (int c = lane; c < parts; c += 32) top = fmaxf(top, partial_ml[place(c)].x);
    top = warp_max(top);
    if (top == -INFINITY) top = 0.0f;
    float total = 0.0f;
    for (int c = lane; c < parts; c += 32) {
        const float2 ml = partial_ml[place(c)];
        total += exp2f(ml.x - top) * ml.y;
    }
    total = warp_sum(total);
    float acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
    for (int c = 0; c < parts; ++c) {
        const size_t at = place(c);
        const float2 ml = partial_ml[at];
        if (ml.x == -INFINITY && ml.y == 0.0f) continue;             // no key in this range
        const float w = exp2f(ml.x - top);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int f = lane + 32 * i;
            if (f < d) acc[i] = fmaf(w, partial_acc[at * d + f], acc[i]);
        }
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int f = lane + 32 * i;
        if (f < d) out[(size_t)token * out_stride + h * d + f] = from_float<T>(acc[i] * inv);
    }
}

template <typename T>
int rows_of(const void* q, int q_stride, const void* k_pages, const void* v_pages,
            const int* block_table, int table_stride, int num_pages, const int* seq_slot,
            const int* seq_pos0, const int* items, int num_items, int tile_rows, int unit,
            int behind, float* partial_acc, float* partial_ml, int heads, int kv_heads, int d, int page,
            float scale, int* status, cudaStream_t stream) {
    const int smem = (ROWS * d + 2 * KT * (d + 1)) * 4;
    if (smem > 40 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(
            shared_rows_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return (int)e;
    }
    return de_launch(shared_rows_kernel<T>, dim3((unsigned)num_items * kv_heads, (tile_rows + ROWS - 1) / ROWS),
                     dim3(THREADS), smem, stream, (const T*)q, q_stride, (const T*)k_pages, (const T*)v_pages, block_table,
                     table_stride, num_pages, seq_slot, seq_pos0, (const Item*)items, partial_acc,
                     (float2*)partial_ml, heads, kv_heads, d, page, scale, unit, behind, status);
}

}  // namespace

// `tile_rows`: most rows of an item; `unit`: what the ranges of own keys are a multiple of; `behind`:
// the launch before this one is another of the same step's (see shared_prefix.cuh).
DE_EXPORT int de_shared_rows(int dtype, const void* q, int q_stride, const void* k_pages,
                             const void* v_pages, const int* block_table, int table_stride,
                             int num_pages, const int* seq_slot, const int* seq_pos0,
                             const int* items, int num_items, int tile_rows, int unit,
                             int behind, float* partial_acc, float* partial_ml, int heads, int kv_heads,
                             int head_dim, int page, float scale, int* status, void* stream) {
    if (num_items <= 0) return 0;
    if (tile_rows < 1 || tile_rows > 1024 || unit < 1) return -3;
    if (head_dim < 2 || head_dim > 256 || head_dim % 2 || kv_heads < 1 || heads % kv_heads || page < 1 ||
        (long long)num_items * kv_heads > 0x7fffffffll)
        return -2;
    const auto f = dtype == DE_F32 ? rows_of<float> : rows_of<__nv_bfloat16>;
    return f(q, q_stride, k_pages, v_pages, block_table, table_stride, num_pages, seq_slot, seq_pos0,
             items, num_items, tile_rows, unit, behind, partial_acc, partial_ml, heads, kv_heads, head_dim, page, scale, status,
             (cudaStream_t)stream);
}

DE_EXPORT int de_shared_merge(int dtype, void* out, int out_stride, const int* token_seq,
                              const int* seqs, const float* partial_acc, const float* partial_ml,
                              int tokens, int heads, int kv_heads, int head_dim, void* stream) {
    if (tokens <= 0) return 0;
    if (head_dim < 2 || head_dim > 256 || head_dim % 2 || kv_heads < 1 || heads % kv_heads) return -2;
    const dim3 grid((unsigned)(((long long)tokens * heads + 3) / 4)), block(128);
    if (dtype == DE_F32)
        return de_launch(shared_merge_kernel<float>, grid, block, 0, (cudaStream_t)stream, (float*)out,
                         out_stride, token_seq, (const Joined*)seqs, partial_acc,
                         (const float2*)partial_ml, tokens, heads, kv_heads, head_dim);
    return de_launch(shared_merge_kernel<__nv_bfloat16>, grid, block, 0, (cudaStream_t)stream,
                     (__nv_bfloat16*)out, out_stride, token_seq, (const Joined*)seqs, partial_acc,
                     (const float2*)partial_ml, tokens, heads, kv_heads, head_dim);
}
