// Attention whose requests share a prefix in true 32-bit arithmetic (shared_prefix.cu has the formulas and
// the merge): float32 on the CUDA cores, head sizes that are a multiple of 4.
//
// A block of 128 threads takes 8, 16 or 32 query rows with a range of keys, in tiles of 64.  Both products
// are tiled in registers: a thread has ROWS / 8 rows and, of the scores, four keys, of the results, four
// features in 64.  With r rows a key's element is read once from memory for r multiply-adds: few rows wait for
// the cache (4 rows behind 2,001 keys of 32 kv heads, 66 MB, 34 us), many for shared memory, whose 16-byte reads
// take four cycles of its pipe whoever shares their addresses: eight for 64 multiply-adds of the first product
// (160 rows a group behind 1,656 keys of 8 kv heads of 128, twice: 141 us, 15 TFLOP/s).  The keys of
// the next tile are copied while the values are at work and the next values while the keys are.

#include "shared_prefix.cuh"

DE_DEFINE_PDL_SWITCH

namespace {

using namespace shared_prefix;

constexpr int THREADS = 128;
constexpr int KT = 64;

__device__ __forceinline__ void copy16(float* smem, const float* gmem, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n"
                 ::"r"((unsigned)__cvta_generic_to_shared(smem)), "l"(gmem), "r"(there ? 16 : 0));
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;\n" ::); }
template <int N> __device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}

template <int RPT> __host__ __device__ constexpr int weight_stride() { return RPT == 4 ? 36 : 8 * RPT + 1; }
template <int RPT> int smem_floats(int d) {
    return 8 * RPT * d + KT * (d + 4) + KT * d + KT * weight_stride<RPT>();
}

// DMAX: 64, 128 or 256, at least d; RPT: rows of a thread
template <int DMAX, int RPT>
__global__ void __launch_bounds__(THREADS)
shared_f32_kernel(const float* __restrict__ q, int q_stride, const float* __restrict__ k_pages,
                  const float* __restrict__ v_pages, const int* __restrict__ block_table,
                  int table_stride, int num_pages, const int* __restrict__ seq_slot,
                  const int* __restrict__ seq_pos0, const Item* __restrict__ items,
                  float* __restrict__ partial_acc, float2* __restrict__ partial_ml, int heads,
                  int kv_heads, int d, int page, float scale, int order, int* __restrict__ status) {
    constexpr int ROWS = 8 * RPT, GROUPS = DMAX / 64, PS = weight_stride<RPT>();
    extern __shared__ __align__(16) float smem[];
    float* q_s = smem;                                    // [ROWS][d]
    float* k_s = q_s + ROWS * d;                          // [KT][d + 4]
    float* v_s = k_s + KT * (d + 4);                      // [KT][d]
    float* p_s = v_s + KT * d;                            // [KT][PS]
    __shared__ long long row_s[2][KT];                    // places of a tile's rows, -1 where there is none
    const Item it = items[blockIdx.x / kv_heads];
    const int hk = blockIdx.x % kv_heads, g = heads / kv_heads;
    const int tid = threadIdx.x, tr = tid >> 4, tc = tid & 15;
    const bool behind = order & BEHIND;
    if (!behind) pdl_wait();
    if (order & FOLLOWED) pdl_trigger();
    const Range range = range_of(it, seq_pos0, g, KT);
    const int slot = seq_slot[it.seq];
    const int tiles = (range.end - range.begin + KT - 1) / KT;
    const int pieces = d >> 2, ld = d + 4;

    auto look_up = [&](int t) {
        if (tid >= KT) return;
        const int key = range.begin + t * KT + tid;
        long long at = -1;
        if (t < tiles && key < range.end) {
            const int id = page_of(block_table, table_stride, num_pages, slot, key / page, status);
            if (id >= 0) at = (((long long)id * kv_heads + hk) * page + key % page) * d;
        }
        row_s[t & 1][tid] = at;
    };
    // rows of d features go by in pieces of four, a thread every 128th of them
    const int first_j = tid / pieces, first_f = tid - first_j * pieces;
    const int step_j = THREADS / pieces, step_f = THREADS - step_j * pieces;
    auto over_pieces = [&](int rows, auto each) {
        for (int j = first_j, f = first_f; j < rows;) {
            each(j, 4 * f);
            j += step_j;
            f += step_f;
            if (f >= pieces) { f -= pieces; ++j; }
        }
    };
    auto copy = [&](int t, const float* pages, float* to, int stride) {
        if (t < tiles)
            over_pieces(KT, [&](int j, int f) {
                const long long at = row_s[t & 1][j];
                copy16(to + j * stride + f, pages + (at < 0 ? 0 : at + f), at >= 0);
            });
        copies_end();
    };
    look_up(0);
    over_pieces(ROWS, [&](int row, int f) {
        const int r = it.row0 + row;
        const float* src = q + (size_t)(it.tok0 + r / g) * q_stride + (hk * g + r % g) * d + f;
        const bool live = row < it.count;
#pragma unroll
        for (int e = 0; e < 4; ++e) q_s[row * d + f + e] = live ? src[e] : 0.0f;
    });
    __syncthreads();
    copy(0, k_pages, k_s, ld);
    copy(0, v_pages, v_s, d);

    const float sl = scale * 1.4426950408889634f;
    float acc[RPT][GROUPS][4], m[RPT], l[RPT];
    int hi[RPT];
#pragma unroll
    for (int r = 0; r < RPT; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.0f;
        hi[r] = range.row_end(it, tr * RPT + r, g);
#pragma unroll
        for (int i = 0; i < GROUPS; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[r][i][e] = 0.0f;
    }
    const int min_hi = range.row_end(it, 0, g);           // up to here every row sees every key

    for (int t = 0; t < tiles; ++t) {
        const int kt = range.begin + t * KT;
        copies_wait<1>();
        __syncthreads();
        float s[RPT][4];
#pragma unroll
        for (int r = 0; r < RPT; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[r][j] = 0.0f;
#pragma unroll 4
        for (int f = 0; f < d; f += 4) {
            float4 a[RPT], b[4];
#pragma unroll
            for (int r = 0; r < RPT; ++r)
                a[r] = *reinterpret_cast<const float4*>(q_s + (tr * RPT + r) * d + f);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                b[j] = *reinterpret_cast<const float4*>(k_s + (tc + 16 * j) * ld + f);
#pragma unroll
            for (int r = 0; r < RPT; ++r)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[r][j] = fmaf(a[r].x, b[j].x, s[r][j]);
                    s[r][j] = fmaf(a[r].y, b[j].y, s[r][j]);
                    s[r][j] = fmaf(a[r].z, b[j].z, s[r][j]);
                    s[r][j] = fmaf(a[r].w, b[j].w, s[r][j]);
                }
        }
        bool there[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) there[j] = row_s[t & 1][tc + 16 * j] >= 0;
        look_up(t + 1);
#pragma unroll
        for (int r = 0; r < RPT; ++r) {
            bool seen[4];
            float top = m[r];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                seen[j] = there[j] && kt + tc + 16 * j < hi[r];
                if (!seen[j]) s[r][j] = -INFINITY;
                top = fmaxf(top, s[r][j]);
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float base = top == -INFINITY ? 0.0f : top * sl;
            const float corr = exp2f(m[r] * sl - base);
            m[r] = top;
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[r][j] = seen[j] ? exp2f(fmaf(s[r][j], sl, -base)) : 0.0f;
                sum += s[r][j];
            }
            l[r] = l[r] * corr + sum;                     // (a thread's four keys: added up at the end)
#pragma unroll
            for (int i = 0; i < GROUPS; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[r][i][e] *= corr;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float* dst = p_s + (tc + 16 * j) * PS + tr * RPT;
            if constexpr (RPT == 4) {
                *reinterpret_cast<float4*>(dst) = make_float4(s[0][j], s[1][j], s[2][j], s[3][j]);
            } else {
#pragma unroll
                for (int r = 0; r < RPT; ++r) dst[r] = s[r][j];
            }
        }
        copies_wait<0>();
        __syncthreads();
        copy(t + 1, k_pages, k_s, ld);
        const bool whole = kt + KT <= min_hi;
#pragma unroll 4
        for (int n = 0; n < KT; ++n) {
            float w[RPT];
            if constexpr (RPT == 4) {
                const float4 x = *reinterpret_cast<const float4*>(p_s + n * PS + tr * 4);
                w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
            } else {
#pragma unroll
                for (int r = 0; r < RPT; ++r) w[r] = p_s[n * PS + tr * RPT + r];
            }
#pragma unroll
            for (int i = 0; i < GROUPS; ++i) {
                const int f = 4 * tc + 64 * i;
                if (f >= d) continue;
                const float4 v = *reinterpret_cast<const float4*>(v_s + n * d + f);
#pragma unroll
                for (int r = 0; r < RPT; ++r) {
                    // (a value that is not finite must not reach a row that does not see its key)
                    if (!whole && kt + n >= hi[r]) continue;
                    acc[r][i][0] = fmaf(w[r], v.x, acc[r][i][0]);
                    acc[r][i][1] = fmaf(w[r], v.y, acc[r][i][1]);
                    acc[r][i][2] = fmaf(w[r], v.z, acc[r][i][2]);
                    acc[r][i][3] = fmaf(w[r], v.w, acc[r][i][3]);
                }
            }
        }
        __syncthreads();
        copy(t + 1, v_pages, v_s, d);
    }
    copies_wait<0>();
    pdl_trigger();
#pragma unroll
    for (int r = 0; r < RPT; ++r) {
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], o);
        const int row = tr * RPT + r;
        if (row >= it.count) continue;
        const size_t at = (size_t)(it.base + row) * kv_heads + hk;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            const int f = 4 * tc + 64 * i;
            if (f < d)
                *reinterpret_cast<float4*>(partial_acc + at * d + f) =
                    make_float4(acc[r][i][0], acc[r][i][1], acc[r][i][2], acc[r][i][3]);
        }
        if (tc == 0) partial_ml[at] = make_float2(m[r] * sl, l[r]);
    }
    if (behind) pdl_wait();
}

template <int DMAX, int RPT>
int launch(const float* q, int q_stride, const float* k_pages, const float* v_pages,
           const int* block_table, int table_stride, int num_pages, const int* seq_slot,
           const int* seq_pos0, const int* items, int num_items, int order, float* partial_acc,
           float* partial_ml, int heads, int kv_heads, int d, int page, float scale, int* status,
           cudaStream_t stream) {
    const int smem = smem_floats<RPT>(d) * 4;
    if (smem > 40 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(
            shared_f32_kernel<DMAX, RPT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return (int)e;
    }
    return de_launch(shared_f32_kernel<DMAX, RPT>, dim3((unsigned)num_items * kv_heads), dim3(THREADS),
                     smem, stream, q, q_stride, k_pages, v_pages, block_table, table_stride, num_pages,
                     seq_slot, seq_pos0, (const Item*)items, partial_acc, (float2*)partial_ml, heads,
                     kv_heads, d, page, scale, order, status);
}

}  // namespace

DE_EXPORT int de_shared_f32_unit() { return KT; }
// blocks of `rows` (8, 16, 32) query rows that an SM holds at once; 0: not a size that is taken
DE_EXPORT int de_shared_f32_held(int rows, int head_dim) {
    if (head_dim < 4 || head_dim > 256 || head_dim % 4 || (rows != 8 && rows != 16 && rows != 32)) return 0;
    const int bytes = 4 * (rows == 8 ? smem_floats<1>(head_dim) : rows == 16 ? smem_floats<2>(head_dim)
                                                                             : smem_floats<4>(head_dim));
    const int blocks = 227 * 1024 / (bytes + 2048);
    return blocks > 6 ? 6 : blocks;
}

// Items of up to `rows` rows; pages in 16-byte pieces; `order` as in shared_prefix.cu.
DE_EXPORT int de_shared_f32(const float* q, int q_stride, const float* k_pages, const float* v_pages,
                            const int* block_table, int table_stride, int num_pages,
                            const int* seq_slot, const int* seq_pos0, const int* items, int num_items,
                            int rows, int order, float* partial_acc, float* partial_ml, int heads,
                            int kv_heads, int head_dim, int page, float scale, int* status,
                            void* stream) {
    if (num_items <= 0) return 0;
    if (de_shared_f32_held(rows, head_dim) < 1 || kv_heads < 1 || heads % kv_heads || page < 1 ||
        (long long)num_items * kv_heads > 0x7fffffffll)
        return -2;
    if (((uintptr_t)k_pages & 15) || ((uintptr_t)v_pages & 15)) return -3;
    const int sizes = head_dim <= 64 ? 0 : head_dim <= 128 ? 1 : 2;
    const auto f = rows == 8    ? (sizes == 0 ? launch<64, 1> : sizes == 1 ? launch<128, 1> : launch<256, 1>)
                   : rows == 16 ? (sizes == 0 ? launch<64, 2> : sizes == 1 ? launch<128, 2> : launch<256, 2>)
                                : (sizes == 0 ? launch<64, 4> : sizes == 1 ? launch<128, 4> : launch<256, 4>);
    return f(q, q_stride, k_pages, v_pages, block_table, table_stride, num_pages, seq_slot, seq_pos0, items,
             num_items, order, partial_acc, partial_ml, heads, kv_heads, head_dim, page, scale, status,
             (cudaStream_t)stream);
}
