// Attention whose requests share a prefix, on the tensor cores by mma.sync (shared_prefix.cu has the
// formulas and the merge): bfloat16, float32 softmax.  Compiled once per head size (-DHEAD_DIM=d).
//
// An item is up to 16 query rows with a range of keys: the keys of one request for its own rows
// (few rows, every key read once), or a prefix for the rows of a small group.  Both are bound by the
// keys' and values' way from memory.  A warp takes an item and kv head alone, in tiles of 16 keys with a
// ring of tiles of its own, so no warp waits for another; the host cuts the ranges so that all warps
// that the device holds have one.  (Four warps a range, joined in shared memory, for ranges above 256 keys:
// 16 prompts x 4 beams 73 us instead of 56, 64 requests with 500 own keys behind 8,192 57 instead of 49.)
//
// A row's exponentials refer to a maximum that is raised only when a score has grown by more than 2^8
// beyond it (the quotient does not depend on it), so most tiles need no exchange between lanes and no
// rescaling of the results.
// Weights enter the second product as bfloat16, which its operands are (half a step of 2^-8 each); their sum is
// of the float32 ones.

#include "shared_prefix.cuh"

DE_DEFINE_PDL_SWITCH

#include "attention_mma_common.cuh"

namespace {

using namespace shared_prefix;

constexpr int WARPS = THREADS / 32;
constexpr int NK = 16;                                    // keys of a warp's tile
constexpr int DT = D / 8;
constexpr int CHUNKS = D / 8;                             // 16-byte pieces of a key's row
constexpr int STAGE = 2 * NK * LDS;                       // keys and values of a tile, in elements
constexpr float RAISE = 8.0f;

constexpr int ROWS = 16;                                  // of a warp
constexpr int STAGES = 2;                                 // tiles of a warp in flight or in use
constexpr int SMEM = WARPS * STAGES * STAGE * 2;
constexpr int BLOCKS = 227 * 1024 / (SMEM + 1024) < 4 ? 227 * 1024 / (SMEM + 1024) : 4;      // an SM holds

__device__ __forceinline__ bool odd_pair(unsigned x) {    // an infinity or NaN among two bfloat16
    return (x & 0x7f80u) == 0x7f80u || (x & 0x7f800000u) == 0x7f800000u;
}

__global__ void __launch_bounds__(THREADS)
shared_mma_kernel(const __nv_bfloat16* __restrict__ q, int q_stride,
                  const __nv_bfloat16* __restrict__ k_pages,
                  const __nv_bfloat16* __restrict__ v_pages, const int* __restrict__ block_table,
                  int table_stride, int num_pages, const int* __restrict__ seq_slot,
                  const int* __restrict__ seq_pos0, const Item* __restrict__ items, int num_items,
                  float* __restrict__ partial_acc, float2* __restrict__ partial_ml, int heads,
                  int kv_heads, int page, float scale, int order, int* __restrict__ status) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int gid = lane >> 2, tig = lane & 3;
    const int g = heads / kv_heads;
    const bool behind = order & BEHIND;
    const long long place = (long long)blockIdx.x * WARPS + warp;
    if (place >= (long long)num_items * kv_heads) {       // (a warp of the last block)
        pdl_wait();
        return;
    }
    Item it = items[place / kv_heads];
    const int hk = (int)(place % kv_heads);
    __nv_bfloat16* ring = reinterpret_cast<__nv_bfloat16*>(smem_raw) + warp * STAGES * STAGE;
    const bool second = has_second_place(it);
    if (!behind) pdl_wait();
    if (order & FOLLOWED) pdl_trigger();
    const Range range = range_of(it, seq_pos0, g, NK);
    // of an item with more rows than a warp takes, the warp's
    it.row0 += blockIdx.y * ROWS;
    it.base += blockIdx.y * ROWS;
    it.count = min(ROWS, it.count - (int)blockIdx.y * ROWS);
    if (it.count <= 0) {
        if (behind) pdl_wait();
        return;
    }

    const int slot = seq_slot[it.seq];
    const int tiles = (range.end - range.begin + NK - 1) / NK;

    // A tile's pages: lane j looks the page of key j up, a tile ahead of its copies.  The place of a
    // key's row in units of rows of D features, or -1.
    auto look_up = [&](int i) {
        const int key = range.begin + i * NK + (lane & 15);
        long long at = -1;
        if (lane < 16 && i < tiles && key < range.end) {
            const int id = page_of(block_table, table_stride, num_pages, slot, key / page, status);
            if (id >= 0) at = ((long long)id * kv_heads + hk) * page + key % page;
        }
        return at;
    };
    // which keys of a tile are there, as bits
    auto copy = [&](int i, long long at) {
        const unsigned there = __ballot_sync(0xffffffffu, at >= 0) & 0xffffu;
        __nv_bfloat16* k_s = ring + (i % STAGES) * STAGE;
        __nv_bfloat16* v_s = k_s + NK * LDS;
#pragma unroll
        for (int c = 0; c < NK * CHUNKS / 32; ++c) {
            const int piece = lane + 32 * c, j = piece / CHUNKS, ch = piece % CHUNKS;
            const long long row = __shfl_sync(0xffffffffu, at, j);
            const size_t off = row < 0 ? 0 : (size_t)row * D + ch * 8;
            cp_async16(k_s + j * LDS + ch * 8, k_pages + off, row >= 0);
            cp_async16(v_s + j * LDS + ch * 8, v_pages + off, row >= 0);
        }
        return there;
    };

    unsigned there[STAGES];                               // of the tiles in the ring
    long long next = look_up(0);
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) {
        const long long at = next;
        next = look_up(i + 1);
        there[i] = i < tiles ? copy(i, at) : 0;
        cp_async_commit();
    }

    // the rows of this thread: gid and gid + 8 of each row tile
    unsigned qf[D / 16][4];
    int hi[2];
    int min_hi = range.end;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int row = 8 * i + gid, r = it.row0 + row;
        const bool ok = row < it.count;
        const __nv_bfloat16* p = q + (size_t)(it.tok0 + (ok ? r / g : 0)) * q_stride +
                                 (hk * g + (ok ? r % g : 0)) * D + 2 * tig;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
            qf[kk][i] = ok ? *reinterpret_cast<const unsigned*>(p + kk * 16) : 0u;
            qf[kk][i + 2] = ok ? *reinterpret_cast<const unsigned*>(p + kk * 16 + 8) : 0u;
        }
        hi[i] = range.row_end(it, row, g);
        if (ok) min_hi = min(min_hi, hi[i]);
    }
    min_hi = __reduce_min_sync(0xffffffffu, min_hi);      // up to here every row sees every key

    const float sl = scale * 1.4426950408889634f;
    float o_acc[DT][4], m_ref[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < DT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o_acc[j][e] = 0.0f;

    for (int i = 0; i < tiles; ++i) {
        {   // the tile STAGES - 1 ahead, into the place of the one that is done
            const long long at = next;
            next = look_up(i + STAGES);
            unsigned bits = 0;
            if (i + STAGES - 1 < tiles) bits = copy(i + STAGES - 1, at);
            cp_async_commit();
            there[STAGES - 1] = bits;
        }
        cp_async_wait<STAGES - 1>();
        __syncwarp();
        const __nv_bfloat16* kb = ring + (i % STAGES) * STAGE;
        __nv_bfloat16* vb = ring + (i % STAGES) * STAGE + NK * LDS;
        const int kt = range.begin + i * NK;
        const int mat = lane >> 3, mr = lane & 7;

        float s[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[j][e] = 0.0f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
            unsigned b[4];
            ldmatrix_x4(b, kb + ((mat >> 1) * 8 + mr) * LDS + kk * 16 + (mat & 1) * 8);
            mma_bf16(s[0], qf[kk], b[0], b[1]);
            mma_bf16(s[1], qf[kk], b[2], b[3]);
        }
        const unsigned here = there[0];
        const bool whole = kt + NK <= min_hi;             // no row's limit is in this tile
        if (!whole || here != 0xffffu) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int key = j * 8 + 2 * tig + (e & 1);
                    if (!(here >> key & 1) || kt + key >= hi[e >> 1]) s[j][e] = -INFINITY;
                }
        }
        // raise the references that a score has left behind
        bool raise = false;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 2; ++r)
                raise |= (fmaxf(s[j][2 * r], s[j][2 * r + 1]) - m_ref[r]) * sl > RAISE;
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float m = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                m = fmaxf(m, m_ref[r]);
                const float f = m == m_ref[r] ? 1.0f : fast_exp2((m_ref[r] - m) * sl);
                m_ref[r] = m;
                l_run[r] *= f;
#pragma unroll
                for (int j = 0; j < DT; ++j) {
                    o_acc[j][2 * r] *= f;
                    o_acc[j][2 * r + 1] *= f;
                }
            }
        }
        // weights; the sum takes them before they are rounded to bfloat16 for their product
        unsigned pf[4];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const float base = m_ref[r] == -INFINITY ? 0.0f : m_ref[r] * sl;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float a = fast_exp2(fmaf(s[j][2 * r], sl, -base));
                const float b = fast_exp2(fmaf(s[j][2 * r + 1], sl, -base));
                l_run[r] += a + b;
                pf[2 * j + r] = pack_bf16(a, b);
            }
        }
        // A value that is not finite would reach rows that do not see its key (0 * inf is NaN): where
        // a tile has keys that only some rows see, such values are added to the rows that do, without
        // their weights, which are above 0, and left out of the product.
        if (!whole) {
            bool odd = false;
            for (int c = lane; c < NK * CHUNKS; c += 32) {
                const uint4 x = *reinterpret_cast<const uint4*>(vb + c / CHUNKS * LDS + c % CHUNKS * 8);
                odd |= odd_pair(x.x) | odd_pair(x.y) | odd_pair(x.z) | odd_pair(x.w);
            }
            if (__any_sync(0xffffffffu, odd)) {
                for (int key = 0; key < NK; ++key) {
#pragma unroll
                    for (int j = 0; j < DT; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float v = to_float(vb[key * LDS + j * 8 + 2 * tig + e]);
                            if (fabsf(v) < INFINITY) continue;
#pragma unroll
                            for (int r = 0; r < 2; ++r)
                                if (kt + key < hi[r]) o_acc[j][2 * r + e] += v;
                        }
                }
                __syncwarp();
                for (int c = lane; c < NK * D; c += 32) {
                    __nv_bfloat16* v = vb + c / D * LDS + c % D;
                    if (!(fabsf(to_float(*v)) < INFINITY)) *v = __float2bfloat16_rn(0.0f);
                }
                __syncwarp();
            }
        }
#pragma unroll
        for (int jd = 0; jd < DT; jd += 2) {
            unsigned b[4];
            ldmatrix_x4_trans(b, vb + ((mat & 1) * 8 + mr) * LDS + (jd + (mat >> 1)) * 8);
            mma_bf16(o_acc[jd], pf, b[0], b[1]);
            mma_bf16(o_acc[jd + 1], pf, b[2], b[3]);
        }
        __syncwarp();                                     // this tile's place may be filled again
#pragma unroll
        for (int n = 0; n + 1 < STAGES; ++n) there[n] = there[n + 1];
    }
    cp_async_wait<0>();
    pdl_trigger();

#pragma unroll
    for (int r = 0; r < 2; ++r) {
        l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 1);
        l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 2);
        const int row = 8 * r + gid;
        if (row >= it.count) continue;
        const size_t at = (size_t)(it.base + row) * kv_heads + hk;
        float* dst = partial_acc + at * D + 2 * tig;
#pragma unroll
        for (int j = 0; j < DT; ++j)
            *reinterpret_cast<float2*>(dst + j * 8) = make_float2(o_acc[j][2 * r], o_acc[j][2 * r + 1]);
        if (tig == 0) {
            partial_ml[at] = make_float2(m_ref[r] * sl, l_run[r]);
            if (second) partial_ml[at + (size_t)HALF_ROWS * kv_heads] = make_float2(-INFINITY, 0.0f);
        }
    }
    if (behind) pdl_wait();
}

}  // namespace

// Rows of an item that a warp takes, keys that the ranges of own keys are a multiple of, and warps that
// an SM holds at once.
DE_EXPORT int de_shared_mma_rows() { return ROWS; }
DE_EXPORT int de_shared_mma_unit() { return NK; }
DE_EXPORT int de_shared_mma_held() { return BLOCKS * WARPS; }

// `tile_rows`: most rows of an item (above de_shared_mma_rows() several warps'); `order` as in
// shared_prefix.cu; q in 4-byte pieces, pages in 16-byte ones.
DE_EXPORT int de_shared_mma(const void* q, int q_stride, const void* k_pages, const void* v_pages,
                            const int* block_table, int table_stride, int num_pages,
                            const int* seq_slot, const int* seq_pos0, const int* items, int num_items,
                            int tile_rows, int order, float* partial_acc, float* partial_ml, int heads,
                            int kv_heads, int head_dim, int page, float scale, int* status,
                            void* stream) {
    if (num_items <= 0) return 0;
    if (tile_rows < 1 || tile_rows > 1024) return -3;
    if (head_dim != D || kv_heads < 1 || heads % kv_heads || page < 1 ||
        (long long)num_items * kv_heads > 0x7fffffffll)
        return -2;
    if (q_stride % 2 || ((uintptr_t)q & 3) || ((uintptr_t)k_pages & 15) || ((uintptr_t)v_pages & 15))
        return -3;
    if (SMEM > 40 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(
            shared_mma_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
        if (e != cudaSuccess) return (int)e;
    }
    const long long places = (long long)num_items * kv_heads;
    const dim3 grid((unsigned)((places + WARPS - 1) / WARPS), (tile_rows + ROWS - 1) / ROWS);
    return de_launch(shared_mma_kernel, grid, dim3(THREADS), SMEM, (cudaStream_t)stream,
                     (const __nv_bfloat16*)q, q_stride, (const __nv_bfloat16*)k_pages,
                     (const __nv_bfloat16*)v_pages, block_table, table_stride, num_pages, seq_slot,
                     seq_pos0, (const Item*)items, num_items, partial_acc, (float2*)partial_ml, heads,
                     kv_heads, page, scale, order, status);
}
