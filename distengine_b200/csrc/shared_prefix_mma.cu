// Attention whose requests share a prefix, on the tensor cores by mma.sync (shared_prefix.cu has the
// formulas and the merge): bfloat16, float32 softmax.  Compiled once per head size (-DHEAD_DIM=d).
//
// An item is up to 16 RT query rows with a range of keys: the keys of one request for its own rows
// (few rows, every key read once), or a prefix for the rows of a small group.  Both are bound by the
// keys' and values' way from memory.  So each of the four warps goes through key tiles of its own, 16
// keys each, every fourth of the range, with a ring of tiles that it alone fills and reads: a warp that waits
// holds up no other.  The four results are joined in shared memory at the end.
//
// A row's exponentials refer to a maximum that is raised only when a score has grown by more than 2^8
// beyond it (the quotient does not depend on it), so most tiles need no exchange between lanes and no
// rescaling of the results.

#include "shared_prefix.cuh"

DE_DEFINE_PDL_SWITCH

#include "attention_mma_common.cuh"

namespace {

using namespace shared_prefix;

constexpr int WARPS = THREADS / 32;
constexpr int NK = 16;                                    // keys of a warp's tile
constexpr int RT = D <= 128 ? 2 : 1;                     // row tiles of 16: what the registers hold
constexpr int ROWS = 16 * RT;
constexpr int STAGES = D <= 64 ? 4 : D <= 128 ? 3 : 2;    // tiles of a warp in flight or in use
constexpr int DT = D / 8;
constexpr int CHUNKS = D / 8;                             // 16-byte pieces of a key's row
constexpr int STAGE = 2 * NK * LDS;                       // keys and values of a tile, in elements
constexpr int RING_BYTES = WARPS * STAGES * STAGE * 2;
constexpr int LDO = D + 4;                                // row stride of a warp's results (float32)
constexpr int JOIN_BYTES = WARPS * 16 * (LDO + 2) * 4;    // one row tile of 16 at a time
constexpr int SMEM = RING_BYTES > JOIN_BYTES ? RING_BYTES : JOIN_BYTES;
constexpr int UNIT = WARPS * NK;
constexpr float RAISE = 8.0f;

__device__ __forceinline__ bool odd_pair(unsigned x) {    // an infinity or NaN among two bfloat16
    return (x & 0x7f80u) == 0x7f80u || (x & 0x7f800000u) == 0x7f800000u;
}

__global__ void __launch_bounds__(THREADS)
shared_mma_kernel(const __nv_bfloat16* __restrict__ q, int q_stride,
                  const __nv_bfloat16* __restrict__ k_pages,
                  const __nv_bfloat16* __restrict__ v_pages, const int* __restrict__ block_table,
                  int table_stride, int num_pages, const int* __restrict__ seq_slot,
                  const int* __restrict__ seq_pos0, const Item* __restrict__ items,
                  float* __restrict__ partial_acc, float2* __restrict__ partial_ml, int heads,
                  int kv_heads, int page, float scale, int behind, int* __restrict__ status) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int gid = lane >> 2, tig = lane & 3;
    Item it = items[blockIdx.x / kv_heads];
    const int hk = blockIdx.x % kv_heads, g = heads / kv_heads;
    const bool second = has_second_place(it);
    if (!behind) pdl_wait();
    const Range range = range_of(it, seq_pos0, g, UNIT);
    // of an item with more rows than a block takes, the block's
    it.row0 += blockIdx.y * ROWS;
    it.base += blockIdx.y * ROWS;
    it.count = min(ROWS, it.count - (int)blockIdx.y * ROWS);
    if (it.count <= 0) {
        if (behind) pdl_wait();
        return;
    }
    const int live = (it.count + 15) >> 4;                // row tiles that hold rows
    __nv_bfloat16* ring = reinterpret_cast<__nv_bfloat16*>(smem_raw) + warp * STAGES * STAGE;

    const int slot = seq_slot[it.seq];
    const int tiles = (range.end - range.begin + NK - 1) / NK;
    const int mine = tiles > warp ? (tiles - warp + WARPS - 1) / WARPS : 0;

    // A tile's pages: lane j looks the page of key j up, a tile ahead of its copies.  The place of a
    // key's row in units of rows of D features, or -1.
    auto look_up = [&](int i) {
        const int key = range.begin + (i * WARPS + warp) * NK + (lane & 15);
        long long at = -1;
        if (lane < 16 && i < mine && key < range.end) {
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
        there[i] = i < mine ? copy(i, at) : 0;
        cp_async_commit();
    }

    // the rows of this thread: gid and gid + 8 of each row tile
    unsigned qf[RT][D / 16][4];
    int hi[2 * RT];
    int min_hi = range.end;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = rt * 16 + 8 * i + gid, r = it.row0 + row;
            const bool ok = row < it.count;
            const __nv_bfloat16* p = q + (size_t)(it.tok0 + (ok ? r / g : 0)) * q_stride +
                                     (hk * g + (ok ? r % g : 0)) * D + 2 * tig;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                qf[rt][kk][i] = ok ? *reinterpret_cast<const unsigned*>(p + kk * 16) : 0u;
                qf[rt][kk][i + 2] = ok ? *reinterpret_cast<const unsigned*>(p + kk * 16 + 8) : 0u;
            }
            hi[2 * rt + i] = range.row_end(it, row, g);
            if (ok) min_hi = min(min_hi, hi[2 * rt + i]);
        }
    min_hi = __reduce_min_sync(0xffffffffu, min_hi);      // up to here every row sees every key

    const float sl = scale * 1.4426950408889634f;
    float o_acc[RT][DT][4], m_ref[2 * RT], l_run[2 * RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int j = 0; j < DT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o_acc[rt][j][e] = 0.0f;
        m_ref[2 * rt] = m_ref[2 * rt + 1] = -INFINITY;
        l_run[2 * rt] = l_run[2 * rt + 1] = 0.0f;
    }

    for (int i = 0; i < mine; ++i) {
        {   // the tile STAGES - 1 ahead, into the place of the one that is done
            const long long at = next;
            next = look_up(i + STAGES);
            unsigned bits = 0;
            if (i + STAGES - 1 < mine) bits = copy(i + STAGES - 1, at);
            cp_async_commit();
            there[STAGES - 1] = bits;
        }
        cp_async_wait<STAGES - 1>();
        __syncwarp();
        const __nv_bfloat16* kb = ring + (i % STAGES) * STAGE;
        __nv_bfloat16* vb = ring + (i % STAGES) * STAGE + NK * LDS;
        const int kt = range.begin + (i * WARPS + warp) * NK;
        const int mat = lane >> 3, mr = lane & 7;

        float s[RT][2][4];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[rt][j][e] = 0.0f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
            unsigned b[4];
            ldmatrix_x4(b, kb + ((mat >> 1) * 8 + mr) * LDS + kk * 16 + (mat & 1) * 8);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                if (rt >= live) break;
                mma_bf16(s[rt][0], qf[rt][kk], b[0], b[1]);
                mma_bf16(s[rt][1], qf[rt][kk], b[2], b[3]);
            }
        }
        const unsigned here = there[0];
        const bool whole = kt + NK <= min_hi;             // no row's limit is in this tile
        if (!whole || here != 0xffffu) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = j * 8 + 2 * tig + (e & 1);
                        if (!(here >> key & 1) || kt + key >= hi[2 * rt + (e >> 1)])
                            s[rt][j][e] = -INFINITY;
                    }
        }
        // raise the references that a score has left behind
        bool raise = false;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float top = fmaxf(s[rt][e >> 1][2 * (e & 1)], s[rt][e >> 1][2 * (e & 1) + 1]);
                raise |= (top - m_ref[2 * rt + (e & 1)]) * sl > RAISE;
            }
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
            for (int r = 0; r < 2 * RT; ++r) {
                const int rt = r >> 1, x = 2 * (r & 1);
                float m = fmaxf(fmaxf(s[rt][0][x], s[rt][0][x + 1]), fmaxf(s[rt][1][x], s[rt][1][x + 1]));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                m = fmaxf(m, m_ref[r]);
                const float f = m == m_ref[r] ? 1.0f : fast_exp2((m_ref[r] - m) * sl);
                m_ref[r] = m;
                l_run[r] *= f;
#pragma unroll
                for (int j = 0; j < DT; ++j) {
                    o_acc[rt][j][x] *= f;
                    o_acc[rt][j][x + 1] *= f;
                }
            }
        }
        // weights; the sum takes them before they are rounded to bfloat16 for their product
        unsigned pf[RT][4];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const float base0 = m_ref[2 * rt] == -INFINITY ? 0.0f : m_ref[2 * rt] * sl;
            const float base1 = m_ref[2 * rt + 1] == -INFINITY ? 0.0f : m_ref[2 * rt + 1] * sl;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float p0 = fast_exp2(fmaf(s[rt][j][0], sl, -base0));
                const float p1 = fast_exp2(fmaf(s[rt][j][1], sl, -base0));
                const float p2 = fast_exp2(fmaf(s[rt][j][2], sl, -base1));
                const float p3 = fast_exp2(fmaf(s[rt][j][3], sl, -base1));
                l_run[2 * rt] += p0 + p1;
                l_run[2 * rt + 1] += p2 + p3;
                pf[rt][2 * j] = pack_bf16(p0, p1);
                pf[rt][2 * j + 1] = pack_bf16(p2, p3);
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
                            for (int r = 0; r < 2 * RT; ++r)
                                if (kt + key < hi[r]) o_acc[r >> 1][j][2 * (r & 1) + e] += v;
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
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                if (rt >= live) break;
                mma_bf16(o_acc[rt][jd], pf[rt], b[0], b[1]);
                mma_bf16(o_acc[rt][jd + 1], pf[rt], b[2], b[3]);
            }
        }
        __syncwarp();                                     // this tile's place may be filled again
#pragma unroll
        for (int n = 0; n + 1 < STAGES; ++n) there[n] = there[n + 1];
    }
    cp_async_wait<0>();
    pdl_trigger();

    // join the warps' results, a row tile at a time
#pragma unroll
    for (int r = 0; r < 2 * RT; ++r) {
        l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 1);
        l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 2);
    }
    float* res = reinterpret_cast<float*>(smem_raw);      // [WARPS][16][LDO]
    float2* res_ml = reinterpret_cast<float2*>(res + WARPS * 16 * LDO);       // [WARPS][16]
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        if (rt >= live) break;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float* dst = res + (warp * 16 + gid + 8 * i) * LDO + 2 * tig;
#pragma unroll
            for (int j = 0; j < DT; ++j)
                *reinterpret_cast<float2*>(dst + j * 8) =
                    make_float2(o_acc[rt][j][2 * i], o_acc[rt][j][2 * i + 1]);
            if (tig == 0)
                res_ml[warp * 16 + gid + 8 * i] =
                    make_float2(m_ref[2 * rt + i] * sl, l_run[2 * rt + i]);
        }
        __syncthreads();
        const int rows = min(16, it.count - rt * 16);
        for (int c = tid; c < rows * (D / 4); c += THREADS) {
            const int r = c / (D / 4), f = c % (D / 4) * 4;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) top = fmaxf(top, res_ml[w * 16 + r].x);
            const float base = top == -INFINITY ? 0.0f : top;
            float l = 0.0f;
            float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float2 ml = res_ml[w * 16 + r];
                if (ml.x == -INFINITY && ml.y == 0.0f) continue;
                const float x = exp2f(ml.x - base);
                const float4 v = *reinterpret_cast<const float4*>(res + (w * 16 + r) * LDO + f);
                l = fmaf(x, ml.y, l);
                a.x = fmaf(x, v.x, a.x);
                a.y = fmaf(x, v.y, a.y);
                a.z = fmaf(x, v.z, a.z);
                a.w = fmaf(x, v.w, a.w);
            }
            const size_t at = (size_t)(it.base + rt * 16 + r) * kv_heads + hk;
            *reinterpret_cast<float4*>(partial_acc + at * D + f) = a;
            if (f == 0) {
                partial_ml[at] = make_float2(top, l);
                if (second)
                    partial_ml[at + (size_t)HALF_ROWS * kv_heads] = make_float2(-INFINITY, 0.0f);
            }
        }
    }
    if (behind) pdl_wait();
}

}  // namespace

DE_EXPORT int de_shared_mma_rows() { return ROWS; }
// blocks that an SM holds at once
DE_EXPORT int de_shared_mma_blocks_per_sm() {
    return 227 * 1024 / (SMEM + 1024) < 4 ? 227 * 1024 / (SMEM + 1024) : 4;
}

// `tile_rows`: most rows of an item (above de_shared_mma_rows() in several blocks); `behind` as in
// shared_prefix.cu; q in 4-byte pieces, pages in 16-byte ones.
DE_EXPORT int de_shared_mma(const void* q, int q_stride, const void* k_pages, const void* v_pages,
                            const int* block_table, int table_stride, int num_pages,
                            const int* seq_slot, const int* seq_pos0, const int* items, int num_items,
                            int tile_rows, int behind, float* partial_acc, float* partial_ml, int heads, int kv_heads,
                            int head_dim, int page, float scale, int* status, void* stream) {
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
    return de_launch(shared_mma_kernel, dim3((unsigned)num_items * kv_heads, (tile_rows + ROWS - 1) / ROWS),
                     dim3(THREADS), SMEM,
                     (cudaStream_t)stream, (const __nv_bfloat16*)q, q_stride,
                     (const __nv_bfloat16*)k_pages, (const __nv_bfloat16*)v_pages, block_table,
                     table_stride, num_pages, seq_slot, seq_pos0, (const Item*)items, partial_acc,
                     (float2*)partial_ml, heads, kv_heads, page, scale, behind, status);
}
