// Attention whose requests share a prefix, on the 5th-generation tensor cores (shared_prefix.cu has the
// formulas and the merge): bfloat16, head sizes 64 and 128 (-DHEAD_DIM=d), shared keys only.
//
// All rows of a group see every key of its prefix, so this is a product of many rows with many keys
// without a mask.  A block holds up to 256 rows (token, query head) of one kv head as two pipelines of 128:
//   * more than 128 rows: a pipeline a half of the rows, both on every tile of 128 keys;
//   * up to 128 rows: both pipelines have the same rows and take the key tiles in turn, each for a
//     partial result of its own, so that one's exponentials run beside the other's products here too.
// Warps:
//   * warps 0-3 and 4-7 are the pipelines' softmax threads, one thread a row (= a lane of tensor
//     memory): a tile's 128 scores into registers, exponentials in float32, weights as bfloat16 back
//     into tensor memory as the A operand of the second product;
//   * warp 8, one thread, issues s = q k^T (operands in shared memory) and o += p v (p in tensor
//     memory, v MN-major straight from the pages) for whichever pipeline is ready;
//   * warp 9 fetches: a ring of buffers of 128 keys or 128 values, one TMA box a page and 64 features.
// A row's exponentials refer to a maximum that is raised, and o rescaled, only when a score has grown by
// more than 2^8 beyond it.
//
// What bounds it: with r rows a block a byte of keys and values takes r multiply-adds, so up to 128 rows
// it is the cache's way from memory (at head size 128), beyond it the tensor cores and, as much, the
// exponentials: a tile of 128 x 128 scores takes the tensor cores 1,024 cycles at head size 128 and 512
// at 64, its exponentials 1,024 (16 a cycle).
//
// Every wait is bounded (status 3; the block then stores no result, runs to its end and frees its tensor
// memory).  One block an SM.

#include <cuda.h>

#include "shared_prefix.cuh"
#include "tcgen05_common.cuh"
#include "tensor_maps.cuh"

DE_DEFINE_PDL_SWITCH

namespace {

using namespace shared_prefix;
using namespace tc5;

#ifndef HEAD_DIM
#define HEAD_DIM 64
#endif
constexpr int D = HEAD_DIM;
static_assert(D == 64 || D == 128, "built for head sizes 64 and 128");
constexpr int KS = D / 64;                    // 64-feature sub-tiles of a row
constexpr int LANES = HALF_ROWS;              // rows of a pipeline
constexpr int KT = 128;                       // keys of a tile
constexpr int SUB = 128 * 128;                // bytes of a sub-tile: 128 rows of 64 features
constexpr int BUFFER = KS * SUB;              // 128 keys, or their values
constexpr int BUFFERS = D == 64 ? 10 : 5;     // what shared memory has room for beside q
constexpr int THREADS = 10 * 32;
constexpr int MMA_WARP = 8, COPY_WARP = 9;
constexpr int SMEM = 2 * BUFFER + BUFFERS * BUFFER + 512;
constexpr int COLUMNS = 512;
// columns of tensor memory: scores of pipeline x at 128 x; results at 256 + D x; weights (64 columns) over
// the scores at head size 128, where there is no other room, and at 384 + 64 x at head size 64
constexpr bool OVER = D == 128;
constexpr int O_COL = 256;
__device__ __forceinline__ unsigned p_col(int x) { return OVER ? 128u * x : 384u + 64u * x; }
constexpr float RAISE = 8.0f;

__device__ __forceinline__ bool mbar_test(void* bar, unsigned parity) {
    unsigned done;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return done != 0;
}
__device__ __forceinline__ void umma_a_tmem(unsigned d, unsigned a, unsigned long long b_desc,
                                            unsigned idesc, bool accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.u32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
        "}\n"
        ::"r"(d), "r"(a), "l"(b_desc), "r"(idesc), "r"((unsigned)accumulate) : "memory");
}
__device__ __forceinline__ void tmem_store_32cols(unsigned taddr, const unsigned (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};\n"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]),
          "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
          "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
          "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
          "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_stores() {
    asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void before_sync() {
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
}
__device__ __forceinline__ void after_sync() {
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void cp_async16(void* smem, const void* gmem, bool pred) {
    const int bytes = pred ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(smem_u32(smem)), "l"(gmem),
                 "r"(bytes));
}
// v as the second operand: MN-major, 128-byte swizzle, from 64 features to the next 64 a sub-tile
__device__ __forceinline__ unsigned long long value_desc(const void* tile) {
    unsigned long long d = smem_desc(tile);
    if (KS == 2) d += (unsigned long long)((SUB >> 4) - 1) << 16;
    return d;
}
constexpr unsigned DESC_S = instr_desc(128, KT);
constexpr unsigned DESC_O = instr_desc(128, D) | 1u << 16;

__global__ void __launch_bounds__(THREADS, 1)
shared_tcgen05_kernel(const __nv_bfloat16* __restrict__ q, int q_stride,
                      const __grid_constant__ CUtensorMap map_k,
                      const __grid_constant__ CUtensorMap map_v, const int* __restrict__ block_table,
                      int table_stride, int num_pages, const int* __restrict__ seq_slot,
                      const Item* __restrict__ items, float* __restrict__ partial_acc,
                      float2* __restrict__ partial_ml, int heads, int kv_heads, int page, float scale,
                      int* status) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* q_s = smem_raw;                        // [2][KS] sub-tiles
    unsigned char* ring = q_s + 2 * BUFFER;
    unsigned long long* bars = reinterpret_cast<unsigned long long*>(ring + BUFFERS * BUFFER);
    unsigned long long* full = bars;                      // [BUFFERS] the pages have landed
    unsigned long long* empty = bars + BUFFERS;           // [BUFFERS] the products that read it are done
    unsigned long long* s_done = bars + 2 * BUFFERS;      // [2] scores are complete
    unsigned long long* p_ready = s_done + 2;             // [2] weights are written (128 arrivals)
    unsigned long long* o_done = s_done + 4;              // [2] weights times values is complete
    unsigned long long* s_free = s_done + 6;              // [2] scores are in registers (128 arrivals)
    unsigned long long* drained = s_done + 8;             // everything issued is complete, after a failed wait
    unsigned& tmem_slot = *reinterpret_cast<unsigned*>(s_done + 9);
    int& missing_s = *reinterpret_cast<int*>(s_done + 10);

    const Item it = items[blockIdx.x / kv_heads];
    const int hk = blockIdx.x % kv_heads, g = heads / kv_heads;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool turns = it.split != 0;                     // the pipelines take the tiles in turn
    const int n_tiles = (it.end - it.begin + KT - 1) / KT;
    const bool aligned = (smem_u32(smem_raw) & 1023u) == 0;
    if (!aligned && tid == 0) atomicExch(status, 4);
    // tiles of a pipeline, and which
    const int n_of[2] = {turns ? (n_tiles + 1) / 2 : n_tiles,
                         turns ? n_tiles / 2 : it.count > LANES ? n_tiles : 0};
    auto tile_of = [&](int x, int j) { return turns ? 2 * j + x : j; };

    if (tid == 0) {
        missing_s = 0;
        mbar_init(drained, 1);
        for (int i = 0; i < BUFFERS; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int x = 0; x < 2; ++x) {
            mbar_init(&s_done[x], 1);
            mbar_init(&p_ready[x], LANES);
            mbar_init(&o_done[x], 1);
            mbar_init(&s_free[x], LANES);
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == MMA_WARP) tmem_alloc(&tmem_slot, COLUMNS);
    __syncthreads();
    pdl_wait();
    pdl_trigger();                    // what follows in the stream may fill the SMs that are left
    const int slot = seq_slot[it.seq];
    const int box = page < KT ? page : KT;                // keys of a box, boxes of a tile
    const int boxes = KT / box;
    auto page_at = [&](int key) {
        const int logical = key / page;
        int id = -1;
        if (logical < table_stride && slot >= 0)
            id = block_table[(size_t)slot * table_stride + logical];
        return id >= 0 && id < num_pages ? id : -1;
    };
    // does every key of the range have a page?  If not the softmax threads look their pages up too.
    {
        bool gone = false;
        for (int key = it.begin / page * page + tid * page; key < it.end; key += THREADS * page)
            gone |= page_at(key) < 0;
        if (gone) {
            atomicExch(status, 2);
            missing_s = 1;
        }
    }
    const int x = warp < 8 ? warp >> 2 : 0;               // pipeline
    const int rowi = (warp & 3) * 32 + lane;              // row of the pipeline
    const int row = turns ? rowi : x * LANES + rowi;      // of the item
    const bool live = warp < 8 && row < it.count;
    if (warp < 8) {                   // q in the operand layout: 16-byte piece c at place c xor row % 8
        const int r = it.row0 + (live ? row : 0);
        const __nv_bfloat16* src = q + (size_t)(it.tok0 + r / g) * q_stride + (hk * g + r % g) * D;
        unsigned char* dst = q_s + x * BUFFER + rowi * 128;
#pragma unroll
        for (int c = 0; c < D / 8; ++c)
            cp_async16(dst + (c >> 3) * SUB + (((c & 7) ^ (rowi & 7)) << 4), src + c * 8, live);
        asm volatile("cp.async.commit_group;\n" ::);
        asm volatile("cp.async.wait_group 0;\n" ::: "memory");
    }
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    before_sync();
    __syncthreads();
    after_sync();
    const unsigned tmem = tmem_slot;
    const bool missing = missing_s != 0;
    bool ok = aligned;

    if (warp == COPY_WARP) {
        // ------------------------------------------------------------------ copies
        // unit 2 t: the keys of tile t, unit 2 t + 1: its values
        int issued = 0;
        for (int t = 0; t < n_tiles; ++t) {
            const int key = it.begin + t * KT + lane * box;
            int id = -1;
            if (lane < boxes && key < it.end) id = page_at(key);
            const unsigned there = __ballot_sync(0xffffffffu, id >= 0);
            const unsigned bytes = __popc(there) * (unsigned)(box * 128 * KS);
            const int y = (int)((((long long)id * kv_heads + hk) * page + key % page));
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const int unit = 2 * t + v, b = unit % BUFFERS;
                if (unit >= BUFFERS && ok) ok = mbar_wait(&empty[b], (unit / BUFFERS - 1) & 1, status);
                ok = __shfl_sync(0xffffffffu, ok, 0);
                if (!ok) break;
                if (lane == 0) mbar_expect_tx(&full[b], bytes);
                ++issued;
                __syncwarp();
                if (id >= 0)
#pragma unroll
                    for (int sub = 0; sub < KS; ++sub)
                        tma_load_2d(ring + b * BUFFER + sub * SUB + lane * box * 128, v ? &map_v : &map_k,
                                    &full[b], 64 * sub, y);
            }
            if (!ok) break;
        }
        if (!ok)                      // what is on its way lands before the block ends
            for (int u = max(0, issued - BUFFERS); u < issued; ++u)
                mbar_wait(&full[u % BUFFERS], (u / BUFFERS) & 1, status);
    } else if (warp == MMA_WARP) {
        // ------------------------------------------------------------------ tensor cores
        if (lane == 0) {
            int s_next[2] = {0, 0}, o_next[2] = {0, 0};   // products of each pipeline issued so far
            int k_freed = 0, v_freed = 0;                 // tiles whose buffers are handed back
            unsigned idle = 0;
            while (ok && (o_next[0] < n_of[0] || o_next[1] < n_of[1])) {
                bool progress = false;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (o_next[i] < s_next[i]) {
                        const int j = o_next[i], unit = 2 * tile_of(i, j) + 1, b = unit % BUFFERS;
                        if (mbar_test(&p_ready[i], j & 1) && mbar_test(&full[b], (unit / BUFFERS) & 1)) {
                            after_sync();
                            const unsigned long long vb = value_desc(ring + b * BUFFER);
#pragma unroll
                            for (int k = 0; k < KT / 16; ++k)
                                umma_a_tmem(tmem + O_COL + D * i, tmem + p_col(i) + 8 * k,
                                            vb + (unsigned long long)(k * 2048 >> 4), DESC_O,
                                            j > 0 || k > 0);
                            umma_commit(&o_done[i]);
                            ++o_next[i];
                            progress = true;
                            if (turns) umma_commit(&empty[b]);
                        }
                    }
                    if (s_next[i] < n_of[i]) {
                        const int j = s_next[i], unit = 2 * tile_of(i, j), b = unit % BUFFERS;
                        // the columns are free: the last weights are multiplied (where they lie over the
                        // scores), or the last scores in registers
                        const bool free = j == 0 || (OVER ? o_next[i] == j && mbar_test(&o_done[i], (j - 1) & 1)
                                                          : mbar_test(&s_free[i], (j - 1) & 1));
                        if (free && mbar_test(&full[b], (unit / BUFFERS) & 1)) {
                            after_sync();
#pragma unroll
                            for (int sub = 0; sub < KS; ++sub) {
                                const unsigned long long a = smem_desc(q_s + i * BUFFER + sub * SUB);
                                const unsigned long long kb = smem_desc(ring + b * BUFFER + sub * SUB);
#pragma unroll
                                for (int k = 0; k < 4; ++k)
                                    umma_bf16(tmem + 128 * i, a + 2 * k, kb + 2 * k, DESC_S,
                                              sub > 0 || k > 0);
                            }
                            umma_commit(&s_done[i]);
                            ++s_next[i];
                            progress = true;
                            if (turns) umma_commit(&empty[b]);
                        }
                    }
                }
                if (!turns) {                             // a buffer goes back when both have read it
                    while (k_freed < s_next[0] && (n_of[1] == 0 || k_freed < s_next[1]))
                        umma_commit(&empty[2 * k_freed++ % BUFFERS]);
                    while (v_freed < o_next[0] && (n_of[1] == 0 || v_freed < o_next[1]))
                        umma_commit(&empty[(2 * v_freed++ + 1) % BUFFERS]);
                }
                if (progress) {
                    idle = 0;
                } else if (++idle > SPIN_LIMIT) {
                    atomicExch(status, 3);
                    ok = false;
                }
            }
            if (!ok) {                // what is issued ends before the tensor memory is freed
                umma_commit(drained);
                mbar_wait(drained, 0, status);
            }
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------------ softmax
        const unsigned lanes = (unsigned)((warp & 3) * 32) << 16;
        const unsigned s_addr = tmem + 128 * x + lanes, p_addr = tmem + p_col(x) + lanes;
        const unsigned o_addr = tmem + O_COL + D * x + lanes;
        const float sl = scale * 1.4426950408889634f;
        float m_ref = -INFINITY, l_run = 0.0f;
        for (int j = 0; j < n_of[x]; ++j) {
            const int t = tile_of(x, j), kt = it.begin + t * KT;
            if (ok) ok = mbar_wait(&s_done[x], j & 1, status);
            after_sync();
            unsigned sv[4][32];
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_load_32cols(s_addr + 32 * c, sv[c]);
            tmem_wait_loads();
            if (!OVER) {
                before_sync();
                mbar_arrive(&s_free[x]);
            }
            // keys behind the range, or without a page, are not seen
            unsigned gone = 0;                            // boxes without a page
            if (missing) {
                const int key = kt + lane * box;
                gone = __ballot_sync(0xffffffffu, lane < boxes && key < it.end && page_at(key) < 0);
            }
            if (kt + KT > it.end || gone) {
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const int n = 32 * c + i;
                        if (kt + n >= it.end || (gone >> (n / box) & 1)) sv[c][i] = 0xff800000u;
                    }
            }
            float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int i = 0; i < 32; ++i) m4[i & 3] = fmaxf(m4[i & 3], __uint_as_float(sv[c][i]));
            const float m = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
            const bool raise = (m - m_ref) * sl > RAISE;
            bool rest = OVER || j == 0;                   // the last product is known to be complete
            if (__any_sync(0xffffffffu, raise)) {
                if (!rest) {
                    if (ok) ok = mbar_wait(&o_done[x], (j - 1) & 1, status);
                    after_sync();
                    rest = true;
                }
                const float f = raise ? exp2_fast((m_ref - m) * sl) : 1.0f;
                if (j > 0) {
#pragma unroll 1
                    for (int c = 0; c < D / 32; ++c) {
                        unsigned ov[32];
                        tmem_load_32cols(o_addr + 32 * c, ov);
                        tmem_wait_loads();
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            ov[i] = __float_as_uint(__uint_as_float(ov[i]) * f);
                        tmem_store_32cols(o_addr + 32 * c, ov);
                    }
                    tmem_wait_stores();
                }
                l_run *= f;
                if (raise) m_ref = m;
            }
            const float off = m_ref == -INFINITY ? 0.0f : -m_ref * sl;
            float l4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            unsigned pw[2][32];
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const float a = exp2_fast(fmaf(__uint_as_float(sv[c][i]), sl, off));
                    const float b = exp2_fast(fmaf(__uint_as_float(sv[c][i + 1]), sl, off));
                    l4[i & 2] += a;
                    l4[(i & 2) + 1] += b;
                    pw[c >> 1][(c & 1) * 16 + i / 2] = pack2(a, b);
                }
            l_run += (l4[0] + l4[1]) + (l4[2] + l4[3]);
            if (!rest) {                                  // the weights' columns are free
                if (ok) ok = mbar_wait(&o_done[x], (j - 1) & 1, status);
                after_sync();
            }
            tmem_store_32cols(p_addr, pw[0]);
            tmem_store_32cols(p_addr + 32, pw[1]);
            // values that no row sees may be anything, and 0 * NaN is NaN in the product: thread i has
            // row i (both pipelines write the same zeros)
            if (kt + rowi >= it.end || (gone >> (rowi / box) & 1)) {
                const int unit = 2 * t + 1, b = unit % BUFFERS;
                if (ok) ok = mbar_wait(&full[b], (unit / BUFFERS) & 1, status);
#pragma unroll
                for (int sub = 0; sub < KS; ++sub) {
                    uint4* v = reinterpret_cast<uint4*>(ring + b * BUFFER + sub * SUB + rowi * 128);
#pragma unroll
                    for (int c = 0; c < 8; ++c) v[c] = make_uint4(0u, 0u, 0u, 0u);
                }
                asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            }
            tmem_wait_stores();
            before_sync();
            mbar_arrive(&p_ready[x]);
        }
        const int base = it.base + x * LANES + rowi;
        const size_t at = (size_t)base * kv_heads + hk;
        if (n_of[x] > 0) {
            if (ok) ok = mbar_wait(&o_done[x], (n_of[x] - 1) & 1, status);
            after_sync();
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                unsigned ov[32];
                tmem_load_32cols(o_addr + 32 * c, ov);
                tmem_wait_loads();
                if (!ok || !live) continue;
                uint4* dst = reinterpret_cast<uint4*>(partial_acc + at * D + 32 * c);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    dst[i] = make_uint4(ov[4 * i], ov[4 * i + 1], ov[4 * i + 2], ov[4 * i + 3]);
            }
        }
        // (nothing where a wait ran out: such a row's results are those of the other ranges)
        if (live)
            partial_ml[at] = n_of[x] > 0 && ok ? make_float2(m_ref * sl, l_run)
                                               : make_float2(-INFINITY, 0.0f);
    }
    before_sync();
    __syncthreads();
    if (warp == MMA_WARP) tmem_dealloc(tmem, COLUMNS);
}

}  // namespace

// What the kernel takes: pages of a multiple of 8 keys that divide 128 or that 128 divides.
DE_EXPORT int de_shared_tcgen05_page_ok(int page) {
    return page >= 8 && page % 8 == 0 && (KT % page == 0 || page % KT == 0);
}

// Items of shared keys; q, pages in 16-byte pieces.
DE_EXPORT int de_shared_tcgen05(const void* q, int q_stride, const void* k_pages, const void* v_pages,
                                const int* block_table, int table_stride, int num_pages,
                                const int* seq_slot, const int* seq_pos0, const int* items,
                                int num_items, float* partial_acc, float* partial_ml, int heads,
                                int kv_heads, int head_dim, int page, float scale, int* status,
                                void* stream) {
    (void)seq_pos0;
    if (num_items <= 0) return 0;
    if (head_dim != D || kv_heads < 1 || heads % kv_heads || !de_shared_tcgen05_page_ok(page) ||
        (long long)num_items * kv_heads > 0x7fffffffll ||
        (long long)num_pages * kv_heads * page > 0x7fffffffll)
        return -2;
    if (q_stride % 8 || ((uintptr_t)q & 15) || ((uintptr_t)k_pages & 15) || ((uintptr_t)v_pages & 15))
        return -3;
    CUtensorMap map_k, map_v;
    const long long rows = (long long)num_pages * kv_heads * page;
    int code = tensor_maps::make(&map_k, k_pages, rows, D, D, page < KT ? page : KT, 64);
    if (code) return code;
    code = tensor_maps::make(&map_v, v_pages, rows, D, D, page < KT ? page : KT, 64);
    if (code) return code;
    const cudaError_t e = cudaFuncSetAttribute(shared_tcgen05_kernel,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    if (e != cudaSuccess) return (int)e;
    return de_launch(shared_tcgen05_kernel, dim3((unsigned)num_items * kv_heads), dim3(THREADS), SMEM,
                     (cudaStream_t)stream, (const __nv_bfloat16*)q, q_stride, map_k, map_v, block_table,
                     table_stride, num_pages, seq_slot, (const Item*)items, partial_acc,
                     (float2*)partial_ml, heads, kv_heads, page, scale, status);
}
