// Attention whose requests share a prefix, on the 5th-generation tensor cores (shared_prefix.cu has the
// formulas and the merge): bfloat16, head sizes 64 and 128 (-DHEAD_DIM=d), shared keys only.
//
// All rows of a group see every key of its prefix, so this is a product of many rows with many keys
// without a mask.  A block holds up to 256 rows (token, query head) of one kv head as two pipelines of 128:
//   * more than 128 rows: a pipeline a half of the rows, both on every tile of 128 keys;
//   * up to 128 rows: both pipelines have the same rows and take the key tiles in turn, each for a
//     partial result of its own, so that one's exponentials run beside the other's products here too.
// Warps:
//   * warps 0-7 and 8-15 are the pipelines' softmax threads, two threads a row (= a lane of tensor
//     memory), each 32 keys of each half of a tile: scores into registers, exponentials in float32, weights
//     back into tensor memory as the A operand of the second product, which takes bfloat16 (half a step of
//     2^-8 a weight; the sum is of the weights before they are rounded);
//   * warps 16 and 17, one thread each, issue a pipeline's s = q k^T (operands in shared memory) and
//     o += p v (p in tensor memory, v MN-major straight from the pages);
//   * warps 18 and 19 fetch: a ring of buffers of 128 keys or 128 values, one TMA box a page and 64 features.
// A tile goes through in halves of 64 keys, each with columns of tensor memory of its own, so a half's scores
// are formed while the other's exponentials are (512 rows behind 65,003 keys, on one GPU at 1,965 MHz, 151 us;
// tiles of 128 keys at a time, whose scores had to wait for the weights over them, 171).  A row's exponentials
// refer to a maximum that is raised, and o rescaled, only when a score has grown by more than 2^8 beyond it.
//
// What bounds it: with r rows a block a byte of keys and values takes r multiply-adds, so up to 128 rows
// it is the cache's way from memory (at head size 128: 108 rows behind 15,566 keys of 32 kv heads, 255 MB, 53 us
// of the call's 76), beyond it the tensor cores and, as much, the exponentials: 128 x 128 scores take the
// tensor cores 1,024 cycles at head size 128 and 512 at 64, their exponentials 1,024 (16 a cycle).  512 rows
// behind 65,003 keys: a call now and then 155 to 160 us (870 TFLOP/s at 1,965 MHz), call after call 184 (740;
// the power limit of 1,000 W then leaves the SMs 1,580 MHz).
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
constexpr int SOFTMAX_WARPS = 16, MMA_WARP = 16, COPY_WARP = 18;
// Two warps fetch: one issues a box in some 100 cycles, too slowly for small pages (108 rows behind 15,566
// keys in pages of 16: 92 us, with two 77; 512 rows behind 32,000 82.7 and 76.0, in pages of 128 75.9 and 76.1).
constexpr int COPY_WARPS = 2, THREADS = (COPY_WARP + COPY_WARPS) * 32;
constexpr int SMEM = 2 * BUFFER + BUFFERS * BUFFER + 512 + 2 * 2 * LANES * 4;
constexpr int COLUMNS = 512;
// columns of tensor memory: scores of pipeline x and half h of a tile at 128 x + 64 h, weights over the first
// 32 of them; results at 256 + D x
constexpr int O_COL = 256;
constexpr int HK = KT / 2;                    // keys of a half
constexpr float RAISE = 8.0f;
constexpr int ROW_BYTES = D * 4 + 16;         // of a row's results in shared memory: no two lanes on one bank
static_assert(2 * LANES * ROW_BYTES <= BUFFERS * BUFFER, "the ring holds the results");

// Bounded wait for the phase with the given parity, as tc5::mbar_wait, but a thread sleeps for up to
// some microseconds a look: 16 warps that look as often as they can take the issue slots of those
// that have work.
__device__ __forceinline__ bool wait(void* bar, unsigned parity, int* status) {
    const unsigned addr = smem_u32(bar);
    for (unsigned spins = 0; spins < SPIN_LIMIT / 16; ++spins) {
        unsigned done;
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n"
            "selp.u32 %0, 1, 0, p;\n"
            "}\n"
            : "=r"(done) : "r"(addr), "r"(parity), "r"(4000u) : "memory");
        if (done) return true;
    }
    atomicExch(status, 3);
    return false;
}
__device__ __forceinline__ void store_release(int* at, int v) {
    asm volatile("st.release.cta.shared::cta.s32 [%0], %1;\n" ::"r"(smem_u32(at)), "r"(v) : "memory");
}
// Bounded wait for a number above n.
__device__ __forceinline__ bool wait_above(int* at, int n, int* status) {
    for (unsigned spins = 0; spins < SPIN_LIMIT; ++spins) {
        int v;
        asm volatile("ld.acquire.cta.shared::cta.s32 %0, [%1];\n" : "=r"(v) : "r"(smem_u32(at)) : "memory");
        if (v > n) return true;
        if (spins > 8) __nanosleep(100);
    }
    atomicExch(status, 3);
    return false;
}
// The products and their commits are issued by a whole warp, of which one elected thread (the same every
// time) takes effect: so the operands are known to be the same in all lanes.  Behind a branch on the lane
// an instruction takes 160 cycles to issue, eight of 128 x 128 x 16 1,307 instead of their 514.
__device__ __forceinline__ void umma(unsigned d, unsigned long long a_desc, unsigned long long b_desc,
                                     unsigned idesc, bool accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p, e;\n"
        "elect.sync _|e, 0xffffffff;\n"
        "setp.ne.u32 p, %4, 0;\n"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
        "}\n"
        ::"r"(d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"((unsigned)accumulate) : "memory");
}
__device__ __forceinline__ void umma_a_tmem(unsigned d, unsigned a, unsigned long long b_desc,
                                            unsigned idesc, bool accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p, e;\n"
        "elect.sync _|e, 0xffffffff;\n"
        "setp.ne.u32 p, %4, 0;\n"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
        "}\n"
        ::"r"(d), "r"(a), "l"(b_desc), "r"(idesc), "r"((unsigned)accumulate) : "memory");
}
__device__ __forceinline__ void commit(void* bar) {
    asm volatile(
        "{\n"
        ".reg .pred e;\n"
        "elect.sync _|e, 0xffffffff;\n"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n"
        "}\n"
        ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tmem_store_16cols(unsigned taddr, const unsigned (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};\n"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]),
          "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
          "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_load_16cols(unsigned taddr, unsigned (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15])
        : "r"(taddr) : "memory");
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
// pairs of float32 numbers, for the instructions that take two at once
typedef unsigned long long Two;
__device__ __forceinline__ Two two(float a, float b) {
    Two r;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void untwo(Two v, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;\n" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ Two fma_two(Two a, Two b, Two c) {
    Two r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ Two add_two(Two a, Two b) {
    Two r;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max_three(float a, unsigned b, unsigned c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(__uint_as_float(b)), "f"(__uint_as_float(c)));
    return r;
}
__device__ __forceinline__ void cp_async16(void* smem, const void* gmem, bool pred) {
    const int bytes = pred ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(smem_u32(smem)), "l"(gmem),
                 "r"(bytes));
}
// The two warps that share their rows: whether a thread of either says so, and their barrier.
__device__ __forceinline__ bool any_of_pair(int barrier, bool mine) {
    unsigned any;
    asm volatile(
        "{\n"
        ".reg .pred p, q;\n"
        "setp.ne.u32 p, %1, 0;\n"
        "barrier.cta.red.or.pred q, %2, 64, p;\n"
        "selp.u32 %0, 1, 0, q;\n"
        "}\n"
        : "=r"(any) : "r"((unsigned)mine), "r"(barrier) : "memory");
    return any != 0;
}
__device__ __forceinline__ void sync_pair(int barrier) {
    asm volatile("barrier.cta.sync %0, 64;\n" ::"r"(barrier) : "memory");
}
// v as the second operand: MN-major, 128-byte swizzle, from 64 features to the next 64 a sub-tile
__device__ __forceinline__ unsigned long long value_desc(const void* tile) {
    unsigned long long d = smem_desc(tile);
    if (KS == 2) d += (unsigned long long)((SUB >> 4) - 1) << 16;
    return d;
}
constexpr unsigned DESC_S = instr_desc(128, HK);
constexpr unsigned DESC_O = instr_desc(128, D) | 1u << 16;

template <bool B> struct Truth {
    static constexpr bool value = B;
};

// TURNS: there are items of up to 128 rows, whose tiles the pipelines take in turn (a form of its own: for
// others 18 questions behind two documents take 40 us, with this form 43)
template <bool TURNS>
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
    // of each pipeline and half of a tile:
    unsigned long long* s_done = bars + 2 * BUFFERS;      // [2][2] scores are complete
    unsigned long long* p_ready = s_done + 4;             // [2][2] weights are written (256 arrivals)
    unsigned long long* o_done = s_done + 8;              // [2][2] weights times values is complete
    unsigned long long* drained = s_done + 12;            // [2] what is issued is complete
    unsigned& tmem_slot = *reinterpret_cast<unsigned*>(s_done + 14);
    int& missing_s = *reinterpret_cast<int*>(s_done + 15);
    int* issued_s = &missing_s + 1;                       // units whose copies have begun
    float* exchange = reinterpret_cast<float*>(ring + BUFFERS * BUFFER + 512);   // [pipeline][half][row]

    const Item it = items[blockIdx.x / kv_heads];
    const int hk = blockIdx.x % kv_heads, g = heads / kv_heads;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool turns = TURNS && it.split != 0;            // the pipelines take the tiles in turn
    const int n_tiles = (it.end - it.begin + KT - 1) / KT;
    const bool aligned = (smem_u32(smem_raw) & 1023u) == 0;
    if (!aligned && tid == 0) atomicExch(status, 4);
    // tiles of a pipeline, and which
    const int n_of[2] = {turns ? (n_tiles + 1) / 2 : n_tiles,
                         turns ? n_tiles / 2 : it.count > LANES ? n_tiles : 0};
    auto tile_of = [&](int x, int j) { return turns ? 2 * j + x : j; };

    if (tid == 0) {
        missing_s = 0;
        *issued_s = 0;
        mbar_init(&drained[0], 1);
        mbar_init(&drained[1], 1);
        for (int i = 0; i < BUFFERS; ++i) {
            mbar_init(&full[i], COPY_WARPS);
            mbar_init(&empty[i], !turns && it.count > LANES ? 2 : 1);      // pipelines that read it
        }
        for (int x = 0; x < 4; ++x) {
            mbar_init(&s_done[x], 1);
            mbar_init(&p_ready[x], 2 * LANES);
            mbar_init(&o_done[x], 1);
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
    const int x = warp < SOFTMAX_WARPS ? warp >> 3 : 0;   // pipeline
    const int half = warp >> 2 & 1;                       // of a tile's keys, of a row's features
    const int rowi = (warp & 3) * 32 + lane;              // row of the pipeline
    const int row = turns ? rowi : x * LANES + rowi;      // of the item
    const bool live = warp < SOFTMAX_WARPS && row < it.count;
    if (warp < SOFTMAX_WARPS) {                   // q in the operand layout: 16-byte piece c at place c xor row % 8
        const int r = it.row0 + (live ? row : 0);
        const __nv_bfloat16* src = q + (size_t)(it.tok0 + r / g) * q_stride + (hk * g + r % g) * D;
        unsigned char* dst = q_s + x * BUFFER + rowi * 128;
#pragma unroll
        for (int e = 0; e < D / 16; ++e) {
            const int c = half * (D / 16) + e;
            cp_async16(dst + (c >> 3) * SUB + (((c & 7) ^ (rowi & 7)) << 4), src + c * 8, live);
        }
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
    // Waits until unit `u` (keys of tile u / 2, or its values) has landed.  A barrier's wait tells a phase
    // from its neighbours only.  Where the pipelines take turns the last unit in the buffer was the other
    // one's and may still be on its way although later ones have landed; so it is first made sure that the
    // copies of `u` have begun, before which that one has landed and been read.
    auto landed = [&](int u) {
        if (turns && ok) ok = wait_above(issued_s, u, status);
        if (ok) ok = wait(&full[u % BUFFERS], (u / BUFFERS) & 1, status);
    };

    if (warp >= COPY_WARP) {
        // ------------------------------------------------------------------ copies
        // unit 2 t: the keys of tile t, unit 2 t + 1: its values; the warps take the boxes in turn
        const int w = warp - COPY_WARP, i = COPY_WARPS * lane + w;
        int issued = 0;
        for (int t = 0; t < n_tiles; ++t) {
            const int key = it.begin + t * KT + i * box;
            int id = -1;
            if (i < boxes && key < it.end) id = page_at(key);
            const unsigned there = __ballot_sync(0xffffffffu, id >= 0);
            const unsigned bytes = __popc(there) * (unsigned)(box * 128 * KS);
            const int y = (int)((((long long)id * kv_heads + hk) * page + key % page));
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const int unit = 2 * t + v, b = unit % BUFFERS;
                if (unit >= BUFFERS && ok) ok = wait(&empty[b], (unit / BUFFERS - 1) & 1, status);
                ok = __shfl_sync(0xffffffffu, ok, 0);
                if (!ok) break;
                if (lane == 0) {
                    mbar_expect_tx(&full[b], bytes);
                    if (TURNS && w == 0) store_release(issued_s, unit + 1);
                }
                ++issued;
                __syncwarp();
                if (id >= 0)
#pragma unroll
                    for (int sub = 0; sub < KS; ++sub)
                        tma_load_2d(ring + b * BUFFER + sub * SUB + i * box * 128, v ? &map_v : &map_k,
                                    &full[b], 64 * sub, y);
            }
            if (!ok) break;
        }
        if (!ok)                      // what is on its way lands before the block ends
            for (int u = max(0, issued - BUFFERS); u < issued; ++u)
                wait(&full[u % BUFFERS], (u / BUFFERS) & 1, status);
    } else if (warp >= MMA_WARP) {
        // ------------------------------------------------------------------ tensor cores
        const int i = __shfl_sync(0xffffffffu, warp - MMA_WARP, 0);
        const int n = i ? n_of[1] : n_of[0];
        // (all lanes wait, and go on together)
        auto passed = [&](void* bar, unsigned parity) {
            if (ok) ok = wait(bar, parity, status);
            ok = __all_sync(0xffffffffu, ok);
            after_sync();
            return ok;
        };
        // step u is half u % 2 of the pipeline's tile u / 2; use u / 2 of the half's barriers
        auto scores = [&](int u) {
            const int h = u & 1, unit = 2 * tile_of(i, u >> 1), b = unit % BUFFERS;
            if (h == 0) landed(unit);
            // (the half's columns hold the weights of two steps before)
            if (u >= 2 && !passed(&o_done[2 * i + h], ((u >> 1) - 1) & 1)) return;
            if (u < 2) {
                ok = __all_sync(0xffffffffu, ok);
                after_sync();
            }
            if (!ok) return;
#pragma unroll
            for (int sub = 0; sub < KS; ++sub) {
                const unsigned long long a = smem_desc(q_s + i * BUFFER + sub * SUB);
                const unsigned long long kb = smem_desc(ring + b * BUFFER + sub * SUB + h * (SUB / 2));
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    umma(tmem + 128 * i + HK * h, a + 2 * k, kb + 2 * k, DESC_S, sub > 0 || k > 0);
            }
            commit(&s_done[2 * i + h]);
            if (h == 1) commit(&empty[b]);
        };
        if (n > 0) scores(0);
        for (int u = 0; u < 2 * n && ok; ++u) {
            const int h = u & 1;
            // the next scores while this step's exponentials are formed; but where the pipelines take turns
            // the next tile's keys may be far, and this tile's values are released first
            const bool early = !turns || h == 0;
            if (early && u + 1 < 2 * n) scores(u + 1);
            if (!ok) break;
            const int unit = 2 * tile_of(i, u >> 1) + 1, b = unit % BUFFERS;
            const unsigned long long vb = value_desc(ring + b * BUFFER);
            if (h == 0) landed(unit);
            if (!passed(&p_ready[2 * i + h], (u >> 1) & 1)) break;
#pragma unroll
            for (int k = 0; k < HK / 16; ++k)
                umma_a_tmem(tmem + O_COL + D * i, tmem + 128 * i + HK * h + 8 * k,
                            vb + (unsigned long long)((h * (HK / 16) + k) * 2048 >> 4), DESC_O,
                            u > 0 || k > 0);
            commit(&o_done[2 * i + h]);
            if (h == 1) commit(&empty[b]);
            if (!early && u + 1 < 2 * n) scores(u + 1);
        }
        // what is issued, the last buffers' commits with it, ends before the block does
        commit(&drained[i]);
        wait(&drained[i], 0, status);
        __syncwarp();
    } else {
        // ------------------------------------------------------------------ softmax
        const unsigned lanes = (unsigned)((warp & 3) * 32) << 16;
        const unsigned s_addr = tmem + 128 * x + 32 * half + lanes;
        const unsigned p_addr = tmem + 128 * x + 16 * half + lanes;
        const unsigned o_addr = tmem + O_COL + D * x + D / 2 * half + lanes;
        const int pair = 1 + 4 * x + (warp & 3);          // the barrier of the two warps of the same rows
        float* mine = exchange + (2 * x + half) * LANES + rowi;
        float* other = exchange + (2 * x + (half ^ 1)) * LANES + rowi;
        const float sl = scale * 1.4426950408889634f;
        float m_ref = -INFINITY, l_run = 0.0f;
        // step u, as above; EDGE: keys are hidden (a form of its own, so that the others' code is free of it)
        auto step = [&](int u, auto edge) {
            constexpr bool EDGE = decltype(edge)::value;
            const int h = u & 1, t = tile_of(x, u >> 1), kt = it.begin + t * KT;
            if (ok) ok = wait(&s_done[2 * x + h], (u >> 1) & 1, status);
            __syncwarp();
            after_sync();
            unsigned sv[32];
            tmem_load_32cols(s_addr + HK * h, sv);
            tmem_wait_loads();
            // keys behind the range, or without a page, are not seen
            unsigned gone = 0;                            // boxes without a page
            if constexpr (EDGE) {
                const int key = kt + lane * box;
                gone = __ballot_sync(0xffffffffu, lane < boxes && key < it.end && page_at(key) < 0);
                const int n = HK * h + 32 * half + lane;
                const unsigned seen =
                    __ballot_sync(0xffffffffu, kt + n < it.end && !(gone >> (n / box) & 1));
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (!(seen >> i & 1)) sv[i] = 0xff800000u;
            }
            float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < 32; i += 8)
#pragma unroll
                for (int c = 0; c < 4; ++c) m4[c] = max_three(m4[c], sv[i + 2 * c], sv[i + 2 * c + 1]);
            const float m = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
            if (any_of_pair(pair, (m - m_ref) * sl > RAISE)) {
                if (u > 0) {                              // no product adds to the results meanwhile
                    if (ok) ok = wait(&o_done[2 * x + (h ^ 1)], ((u - 1) >> 1) & 1, status);
                    __syncwarp();
                    after_sync();
                }
                *mine = m;
                sync_pair(pair);
                const float top = fmaxf(m, *other);       // of the row
                const bool raise = (top - m_ref) * sl > RAISE;
                const float f = raise ? exp2_fast((m_ref - top) * sl) : 1.0f;
                if (u > 0) {
#pragma unroll 1
                    for (int c = 0; c < D / 32; ++c) {
                        unsigned ov[16];
                        tmem_load_16cols(o_addr + 16 * c, ov);
                        tmem_wait_loads();
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            ov[i] = __float_as_uint(__uint_as_float(ov[i]) * f);
                        tmem_store_16cols(o_addr + 16 * c, ov);
                    }
                    tmem_wait_stores();
                    before_sync();
                }
                l_run *= f;
                if (raise) m_ref = top;
                sync_pair(pair);                          // both halves are rescaled before a product
            }
            const float off = m_ref == -INFINITY ? 0.0f : -m_ref * sl;
            const Two sl2 = two(sl, sl), off2 = two(off, off);
            Two sum2[2] = {two(0.0f, 0.0f), two(0.0f, 0.0f)};
            unsigned pw[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float a, b;
                untwo(fma_two(two(__uint_as_float(sv[2 * i]), __uint_as_float(sv[2 * i + 1])), sl2, off2),
                      a, b);
                a = exp2_fast(a);
                b = exp2_fast(b);
                sum2[i & 1] = add_two(sum2[i & 1], two(a, b));
                pw[i] = pack2(a, b);
            }
            tmem_store_16cols(p_addr + HK * h, pw);
            {
                float a, b;
                untwo(add_two(sum2[0], sum2[1]), a, b);
                l_run += a + b;
            }
            // Values that no row sees may be anything, and 0 * NaN is NaN in the product: the first thread of
            // row i has the values of key i (both pipelines write the same zeros).
            if constexpr (EDGE) {
                if (half == 0 && rowi / HK == h &&
                    (kt + rowi >= it.end || (gone >> (rowi / box) & 1))) {
                    const int unit = 2 * t + 1, b = unit % BUFFERS;
                    landed(unit);
#pragma unroll
                    for (int sub = 0; sub < KS; ++sub) {
                        uint4* v = reinterpret_cast<uint4*>(ring + b * BUFFER + sub * SUB + rowi * 128);
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = make_uint4(0u, 0u, 0u, 0u);
                    }
                    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                }
                __syncwarp();
            }
            tmem_wait_stores();
            before_sync();
            mbar_arrive(&p_ready[2 * x + h]);
        };
        for (int u = 0; u < 2 * n_of[x]; ++u) {
            if (missing || it.begin + (tile_of(x, u >> 1) + 1) * KT > it.end) step(u, Truth<true>());
            else step(u, Truth<false>());
        }
        if (n_of[x] > 0) {
            if (ok) ok = wait(&o_done[2 * x + 1], (n_of[x] - 1) & 1, status);
            __syncwarp();
            after_sync();
        }
        // The rows' results go out by way of the ring (which nobody reads any more when both pipelines
        // are through): half a row is one bulk copy of its own.
        *mine = l_run;
        asm volatile("bar.sync 9, %0;\n" ::"n"(SOFTMAX_WARPS * 32) : "memory");
        const size_t at = (size_t)(it.base + x * LANES + rowi) * kv_heads + hk;
        if (n_of[x] > 0) {
            unsigned char* res = ring + (x * LANES + rowi) * ROW_BYTES + half * D * 2;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                unsigned ov[16];
                tmem_load_16cols(o_addr + 16 * c, ov);
                tmem_wait_loads();
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<uint4*>(res + 64 * c + 16 * i) =
                        make_uint4(ov[4 * i], ov[4 * i + 1], ov[4 * i + 2], ov[4 * i + 3]);
            }
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            if (ok && live)
                asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;\n"
                             ::"l"(partial_acc + at * D + D / 2 * half), "r"(smem_u32(res)), "n"(D * 2)
                             : "memory");
            asm volatile("cp.async.bulk.commit_group;\n" ::: "memory");
        }
        // (nothing where a wait ran out: such a row's results are those of the other ranges)
        if (live && half == 0)
            partial_ml[at] = n_of[x] > 0 && ok ? make_float2(m_ref * sl, l_run + *other)
                                               : make_float2(-INFINITY, 0.0f);
        asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory");
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

// Items of shared keys; q, pages in 16-byte pieces.  `turns`: some have two places.
DE_EXPORT int de_shared_tcgen05(const void* q, int q_stride, const void* k_pages, const void* v_pages,
                                const int* block_table, int table_stride, int num_pages,
                                const int* seq_slot, const int* seq_pos0, const int* items,
                                int num_items, int turns, float* partial_acc, float* partial_ml, int heads,
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
    const auto kernel = turns ? shared_tcgen05_kernel<true> : shared_tcgen05_kernel<false>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    if (e != cudaSuccess) return (int)e;
    return de_launch(kernel, dim3((unsigned)num_items * kv_heads), dim3(THREADS), SMEM,
                     (cudaStream_t)stream, (const __nv_bfloat16*)q, q_stride, map_k, map_v,
                     block_table, table_stride, num_pages, seq_slot, (const Item*)items, partial_acc, (float2*)partial_ml, heads, kv_heads, page,
                     scale, status);
}
