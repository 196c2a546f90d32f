// The weights of a prompt's last rows on tcgen05: many rows (token, head) of q against all cached keys, without output.
// Included by attention_weights.cu, whose arguments it takes.
//
// Both passes are one kernel. The rows of q stay in shared memory (up to 512 of them), the keys pass by in tiles of 128 that TMA
// brings from the pages, and every (tile, 128 rows) is one product of 128 x 128 in tensor memory, of which four are in flight.
//
//   SUM false: S = Q K^T, a thread a row (and half of a tile's keys): its running maximum and sum over a stretch of keys
//   SUM true:  S = K Q^T, a thread a key (and half of the rows): the sum of its weights 2^(s - max - log2 sum) over the rows,
//              in registers; the stretches' statistics are joined by every block for itself
//
// Sixteen warps of exponentials, in two sides that take the tiles in turn, one warp that brings keys, one that issues products.
// With eight warps on halves of one tile, all were in the same phase and the exponentials' unit idled half of the time. Measured
// over 64 rows (256 with their heads) of four prompts of 9,001 to 16,384 keys and 8 kv heads: 300 us on mma.sync, 145 with eight
// warps here, 119 with stretches of equal work, 94 with sixteen warps and a ring as deep as shared memory allows, 90 with a shorter
// start. What bounds it: the exponentials of both passes take 48 us (16 a cycle and multiprocessor; their unit is busy 69% and 62% of
// the time), the products, whose two operands pass through shared memory, about as long beside them, the start of both kernels 14.
// One in four to eight of the exponentials as a polynomial on the other pipes made it slower (93 to 100 us).
#pragma once
#include <cuda.h>

#define WT_KEYS 128
#define WT_WORKERS 512                 // threads that work on scores: two sides of two halves of 128
#define WT_THREADS (WT_WORKERS + 64)
#define WT_WAIT_CYCLES 2000000000ll

__device__ __forceinline__ void wt_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void wt_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void wt_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool wt_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// Every wait has an end: past it the flag is set, and all roles run through to the block's last barrier without working.
__device__ __forceinline__ bool wt_wait(uint32_t bar, uint32_t parity, volatile int* gave_up) {
    if (wt_try(bar, parity)) return true;
    const long long t0 = clock64();
    while (true) {
        if (wt_try(bar, parity)) return true;
        if (*gave_up) return false;
        if (clock64() - t0 > WT_WAIT_CYCLES) {
            *gave_up = 1;
            return false;
        }
    }
}
__device__ __forceinline__ void wt_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(dst), "l"((uint64_t)map), "r"(bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void wt_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wt_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wt_fence_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void wt_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void wt_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
// 32 columns of this thread's lane, without waiting.
__device__ __forceinline__ void wt_read32(uint32_t addr, float* r) {
    uint32_t* u = reinterpret_cast<uint32_t*>(r);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
          "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
          "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
          "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
        : "r"(addr));
}
// The loads of these 32 columns are there; nothing uses them before.
__device__ __forceinline__ void wt_read_wait(float* r) {
    uint32_t* u = reinterpret_cast<uint32_t*>(r);
    asm volatile("tcgen05.wait::ld.sync.aligned;"
        : "+r"(u[0]), "+r"(u[1]), "+r"(u[2]), "+r"(u[3]), "+r"(u[4]), "+r"(u[5]), "+r"(u[6]), "+r"(u[7]), "+r"(u[8]),
          "+r"(u[9]), "+r"(u[10]), "+r"(u[11]), "+r"(u[12]), "+r"(u[13]), "+r"(u[14]), "+r"(u[15]), "+r"(u[16]),
          "+r"(u[17]), "+r"(u[18]), "+r"(u[19]), "+r"(u[20]), "+r"(u[21]), "+r"(u[22]), "+r"(u[23]), "+r"(u[24]),
          "+r"(u[25]), "+r"(u[26]), "+r"(u[27]), "+r"(u[28]), "+r"(u[29]), "+r"(u[30]), "+r"(u[31])
        :: "memory");
}
// Rows of 128 bytes, 128-byte swizzle, 1,024 bytes between groups of eight rows: as TMA writes the keys and the workers q.
__device__ __forceinline__ uint64_t wt_desc(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ void wt_workers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(WT_WORKERS) : "memory"); }

template <int HD, int RT> struct WtPlan {
    static constexpr int KB = HD / 64;                                        // 64-channel blocks of a row
    static constexpr uint32_t TILE = 128u * 128u * KB;                        // 128 rows or keys
    static constexpr int ROOM = (227 * 1024 - 1280 - RT * 1024 * 3) / (int)TILE - RT;
    static constexpr int STAGES = ROOM < 6 ? ROOM : 6;                        // what the rows of q leave room for
    static constexpr size_t SMEM = 1024 + (size_t)TILE * (RT + STAGES) + 256 + RT * 128 * 8 * 3;
    static constexpr int BUFS = 2;                                            // products of a side in tensor memory
    static_assert(STAGES >= 2 && SMEM + 64 <= 227 * 1024, "a tile for each side, within a block's shared memory");
};

// Which stretch a block has. All sequences' key tiles are cut into stretches of the same number of tiles, the smallest for which they
// are no more than the blocks of a kv head (and none has more than the statistics have room for): sequences of unequal
// lengths keep all multiprocessors busy to the end (four prompts of 9,001 to 16,384: 142 us with stretches of one length
// made for the longest, 119 with these).
struct WtShare {
    int seq, split, tiles, splits;             // tiles: of a stretch; splits: stretches of the sequence
};
__device__ __forceinline__ WtShare wt_share(const WeightArgs& a, int m0, int block, int blocks) {        // by a whole warp, the same in every lane
    const int lane = threadIdx.x & 31;
    if (a.n_seqs == 1) {                       // (a microsecond less)
        const Seq s = seq_of(a, 0);
        const int total = m0 < s.rows ? (s.length + WT_KEYS - 1) / WT_KEYS : 0, tiles = max(1, (total + blocks - 1) / blocks);
        return {block * tiles < total ? 0 : -1, block, tiles, (total + tiles - 1) / tiles};
    }
    auto look_up = [&](int i) {
        if (i >= a.n_seqs) return 0;
        const Seq s = seq_of(a, i);
        return m0 < s.rows ? (s.length + WT_KEYS - 1) / WT_KEYS : 0;
    };
    const int own = look_up(lane);             // the first 32 sequences are looked up once
    auto tiles_of = [&](int i) { return i < 32 ? own : look_up(i); };
    int total = 0, longest = 0;
    for (int i = lane; i < a.n_seqs; i += 32) {
        const int k = tiles_of(i);
        total += k, longest = max(longest, k);
    }
    total = __reduce_add_sync(0xffffffffu, total);
    // Between what would fill all blocks and what always fits: every sequence has at most one stretch that is not full, and one of the
    // longest's length each fits too.
    int tiles = max(1, (total + blocks - 1) / blocks), fits = max(tiles, __reduce_max_sync(0xffffffffu, longest));
    if (a.n_splits > 1) fits = max(tiles, min(fits, (total + a.n_splits - 2) / (a.n_splits - 1)));
    while (tiles < fits) {
        const int half = (tiles + fits) / 2;
        int n = 0, most = 0;
        for (int i = lane; i < a.n_seqs; i += 32) {
            const int k = (tiles_of(i) + half - 1) / half;
            n += k, most = max(most, k);
        }
        if (__reduce_add_sync(0xffffffffu, n) <= blocks && __reduce_max_sync(0xffffffffu, most) <= a.n_splits) fits = half;
        else tiles = half + 1;
    }
    WtShare w = {-1, 0, tiles, 0};
    int before = 0;
    for (int i0 = 0; i0 < a.n_seqs && w.seq < 0; i0 += 32) {
        const int k = (tiles_of(i0 + lane) + tiles - 1) / tiles;
        int incl = k;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += t;
        }
        const unsigned int mine = __ballot_sync(0xffffffffu, block >= before + incl - k && block < before + incl);
        if (mine) {
            const int who = __ffs(mine) - 1;
            w.seq = i0 + who;
            w.split = block - before - __shfl_sync(0xffffffffu, incl - k, who);
            w.splits = __shfl_sync(0xffffffffu, k, who);
        }
        before += __shfl_sync(0xffffffffu, incl, 31);
    }
    return w;
}

// grid (blocks of a kv head, kv heads). RT: tiles of 128 rows, from row m0 of a sequence on.
template <int HD, int RT, bool SUM>
__global__ void __launch_bounds__(WT_THREADS, 1) weights_tc_kernel(const __grid_constant__ CUtensorMap map, WeightArgs a, int m0, int* err) {
    using P = WtPlan<HD, RT>;
    constexpr int KB = P::KB, STAGES = P::STAGES, BUFS = P::BUFS;
    constexpr uint32_t TILE = P::TILE, BLOCK = 128u * 128u;
    extern __shared__ uint8_t wt_raw[];
    const uint32_t base = ((uint32_t)__cvta_generic_to_shared(wt_raw) + 1023u) & ~1023u;
    uint8_t* const gbase = wt_raw + (base - (uint32_t)__cvta_generic_to_shared(wt_raw));
    const uint32_t sQ = base, sK = sQ + RT * TILE, bars = sK + STAGES * TILE;
    uint8_t* const tail = gbase + (bars - base);
    uint32_t* const slot = reinterpret_cast<uint32_t*>(tail + 24 * 8);
    volatile int* const gave_up = reinterpret_cast<volatile int*>(slot + 1);
    float* const ref_s = reinterpret_cast<float*>(tail + 256);                // SUM: [RT * 128] maximum + log2 sum of a row, and
    int* const place_s = reinterpret_cast<int*>(ref_s + RT * 128);            // the last place it sees
    float* const half_s = reinterpret_cast<float*>(place_s + RT * 128);       // [2 sides][2 tiles][128]: the second half's sums
    float2* const rows_s = reinterpret_cast<float2*>(tail + 256);             // else: [3][RT * 128] the others' maxima and sums
    auto k_full = [&](int s) { return bars + 8u * s; };
    auto k_empty = [&](int s) { return bars + 8u * (STAGES + s); };
    auto s_full = [&](int b) { return bars + 8u * (2 * STAGES + b); };
    auto s_empty = [&](int b) { return bars + 8u * (2 * STAGES + 2 * BUFS + b); };
    const uint32_t q_ready = bars + 8u * (2 * STAGES + 4 * BUFS);             // 21 barriers at most
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    __shared__ WtShare share;
    if (warp == 0) {                                                          // the other warps prepare what does not depend on it
        const WtShare mine = wt_share(a, m0, blockIdx.x, gridDim.x);
        if (lane == 0) share = mine;
    }
    if (threadIdx.x == 32) {
        for (int i = 0; i < STAGES; ++i) wt_init(k_full(i), 1), wt_init(k_empty(i), 1);
        for (int i = 0; i < 2 * BUFS; ++i) wt_init(s_full(i), 1), wt_init(s_empty(i), WT_WORKERS / 64);
        wt_init(q_ready, WT_WORKERS);
        *gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        wt_fence_smem();
    }
    if (warp == WT_WORKERS / 32 + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"((uint32_t)__cvta_generic_to_shared(slot)), "r"(256u * BUFS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    wt_fence_before();
    __syncthreads();
    wt_fence_after();
    // Only now may the next kernel begin: one that takes tensor memory before it waits for this one must not find it before this block.
    pdl_launch_dependents();
    const uint32_t tmem = *slot;
    if (share.seq < 0) {                                                      // more blocks than stretches: the same for the whole block
        if (warp == WT_WORKERS / 32 + 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256u * BUFS) : "memory");
        return;
    }
    const int split = share.split, seq = share.seq, kvh = blockIdx.y, pair = seq * a.kv_heads + kvh;
    const Seq s = seq_of(a, seq);
    const int first = split * share.tiles * WT_KEYS, last = min(s.length, first + share.tiles * WT_KEYS);
    const int group = a.heads / a.kv_heads, group_rows = a.max_new * group;
    const int n_tiles = (last - first + WT_KEYS - 1) / WT_KEYS;
    const int rows = min(s.rows - m0, RT * 128), row_tiles = (rows + 127) / 128;
    const int* const pages = a.table + (size_t)seq * a.width;
    auto page_at = [&](int key) {                                             // the page of a key of this stretch, -1: none
        const int page = key < last ? pages[key / CML_PAGE] : -1;
        return page < a.n_pages ? page : -1;
    };
    if (warp == WT_WORKERS / 32) {
        if (lane == 0) {
            int issued = 0;
            for (int t = 0; t < n_tiles; ++t) {
                const int st = t % STAGES;
                if (!wt_wait(k_empty(st), ((uint32_t)(t / STAGES) & 1u) ^ 1u, gave_up)) break;
                wt_expect(k_full(st), TILE);
#pragma unroll
                for (int h = 0; h < 2; ++h) {                                 // a page that is none: any, its keys are masked
                    const int y = (max(page_at(first + t * WT_KEYS + h * CML_PAGE), 0) * a.kv_heads + kvh) * CML_PAGE;
#pragma unroll
                    for (int b = 0; b < KB; ++b) wt_load(sK + st * TILE + b * BLOCK + h * (BLOCK / 2), &map, k_full(st), b * 64, y);
                }
                issued = t + 1;
            }
            if (*gave_up) {                                                   // copies in flight land before the block ends
                for (int t = max(0, issued - STAGES); t < issued; ++t) {
                    const long long t0 = clock64();
                    while (!wt_try(k_full(t % STAGES), (uint32_t)(t / STAGES) & 1u) && clock64() - t0 < 20000000ll) {}
                }
            }
        }
    } else if (warp == WT_WORKERS / 32 + 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
            bool ok = wt_wait(q_ready, 0, gave_up);
            int item = 0;                                                     // of a side: (tile, 128 rows) in turn
            for (int t0 = 0; t0 < n_tiles && ok; t0 += 2) {
                for (int rt = 0; rt < row_tiles && ok; ++rt, ++item) {
                    for (int side = 0; side < 2 && t0 + side < n_tiles; ++side) {
                        const int t = t0 + side, st = t % STAGES, buf = side * BUFS + item % BUFS;
                        if (rt == 0) ok = wt_wait(k_full(st), (uint32_t)(t / STAGES) & 1u, gave_up);
                        if (ok) ok = wt_wait(s_empty(buf), ((uint32_t)(item / BUFS) & 1u) ^ 1u, gave_up);
                        if (!ok) break;
                        wt_fence_after();
#pragma unroll
                        for (int b = 0; b < KB; ++b) {
                            const uint64_t q = wt_desc(sQ + rt * TILE + b * BLOCK), k = wt_desc(sK + st * TILE + b * BLOCK);
#pragma unroll
                            for (int c = 0; c < 4; ++c)
                                wt_mma(tmem + buf * 128, (SUM ? k : q) + (uint64_t)(c * 2), (SUM ? q : k) + (uint64_t)(c * 2), idesc, (b | c) ? 1u : 0u);
                        }
                        wt_commit(s_full(buf));
                        if (rt == row_tiles - 1) wt_commit(k_empty(st));
                    }
                }
            }
        }
    } else {
        // q into its tiles, zeros where there is no row
        constexpr int ROW = KB * 8, STEP = WT_WORKERS / ROW;                  // 16-byte pieces of a row; rows between this thread's
        const int piece = threadIdx.x % ROW, x0 = threadIdx.x / ROW, j_step = STEP / group, h_step = STEP - j_step * group;
        int j = (m0 + x0) / group, h = m0 + x0 - j * group;                   // token and head of row x0, walked without further divisions
        const bf16* const q0 = (const bf16*)a.q + (long long)s.row0 * a.q_stride + (long long)kvh * group * HD + piece * 8;
#pragma unroll 4
        for (int m = x0; m < row_tiles * 128; m += STEP) {
            const bool in = m < rows;
            const int r = m % 128;
            cp_async16_or_zero(sQ + (m / 128) * TILE + (piece / 8) * BLOCK + (r >> 3) * 1024 + (r & 7) * 128 + (((piece & 7) ^ (r & 7)) << 4),
                               in ? q0 + (long long)j * a.q_stride + h * HD : q0, in);
            j += j_step, h += h_step;
            if (h >= group) h -= group, ++j;
        }
        cp_async_commit();
        if (SUM) {                                                            // the stretches of every row joined, in their order
            const int splits = share.splits;
            for (int m = threadIdx.x; m < RT * 128; m += WT_WORKERS) {
                float top = -CUDART_INF_F, sum = 0.f;
                if (m < rows) {
                    const float* st = a.stats + ((size_t)pair * a.n_splits * group_rows + m0 + m) * 2;
                    for (int i0 = 0; i0 < splits; i0 += 8) {                  // eight at a time, which are asked for at once
                        float2 x[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            x[i] = i0 + i < splits ? *reinterpret_cast<const float2*>(st + (size_t)(i0 + i) * group_rows * 2) : make_float2(-CUDART_INF_F, 0.f);
                        float most = top;
#pragma unroll
                        for (int i = 0; i < 8; ++i) most = fmaxf(most, x[i].x);
                        if (top != -CUDART_INF_F) sum *= exp2f(top - most);
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (x[i].x != -CUDART_INF_F) sum += exp2f(x[i].x - most) * x[i].y;
                        top = most;
                    }
                }
                ref_s[m] = top == -CUDART_INF_F ? CUDART_INF_F : top + log2f(sum);
                place_s[m] = m < rows ? s.start + (m0 + m) / group : -1;
            }
        }
        cp_async_wait<0>();
        wt_fence_smem();
        wt_arrive(q_ready);
        wt_workers_sync();                                                    // ref_s is whole
        const int side = warp >> 3, half = (warp >> 2) & 1, mine = (warp & 3) * 32 + lane;    // mine: this thread's lane of tensor memory
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        float top[RT], sum[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) top[r] = -CUDART_INF_F, sum[r] = 0.f;
        bool ok = true;
        int item = 0;
        for (int t = side; t < n_tiles; t += 2) {                             // (after a wait that ran out: without working)
            const int key0 = first + t * WT_KEYS;
            const int page0 = page_at(key0), page1 = page_at(key0 + CML_PAGE);
            // every row sees every key of the tile
            const bool whole = page0 >= 0 && page1 >= 0 && key0 + WT_KEYS <= last && key0 + WT_KEYS - 1 <= s.start;
            float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                if (rt >= row_tiles) break;
                const int buf = side * BUFS + item % BUFS;
                ok = ok && __all_sync(0xffffffffu, wt_wait(s_full(buf), (uint32_t)(item / BUFS) & 1u, gave_up));
                ++item;
                if (!ok) break;
                wt_fence_after();
                float x[64];
                wt_read32(tmem + buf * 128 + lanes + half * 64, x);
                wt_read32(tmem + buf * 128 + lanes + half * 64 + 32, x + 32);
                wt_read_wait(x);
                wt_read_wait(x + 32);
                wt_fence_before();
                __syncwarp();
                if (lane == 0) wt_arrive(s_empty(buf));                       // read: the next product may come
                if (!SUM) {                                                   // this thread's row, the keys of one page
                    if (!whole) {
                        const int seen = (half ? page1 : page0) < 0 ? -1 : min(last - 1, s.start + (m0 + rt * 128 + mine) / group) - key0 - half * 64;
#pragma unroll
                        for (int i = 0; i < 64; ++i) x[i] = i <= seen ? x[i] : -CUDART_INF_F;
                    }
                    float m[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) m[i] = x[i];
#pragma unroll
                    for (int i = 4; i < 64; ++i) m[i & 3] = fmaxf(m[i & 3], x[i]);
                    const float most = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])) * a.scale;
                    const bool passed = most > top[rt] + 6.f;
                    if (__any_sync(0xffffffffu, passed)) {                    // the reference moves only when a row passes it by 2^6
                        sum[rt] *= passed ? fast_exp2(top[rt] - most) : 1.f;
                        top[rt] = passed ? most : top[rt];
                    }
                    const float ref = top[rt] == -CUDART_INF_F ? 0.f : top[rt];
                    part[0] = part[1] = part[2] = part[3] = 0.f;
#pragma unroll
                    for (int i = 0; i < 64; ++i) part[i & 3] += fast_exp2(fmaf(x[i], a.scale, -ref));
                    sum[rt] += (part[0] + part[1]) + (part[2] + part[3]);
                } else if (whole && rt * 128 + half * 64 + 64 <= rows) {    // this thread's key, 64 rows
#pragma unroll
                    for (int i = 0; i < 64; i += 4) {
                        const float4 ref = *reinterpret_cast<const float4*>(ref_s + rt * 128 + half * 64 + i);
                        part[0] += fast_exp2(fmaf(x[i], a.scale, -ref.x));
                        part[1] += fast_exp2(fmaf(x[i + 1], a.scale, -ref.y));
                        part[2] += fast_exp2(fmaf(x[i + 2], a.scale, -ref.z));
                        part[3] += fast_exp2(fmaf(x[i + 3], a.scale, -ref.w));
                    }
                } else {                                                      // some rows see less (or are none: zero times an infinite key is no zero)
#pragma unroll
                    for (int i = 0; i < 64; ++i)
                        if (key0 + mine <= place_s[rt * 128 + half * 64 + i]) part[i & 3] += fast_exp2(fmaf(x[i], a.scale, -ref_s[rt * 128 + half * 64 + i]));
                }
            }
            if (SUM) {                                                        // the two halves of the rows, then the key's score
                const float gained = (part[0] + part[1]) + (part[2] + part[3]);
                float* const other = half_s + (side * 2 + ((t >> 1) & 1)) * 128 + mine;
                if (half) *other = gained;
                if (side) asm volatile("bar.sync 3, %0;" ::"n"(WT_WORKERS / 2) : "memory");
                else asm volatile("bar.sync 2, %0;" ::"n"(WT_WORKERS / 2) : "memory");
                const int key = key0 + mine, page = mine < CML_PAGE ? page0 : page1;
                if (!half && ok && key < last && page >= 0) {
                    const size_t at = ((size_t)page * a.kv_heads + kvh) * CML_PAGE + key % CML_PAGE;
                    const float old = m0 ? a.scores_out[at] : key < s.old ? a.scores[at] : 0.f;      // (earlier rows' weights are there)
                    a.scores_out[at] = old + (gained + *other);
                }
            }
        }
        if (!SUM) {                                                           // the sides' and halves' keys together
            const int who = warp >> 2;
            if (who) {
#pragma unroll
                for (int r = 0; r < RT; ++r) rows_s[((who - 1) * RT + r) * 128 + mine] = make_float2(top[r], sum[r]);
            }
            wt_workers_sync();
            if (!who) {
                float* const out = a.stats + (((size_t)pair * a.n_splits + split) * group_rows + m0) * 2;
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const int m = r * 128 + mine;
                    if (m >= rows) break;
                    float most = top[r], l = 0.f;
#pragma unroll
                    for (int w = 0; w < 3; ++w) most = fmaxf(most, rows_s[(w * RT + r) * 128 + mine].x);
                    if (top[r] != -CUDART_INF_F) l += fast_exp2(top[r] - most) * sum[r];
#pragma unroll
                    for (int w = 0; w < 3; ++w) {
                        const float2 o = rows_s[(w * RT + r) * 128 + mine];
                        if (o.x != -CUDART_INF_F) l += fast_exp2(o.x - most) * o.y;
                    }
                    *reinterpret_cast<float2*>(out + m * 2) = make_float2(most, l);
                }
            }
        }
    }
    wt_fence_before();
    __syncthreads();
    if (warp == WT_WORKERS / 32 + 1) {
        wt_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256u * BUFS) : "memory");
    }
    if (threadIdx.x == 0 && *gave_up) atomicExch(err, 4);
}

typedef CUresult (*WtEncode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                             const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static WtEncode wt_encode() {
    static WtEncode fn = nullptr;
    if (!fn) {
        void* q = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &q, cudaEnableDefault, &r) == cudaSuccess && r == cudaDriverEntryPointSuccess) fn = (WtEncode)q;
    }
    return fn;
}

template <int HD, int RT>
static cudaError_t launch_tc_rows(const CUtensorMap& map, const WeightArgs& a, int m0, int* err, cudaStream_t s) {
    constexpr size_t smem = WtPlan<HD, RT>::SMEM;
    cudaError_t e = cml_allow_smem<weights_tc_kernel<HD, RT, false>>(smem);
    if (e == cudaSuccess) e = cml_allow_smem<weights_tc_kernel<HD, RT, true>>(smem);
    if (e != cudaSuccess) return e;
    // one block for every multiprocessor in all, one for every sequence at least; n_splits of a sequence at most, so that the others have one
    const dim3 grid((unsigned)(a.n_splits + a.n_seqs - 1), (unsigned)a.kv_heads);
    e = launch_pdl(weights_tc_kernel<HD, RT, false>, grid, dim3(WT_THREADS), smem, s, map, a, m0, err);
    if (e != cudaSuccess) return e;
    return launch_pdl(weights_tc_kernel<HD, RT, true>, grid, dim3(WT_THREADS), smem, s, map, a, m0, err);
}

template <int HD>
static cudaError_t launch_tc(const WeightArgs& a, int* err, cudaStream_t s) {
    const WtEncode encode = wt_encode();
    if (!encode) return cudaErrorNotSupported;
    CUtensorMap map;                                                          // the pool as a matrix [pages * kv heads * 64, HD], boxes of a page and 64 channels
    const cuuint64_t dims[2] = {(cuuint64_t)HD, (cuuint64_t)a.n_pages * a.kv_heads * CML_PAGE}, strides[1] = {(cuuint64_t)HD * 2};
    const cuuint32_t box[2] = {64, CML_PAGE}, steps[2] = {1, 1};
    if (encode(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(a.k), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return cudaErrorInvalidValue;
    // up to 512 rows at a time: as many as shared memory holds beside the keys
    const int rows = a.max_new * (a.heads / a.kv_heads);
    cudaError_t e = cudaSuccess;
    for (int m0 = 0; m0 < rows && e == cudaSuccess; m0 += 512) {
        const int left = rows - m0;
        e = left <= 128 ? launch_tc_rows<HD, 1>(map, a, m0, err, s) : left <= 256 ? launch_tc_rows<HD, 2>(map, a, m0, err, s) : launch_tc_rows<HD, 4>(map, a, m0, err, s);
    }
    return e;
}
