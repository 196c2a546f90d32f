// Eviction from the paged cache by accumulated attention weight.
//
// For every unit (cache entry, sequence, kv head) of length L the first `first` places, the last `recent` places and
// those of the middle with the largest scores stay, M = min(keep, L) in all; among equal scores the lower place stays,
// and a score that is not a number counts as the lowest. The places that stay move up, in order, to the places
// 0 .. M - 1 of the out table's pages with their values and scores. With rotary frequencies the keys are turned by the
// angle of the distance they move, so that a key's place is again its position: (a, b) at place p, moved to j, becomes
// (a cos t - b sin t, b cos t + a sin t) with t = (j - p) f. The angle is formed in double and reduced to one turn
// before it is rounded (positions reach 2^20, where a float product would be off by 0.06 of a radian); the turn itself is
// float, and a bfloat16 key is rounded once per move.
//
// Two launches. (1) A block per unit finds the score at the border by its digits (four passes of 8 bits over the
// unit's scores) and lists the places that stay in order. (2) The rows move through shared memory. The out table may be
// the table itself: place kept[j] >= j, so the rows of an output page come from that page or later ones, and an output
// page may be written once the rows of every earlier page (and its own) are read. A cluster of blocks shares a unit and
// goes page by page in rounds; every block waits for its own rows and then at the cluster's barrier before it writes.
#include "common.cuh"
#include <cooperative_groups.h>
#include <math_constants.h>
namespace cg = cooperative_groups;

#define EV_SELECT_THREADS 512
#define EV_MOVE_THREADS 256
#define EV_MAX_TEAM 8
#define EV_STAGES 4             // rounds of rows in flight

struct EvictArgs {
    void* k;
    void* v;                     // null: the values live in the key rows
    float* scores;
    const int* table;
    int width;
    const int* out_table;
    int out_width;
    const int* lengths;
    const int* keeps;
    int* kept;
    int cap;                     // places a unit of `kept` has room for
    int entries, n_pages, n_seqs, heads, k_dim, v_dim;
    int first, recent;
    const float* inv_freq;       // null: keys keep the angle they have
    int rotary_dim, interleaved;
    int tile;                    // rows that a block moves in a round (a divisor of the page)
};

struct Unit {
    int entry, seq, head, length, keep;
};

__device__ __forceinline__ Unit unit_of(const EvictArgs& a, int u) {
    Unit x;
    x.head = u % a.heads;
    const int es = u / a.heads;
    x.seq = es % a.n_seqs;
    x.entry = es / a.n_seqs;
    x.length = max(0, min(a.lengths[x.seq], a.width * CML_PAGE));
    x.keep = max(0, min(min(a.keeps[x.seq], x.length), min(a.cap, a.out_width * CML_PAGE)));
    return x;
}

// Larger score, larger number; -0 and 0 are equal, not-a-number lies below everything.
__device__ __forceinline__ unsigned int score_key(float s) {
    if (s != s) return 0u;
    const unsigned int u = __float_as_uint(s + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__global__ void __launch_bounds__(EV_SELECT_THREADS) evict_select_kernel(EvictArgs a) {
    __shared__ unsigned int hist[256];
    __shared__ unsigned int s_prefix, s_need;
    __shared__ int s_kept[EV_SELECT_THREADS / 32], s_ties[EV_SELECT_THREADS / 32];
    pdl_wait();
    pdl_launch_dependents();
    const Unit x = unit_of(a, blockIdx.x);
    int* kept = a.kept + (size_t)blockIdx.x * a.cap;
    if (x.keep == x.length) {                                     // everything stays
        for (int j = threadIdx.x; j < x.keep; j += blockDim.x) kept[j] = j;
        return;
    }
    const int first = min(a.first, x.keep), recent = min(a.recent, x.keep - first);
    const int lo = first, hi = x.length - recent;                 // the middle, which competes
    const int want = x.keep - first - recent;
    const int* pages = a.table + (size_t)x.seq * a.width;
    const float* scores = a.scores + (size_t)x.entry * a.n_pages * a.heads * CML_PAGE;
    auto key_at = [&](int place) {
        const int page = pages[place / CML_PAGE];
        if (page < 0 || page >= a.n_pages) return 0u;
        return score_key(scores[((size_t)page * a.heads + x.head) * CML_PAGE + place % CML_PAGE]);
    };
    // the key of the want-th largest, digit by digit
    unsigned int prefix = 0u, need = (unsigned int)want;
    if (want > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int b = threadIdx.x; b < 256; b += blockDim.x) hist[b] = 0u;
            __syncthreads();
            const unsigned int mask = shift == 24 ? 0u : (~0u << (shift + 8));
            for (int p = lo + threadIdx.x; p < hi; p += blockDim.x) {
                const unsigned int k = key_at(p);
                if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1u);
            }
            __syncthreads();
            if (threadIdx.x < 32) {                               // a lane sums eight bins from the top
                const int lane = threadIdx.x;
                unsigned int mine = 0u;
                for (int b = 0; b < 8; ++b) mine += hist[255 - (lane * 8 + b)];
                unsigned int incl = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned int t = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += t;
                }
                const unsigned int who = __ballot_sync(0xffffffffu, incl >= need);
                if (who != 0u && lane == __ffs(who) - 1) {
                    unsigned int before = incl - mine;
                    int b = 0;
                    for (; b < 7; ++b) {
                        const unsigned int c = hist[255 - (lane * 8 + b)];
                        if (before + c >= need) break;
                        before += c;
                    }
                    s_prefix = prefix | ((unsigned int)(255 - (lane * 8 + b)) << shift);
                    s_need = need - before;                       // how many of the border's digit are still wanted
                }
            }
            __syncthreads();
            prefix = s_prefix;
            need = s_need;
            __syncthreads();
        }
    }
    // the places that stay, in order; of those at the border the `need` lowest
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    int done = 0, ties_done = 0;
    for (int p0 = 0; p0 < x.length; p0 += blockDim.x) {
        const int p = p0 + threadIdx.x;
        const bool in = p < x.length;
        const bool outer = in && (p < lo || p >= hi);
        bool above = false, tie = false;
        if (in && !outer && want > 0) {
            const unsigned int k = key_at(p);
            above = k > prefix;
            tie = k == prefix;
        }
        const unsigned int tie_mask = __ballot_sync(0xffffffffu, tie);
        if (lane == 0) s_ties[warp] = __popc(tie_mask);
        __syncthreads();
        int ties_before = ties_done + __popc(tie_mask & ((1u << lane) - 1u)), ties_all = 0;
        for (int w = 0; w < nw; ++w) {
            if (w < warp) ties_before += s_ties[w];
            ties_all += s_ties[w];
        }
        const bool stays = outer || above || (tie && ties_before < (int)need);
        const unsigned int mask = __ballot_sync(0xffffffffu, stays);
        if (lane == 0) s_kept[warp] = __popc(mask);
        __syncthreads();
        int at = done + __popc(mask & ((1u << lane) - 1u)), all = 0;
        for (int w = 0; w < nw; ++w) {
            if (w < warp) at += s_kept[w];
            all += s_kept[w];
        }
        if (stays && at < x.keep) kept[at] = p;
        done += all;
        ties_done += ties_all;
        __syncthreads();
    }
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

template <typename T> struct Chunk {                              // 16 bytes of a row
    static constexpr int N = 16 / sizeof(T);
    T e[N];
};

template <typename T>
__global__ void __launch_bounds__(EV_MOVE_THREADS) evict_move_kernel(EvictArgs a) {
    constexpr int N = Chunk<T>::N;
    extern __shared__ __align__(16) unsigned char raw[];
    pdl_wait();
    pdl_launch_dependents();
    const int team = (int)cg::this_cluster().num_blocks(), rank = (int)cg::this_cluster().block_rank();
    const int u = blockIdx.x / team;
    const Unit x = unit_of(a, u);
    const int* kept = a.kept + (size_t)u * a.cap;
    const int* pages = a.table + (size_t)x.seq * a.width;
    const int* out_pages = a.out_table + (size_t)x.seq * a.out_width;
    const size_t head_rows = (size_t)a.heads * CML_PAGE;
    const size_t entry_rows = (size_t)x.entry * a.n_pages * head_rows;
    T* const k = (T*)a.k + entry_rows * a.k_dim;
    T* const v = a.v ? (T*)a.v + entry_rows * a.v_dim : nullptr;
    float* const scores = a.scores + entry_rows;
    const int k_chunks = a.k_dim / N, v_chunks = v ? a.v_dim / N : 0, chunks = k_chunks + v_chunks;
    const int stage_bytes = a.tile * (chunks * 16 + 8);           // rows, then a score and a source place each
    const int n_tiles = (x.keep + a.tile - 1) / a.tile;
    const int rounds = (n_tiles + team - 1) / team;               // the same for every block of the cluster
    const uint32_t smem = (uint32_t)__cvta_generic_to_shared(raw);
    auto row_at = [&](int place) -> long long {                   // row of the entry's pages, -1: no such page
        const int page = pages[place / CML_PAGE];
        return page < 0 || page >= a.n_pages ? -1ll : (long long)((size_t)page * head_rows + (size_t)x.head * CML_PAGE + place % CML_PAGE);
    };
    auto fetch = [&](int round) {
        const int j0 = (round * team + rank) * a.tile;            // the first output place of this block's rows
        const int rows = round < rounds ? min(a.tile, x.keep - j0) : 0;
        unsigned char* st = raw + (size_t)(round % EV_STAGES) * stage_bytes;
        const uint32_t dst = smem + (uint32_t)(round % EV_STAGES) * stage_bytes;
        for (int c = threadIdx.x; c < rows * chunks; c += blockDim.x) {
            const int j = c / chunks, cc = c - j * chunks;
            const int place = kept[j0 + j];
            const long long row = row_at(place);
            if (row < 0) continue;
            const T* src = cc < k_chunks ? k + row * a.k_dim + cc * N : v + row * a.v_dim + (cc - k_chunks) * N;
            cp_async16(dst + (uint32_t)c * 16, src);
        }
        for (int j = threadIdx.x; j < rows; j += blockDim.x) {
            const int place = kept[j0 + j];
            const long long row = row_at(place);
            float* tail = reinterpret_cast<float*>(st + (size_t)a.tile * chunks * 16);
            tail[2 * j] = row >= 0 ? scores[row] : 0.f;
            reinterpret_cast<int*>(tail)[2 * j + 1] = row >= 0 ? place : -1;
        }
        cp_async_commit();
    };
    constexpr int ahead = EV_STAGES - 1;
    for (int r = 0; r < ahead; ++r) fetch(r);
    const int half = a.rotary_dim / 2;
    for (int round = 0; round < rounds; ++round) {
        fetch(round + ahead);
        asm volatile("cp.async.wait_group 3;" ::: "memory");      // this round's rows: all groups but the three newest
        cg::this_cluster().sync();                                // ... and those of the cluster's other blocks
        const int j0 = (round * team + rank) * a.tile;
        const int rows = min(a.tile, x.keep - j0);
        const unsigned char* st = raw + (size_t)(round % EV_STAGES) * stage_bytes;
        const float* tail = reinterpret_cast<const float*>(st + (size_t)a.tile * chunks * 16);
        const int to = rows > 0 ? out_pages[j0 / CML_PAGE] : -1;
        if (to >= 0 && to < a.n_pages) {
            const size_t out_row0 = (size_t)to * head_rows + (size_t)x.head * CML_PAGE + j0 % CML_PAGE;
            for (int c = threadIdx.x; c < rows * chunks; c += blockDim.x) {
                const int j = c / chunks, cc = c - j * chunks;
                const int place = reinterpret_cast<const int*>(tail)[2 * j + 1];
                if (place < 0) continue;
                const int move = j0 + j - place;
                const size_t row = out_row0 + j;
                Chunk<T> w = *reinterpret_cast<const Chunk<T>*>(st + (size_t)c * 16);
                if (cc < k_chunks) {
                    const int d0 = cc * N;
                    if (a.inv_freq != nullptr && d0 < a.rotary_dim && move != 0) {
                        if (a.interleaved) {
#pragma unroll
                            for (int e = 0; e < N; e += 2) {
                                const double t = (double)move * (double)a.inv_freq[(d0 + e) / 2] * 0.15915494309189535;
                                float sn, cs;
                                sincospif(2.0f * (float)(t - rint(t)), &sn, &cs);
                                const float p = to_f32(w.e[e]), q = to_f32(w.e[e + 1]);
                                w.e[e] = from_f32<T>(p * cs - q * sn);
                                w.e[e + 1] = from_f32<T>(q * cs + p * sn);
                            }
                        } else {
                            const bool low = d0 < half;
                            const Chunk<T> o = *reinterpret_cast<const Chunk<T>*>(st + ((size_t)j * chunks + (low ? d0 + half : d0 - half) / N) * 16);
#pragma unroll
                            for (int e = 0; e < N; ++e) {
                                const double t = (double)move * (double)a.inv_freq[(low ? d0 : d0 - half) + e] * 0.15915494309189535;
                                float sn, cs;
                                sincospif(2.0f * (float)(t - rint(t)), &sn, &cs);
                                const float p = to_f32(w.e[e]), q = to_f32(o.e[e]);
                                w.e[e] = from_f32<T>(low ? p * cs - q * sn : p * cs + q * sn);
                            }
                        }
                    }
                    *reinterpret_cast<Chunk<T>*>(k + row * a.k_dim + d0) = w;
                } else {
                    *reinterpret_cast<Chunk<T>*>(v + row * a.v_dim + (cc - k_chunks) * N) = w;
                }
            }
            for (int j = threadIdx.x; j < rows; j += blockDim.x)
                if (reinterpret_cast<const int*>(tail)[2 * j + 1] >= 0) scores[out_row0 + j] = tail[2 * j];
        }
        __syncthreads();                                          // the stage is fetched into again next
    }
}

extern "C" int cml_evict_positions(void* k, void* v, float* scores, int dtype, const int* table, int width, const int* out_table,
                                   int out_width, const int* lengths, const int* keeps, int* kept, int cap, int entries,
                                   int n_pages, int n_seqs, int heads, int k_dim, int v_dim, int first, int recent,
                                   const float* inv_freq, int rotary_dim, int interleaved, void* stream) {
    if (dtype != CML_DTYPE_F32 && dtype != CML_DTYPE_BF16) return CML_ERR_BAD_DTYPE;
    if (n_seqs <= 0 || entries <= 0 || cap <= 0) return 0;
    const int n = dtype == CML_DTYPE_F32 ? 4 : 8;
    if (heads <= 0 || n_pages <= 0 || width <= 0 || out_width <= 0 || width > (1 << 24) || out_width > (1 << 24)) return CML_ERR_BAD_SIZE;
    if (k_dim <= 0 || k_dim % n || v_dim % n || k_dim + v_dim > 1024 || first < 0 || recent < 0) return CML_ERR_BAD_SIZE;
    if (inv_freq != nullptr && (rotary_dim <= 0 || rotary_dim > k_dim || rotary_dim % (2 * n))) return CML_ERR_BAD_SIZE;
    if (((uintptr_t)k | (uintptr_t)v) & 15) return CML_ERR_BAD_ALIGN;
    const long long units = (long long)entries * n_seqs * heads;
    if (units * EV_MAX_TEAM > 0x7fffffffLL) return CML_ERR_BAD_SIZE;
    EvictArgs a = {};
    a.k = k; a.v = v; a.scores = scores; a.table = table; a.width = width; a.out_table = out_table; a.out_width = out_width;
    a.lengths = lengths; a.keeps = keeps; a.kept = kept; a.cap = cap; a.entries = entries; a.n_pages = n_pages;
    a.n_seqs = n_seqs; a.heads = heads; a.k_dim = k_dim; a.v_dim = v != nullptr ? v_dim : 0; a.first = first; a.recent = recent;
    a.inv_freq = inv_freq; a.rotary_dim = rotary_dim; a.interleaved = interleaved;
    cudaStream_t s = (cudaStream_t)stream;
    cudaError_t e = launch_pdl(evict_select_kernel, dim3((unsigned)units), dim3(EV_SELECT_THREADS), 0, s, a);
    if (e != cudaSuccess) return (int)e;
    // blocks that share a unit: enough for every multiprocessor, none without an output page
    const int out_pages = min(out_width, (cap + CML_PAGE - 1) / CML_PAGE);
    int team = 1;
    while (team < EV_MAX_TEAM && units * team < cml_sm_count() && team < out_pages) team *= 2;
    const size_t row = (size_t)(a.k_dim + a.v_dim) / n * 16 + 8;
    a.tile = CML_PAGE;
    while (row * a.tile * EV_STAGES > 200 * 1024) a.tile /= 2;     // rows of at most 4 KB: 8 of them at least
    const size_t smem = row * a.tile * EV_STAGES;
    e = dtype == CML_DTYPE_F32 ? cml_allow_smem<evict_move_kernel<float>>(smem) : cml_allow_smem<evict_move_kernel<bf16>>(smem);
    if (e != cudaSuccess) return (int)e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(units * team));
    cfg.blockDim = dim3(EV_MOVE_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)team;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cml_pdl_enabled() ? 2 : 1;
    e = dtype == CML_DTYPE_F32 ? cudaLaunchKernelEx(&cfg, evict_move_kernel<float>, a) : cudaLaunchKernelEx(&cfg, evict_move_kernel<bf16>, a);
    if (e != cudaSuccess) return (int)e;
    return cml_launch_status();
}
