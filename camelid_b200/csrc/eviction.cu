// Eviction from the paged cache by accumulated attention weight.
//
// For every unit (cache entry, sequence, kv head) of length L the first `first` places, the last `recent` places and
// those of the middle with the largest scores stay, M = min(keep, L) in all; among equal scores the lower place stays,
// and a score that is not a number counts as the lowest. The places that stay move up, in order, to the places
// 0 .. M - 1 of the out table's pages with their values and scores. With rotary frequencies the keys are turned by the
// angle of the distance they move, so that a key's place is again its position: (a, b) at place p, moved to j, becomes
// (a cos t - b sin t, b cos t + a sin t) with t = (j - p) f. The frequency, formed in double once, is a
// fraction of a turn in 64 bits; its product with the whole places moved wraps to one turn by itself, and only that is rounded (positions
// reach 2^20, where a float product would be off by 0.06 of a radian). The turn itself is float, and a bfloat16 key is rounded once per move.
//
// Two launches. (1) A block per unit finds the score at the border by its digits and lists the places that stay in order.
// (2) The rows move through registers. The out table may be the table itself: place kept[j] >= j, so the rows of the j-th
// output place come from there or from later places, and an output row may be written once the rows of every earlier
// output row (and its own) are read. A cluster of blocks shares a unit and goes through its rows in rounds: every block has
// its round's rows in registers when it arrives at the cluster's barrier, and writes behind it.
//
// Four entries of four sequences of 24,001 to 32,768 places, 8 kv heads of 128, cut to 16,384 with their keys turned (2.2 GB of rows and
// scores): 408 us, 26 of them the choice (bound by the shared-memory atomics of the digits) and 382 the moving, 5.6 TB/s of the 6.6 that
// a copy reaches: reads and writes of one memory at a time, and a barrier between a round's. One sequence of 641 places in 16 entries cut to
// 512 takes 19.4 us, about half each: the steps of two short kernels (loads of table, scores and rows, five barriers), not their bytes (5 us).
#include "common.cuh"
#include <cooperative_groups.h>
#include <math_constants.h>
namespace cg = cooperative_groups;

#define EV_MOVE_THREADS 512
#define EV_ROWS 2               // rows a thread holds at a time (blocks of 1,024 with one: 430 us for 408, 256 with two: 509)
#define EV_MAX_TEAM 8

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

// (1) The keys of the middle are read once into shared memory where they fit (`cached` of them; beyond it they are read
// again). Three passes over digits of 11, 11 and 10 bits find the border, then every warp takes a stretch of its own:
// it counts what stays, the counts are scanned once, and it lists its places without further barriers.
template <int THREADS>
__global__ void __launch_bounds__(THREADS) evict_select_kernel(EvictArgs a, int cached) {
    constexpr int WARPS = THREADS / 32, BINS = 2048;
    extern __shared__ __align__(16) unsigned char raw[];
    unsigned int* hist = reinterpret_cast<unsigned int*>(raw);
    unsigned int* keys = hist + BINS;
    __shared__ unsigned int s_prefix, s_need;
    __shared__ int s_above[WARPS], s_ties[WARPS];
    __shared__ unsigned int s_sum[32];
    pdl_wait();
    const Unit x = unit_of(a, blockIdx.x);
    int* kept = a.kept + (size_t)blockIdx.x * a.cap;
    if (x.keep == x.length) {                                     // everything stays
        for (int j = threadIdx.x; j < x.keep; j += THREADS) kept[j] = j;
        return;
    }
    const int first = min(a.first, x.keep), recent = min(a.recent, x.keep - first);
    const int lo = first, hi = x.length - recent;                 // the middle, which competes
    const int want = x.keep - first - recent;
    const int* pages = a.table + (size_t)x.seq * a.width;
    const float* scores = a.scores + (size_t)x.entry * a.n_pages * a.heads * CML_PAGE;
    auto key_at = [&](int place) {
        if (place < cached) return keys[place];
        const int page = pages[place / CML_PAGE];
        if (page < 0 || page >= a.n_pages) return 0u;
        return score_key(scores[((size_t)page * a.heads + x.head) * CML_PAGE + place % CML_PAGE]);
    };
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int j = threadIdx.x; j < first; j += THREADS) kept[j] = j;
    for (int j = threadIdx.x; j < recent; j += THREADS) kept[x.keep - recent + j] = x.length - recent + j;
    if (want == 0) return;
    for (int b = threadIdx.x; b < BINS; b += THREADS) hist[b] = 0u;
    __syncthreads();
    unsigned int prefix = 0u, need = (unsigned int)want;
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bins = pass == 2 ? 1024 : BINS;
        if (pass == 0) {
            // a warp reads whole pages, two places a lane and four pages in flight
            const int n_pages = (hi + CML_PAGE - 1) / CML_PAGE;
            for (int p0 = lo / CML_PAGE + warp; p0 < n_pages; p0 += 4 * WARPS) {
                float2 v[4];
                bool there[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int page = pages[min(p0 + u * WARPS, n_pages - 1)];
                    there[u] = page >= 0 && page < a.n_pages;
                    v[u] = *reinterpret_cast<const float2*>(scores + ((size_t)(there[u] ? page : 0) * a.heads + x.head) * CML_PAGE + 2 * lane);
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int place = (p0 + u * WARPS) * CML_PAGE + 2 * lane;
                    if (p0 + u * WARPS >= n_pages) break;
                    const unsigned int k0 = there[u] ? score_key(v[u].x) : 0u, k1 = there[u] ? score_key(v[u].y) : 0u;
                    if (place < cached) *reinterpret_cast<uint2*>(keys + place) = make_uint2(k0, k1);
                    if (place >= lo && place < hi) atomicAdd(&hist[k0 >> 21], 1u);
                    if (place + 1 >= lo && place + 1 < hi) atomicAdd(&hist[k1 >> 21], 1u);
                }
            }
        } else {
            const unsigned int mask = ~0u << (pass == 1 ? 21 : 10);
#pragma unroll 4
            for (int p = lo + threadIdx.x; p < hi; p += THREADS) {
                const unsigned int k = key_at(p);
                if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1u);
            }
        }
        __syncthreads();
        // the bin in which the need-th largest lies: warps sum equal shares of the bins from the top
        const int share = bins / 32;                              // bins of a warp's (or, below, lane's) share
        for (int w = warp; w < 32; w += WARPS) {
            unsigned int t = 0u;
            for (int b = lane; b < share; b += 32) t += hist[bins - 1 - (w * share + b)];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
            if (lane == 0) s_sum[w] = t;
        }
        __syncthreads();
        if (warp == 0) {
            unsigned int incl = s_sum[lane];
            const unsigned int mine = incl;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned int t = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += t;
            }
            const int w = __ffs(__ballot_sync(0xffffffffu, incl >= need)) - 1;        // there is one: need <= candidates
            unsigned int before = __shfl_sync(0xffffffffu, incl - mine, w);
            const int per = share / 32;                           // one or two bins a lane
            unsigned int c[2] = {0u, 0u};
            for (int u = 0; u < per; ++u) c[u] = hist[bins - 1 - (w * share + lane * per + u)];
            const unsigned int sum = c[0] + c[1];
            unsigned int run = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned int t = __shfl_up_sync(0xffffffffu, run, o);
                if (lane >= o) run += t;
            }
            const int l = __ffs(__ballot_sync(0xffffffffu, before + run >= need)) - 1;
            if (lane == l) {
                before += run - sum;
                const int u = before + c[0] >= need ? 0 : 1;
                if (u == 1) before += c[0];
                s_prefix = prefix | ((unsigned int)(bins - 1 - (w * share + lane * per + u)) << shift);
                s_need = need - before;                           // how many of the border's digit are still wanted
            }
        }
        __syncthreads();
        prefix = s_prefix;
        need = s_need;
        for (int b = threadIdx.x; b < BINS; b += THREADS) hist[b] = 0u;
        __syncthreads();
    }
    // a warp's stretch of the middle
    const int per = (((hi - lo + WARPS - 1) / WARPS) + 31) & ~31;
    const int begin = min(hi, lo + warp * per), end = min(hi, begin + per);
    int above = 0, ties = 0;
#pragma unroll 4
    for (int p = begin + lane; p < end; p += 32) {
        const unsigned int k = key_at(p);
        above += k > prefix;
        ties += k == prefix;
    }
    above = __reduce_add_sync(0xffffffffu, above);
    ties = __reduce_add_sync(0xffffffffu, ties);
    if (lane == 0) s_above[warp] = above, s_ties[warp] = ties;
    __syncthreads();
    int at = first, ties_before = 0;                              // of the border's equals the `need` lowest places stay
    for (int w = 0; w < warp; ++w) {
        at += s_above[w] + max(0, min(s_ties[w], (int)need - ties_before));
        ties_before += s_ties[w];
    }
    const int stop = x.keep - recent;
    const unsigned int before = (1u << lane) - 1u;
#pragma unroll 2
    for (int p0 = begin; p0 < end; p0 += 32) {
        const int p = p0 + lane;
        const unsigned int k = p < end ? key_at(p) : 0u;
        const bool tie = p < end && k == prefix;
        bool stays = p < end && k > prefix;
        const unsigned int tie_mask = __ballot_sync(0xffffffffu, tie);
        if (tie_mask) {
            stays = stays || (tie && ties_before + __popc(tie_mask & before) < (int)need);
            ties_before += __popc(tie_mask);
        }
        const unsigned int mask = __ballot_sync(0xffffffffu, stays);
        const int j = at + __popc(mask & before);
        if (stays && j < stop) kept[j] = p;
        at += __popc(mask);
    }
}

template <typename T> struct Chunk { static constexpr int N = 16 / sizeof(T); };       // elements of 16 bytes of a row

// An angle of one place, in turns, as 64 bits behind the point: its product with a whole number of places wraps by itself,
// and the upper 32 bits of that are the angle to 2^-32 of a turn.
__device__ __forceinline__ uint2 turns_of(float freq) {
    const double t = (double)freq * 0.15915494309189535;
    const unsigned long long f = (unsigned long long)((t - floor(t)) * 18446744073709551616.0);
    return make_uint2((unsigned int)f, (unsigned int)(f >> 32));
}
__device__ __forceinline__ float phase_of(unsigned int places, uint2 turns) {
    return (float)(int)(__umulhi(places, turns.x) + places * turns.y);        // 2^-32 turns, from -2^31 to 2^31
}
template <typename T> __device__ __forceinline__ void sine_cosine(unsigned int places, uint2 turns, float* sn, float* cs);
template <> __device__ __forceinline__ void sine_cosine<float>(unsigned int places, uint2 turns, float* sn, float* cs) {
    sincospif(phase_of(places, turns) * 4.656612873077393e-10f, sn, cs);      // 2^-31: half turns
}
// bfloat16 keys take the fast functions: off by 2^-20.9, a 7,600th of the keys' own rounding (2^-8)
template <> __device__ __forceinline__ void sine_cosine<bf16>(unsigned int places, uint2 turns, float* sn, float* cs) {
    const float x = phase_of(places, turns) * 1.4629180792671596e-09f;        // 2 pi 2^-32
    asm("sin.approx.ftz.f32 %0, %1;" : "=f"(*sn) : "f"(x));
    asm("cos.approx.ftz.f32 %0, %1;" : "=f"(*cs) : "f"(x));
}
// (l, h) turned back by the angle whose sine and cosine are given (a key moves to a lower place)
__device__ __forceinline__ void turn_back(float& l, float& h, float sn, float cs) {
    const float low = l * cs + h * sn;
    h = h * cs - l * sn;
    l = low;
}
template <typename T> __device__ __forceinline__ void unpack(const uint4& c, float (&e)[Chunk<T>::N]);
template <> __device__ __forceinline__ void unpack<float>(const uint4& c, float (&e)[4]) {
    e[0] = __uint_as_float(c.x), e[1] = __uint_as_float(c.y), e[2] = __uint_as_float(c.z), e[3] = __uint_as_float(c.w);
}
template <> __device__ __forceinline__ void unpack<bf16>(const uint4& c, float (&e)[8]) {
    const unsigned int w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) e[2 * i] = __uint_as_float(w[i] << 16), e[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}
template <typename T> __device__ __forceinline__ uint4 pack(const float (&e)[Chunk<T>::N]);
template <> __device__ __forceinline__ uint4 pack<float>(const float (&e)[4]) {
    return make_uint4(__float_as_uint(e[0]), __float_as_uint(e[1]), __float_as_uint(e[2]), __float_as_uint(e[3]));
}
template <> __device__ __forceinline__ uint4 pack<bf16>(const float (&e)[8]) {
    unsigned int w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(e[2 * i], e[2 * i + 1]);
        w[i] = *reinterpret_cast<const unsigned int*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// (2) A thread owns a column of a row's keys and one of its values, two 16-byte chunks each: of the rotary part the two whose
// elements are turned together (with neighbours as pairs any two), else one of each half of the rest. So all threads turn
// keys and all copy values. A round's rows wait in registers for the barrier; the next round's are asked for right behind
// it, and the places and pages of the two rounds after that are on their way, so that no load waits for another.
template <typename T>
__global__ void __launch_bounds__(EV_MOVE_THREADS) evict_move_kernel(EvictArgs a) {
    constexpr int N = Chunk<T>::N, UNROLL = EV_ROWS;
    extern __shared__ __align__(16) unsigned char raw[];
    uint2* turns = reinterpret_cast<uint2*>(raw);                 // [element of a chunk][columns], or by pair where pairs are neighbours
    pdl_wait();
    const int team = (int)cg::this_cluster().num_blocks(), rank = (int)cg::this_cluster().block_rank();
    const int u = blockIdx.x / team;
    const Unit x = unit_of(a, u);
    const int k_cols = a.k_dim / N / 2, v_cols = a.v ? a.v_dim / N / 2 : 0, cols = max(k_cols, v_cols);
    const int rot_cols = a.inv_freq != nullptr ? a.rotary_dim / N / 2 : 0;
    for (int i = threadIdx.x; i < rot_cols * N; i += EV_MOVE_THREADS)
        turns[a.interleaved ? i : i % N * rot_cols + i / N] = turns_of(a.inv_freq[i]);
    __syncthreads();
    const int* kept = a.kept + (size_t)u * a.cap;
    const int* pages = a.table + (size_t)x.seq * a.width;
    const int* out_pages = a.out_table + (size_t)x.seq * a.out_width;
    const int head_rows = a.heads * CML_PAGE;
    const size_t entry_rows = (size_t)x.entry * a.n_pages * head_rows;
    float* const scores = a.scores + entry_rows;
    const int per_pass = EV_MOVE_THREADS / cols;                  // rows that the block moves in a pass
    const int my_row = threadIdx.x / cols, col = threadIdx.x - my_row * cols;
    const bool has_k = col < k_cols, has_v = col < v_cols, rotates = col < rot_cols;
    const int d0 = rotates ? col * N : a.rotary_dim * (rot_cols > 0) + (col - rot_cols) * N;
    const int d1 = d0 + (rotates ? a.rotary_dim / 2 : (k_cols - rot_cols) * N);
    T* const k = (T*)a.k + entry_rows * a.k_dim + d0;
    T* const v = (T*)a.v + entry_rows * a.v_dim + col * N;
    const int k_step = d1 - d0, v_step = v_cols * N;
    const int tile = per_pass * UNROLL;
    const int rounds = (x.keep + tile * team - 1) / (tile * team);            // the same for every block of the cluster
    auto place_of = [&](int round, int i) {                       // the source place of this thread's i-th row, -1: none
        const int j = (round * team + rank) * tile + i * per_pass + my_row;
        return my_row < per_pass && j < x.keep ? kept[j] : -1;
    };
    auto row_of = [&](int place) {                                // its row in the entry's pages, -1: none
        if (place < 0) return -1;
        const int page = pages[place / CML_PAGE];
        return page < 0 || page >= a.n_pages ? -1 : page * head_rows + x.head * CML_PAGE + place % CML_PAGE;
    };
    struct Row {
        uint4 k0, k1, v0, v1;
        float score;
    };
    auto ask = [&](Row& r, int row) {
        if (row < 0) return;
        if (has_k) {
            const T* src = k + (size_t)row * a.k_dim;
            r.k0 = *reinterpret_cast<const uint4*>(src);
            r.k1 = *reinterpret_cast<const uint4*>(src + k_step);
        }
        if (has_v) {
            const T* src = v + (size_t)row * a.v_dim;
            r.v0 = *reinterpret_cast<const uint4*>(src);
            r.v1 = *reinterpret_cast<const uint4*>(src + v_step);
        }
        if (col == 0) r.score = scores[row];
    };
    int place[UNROLL], place1[UNROLL], place2[UNROLL], row[UNROLL], row1[UNROLL];         // of this round, the next, the one after
    Row now[UNROLL], next[UNROLL];
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) place[i] = place_of(0, i), place1[i] = place_of(1, i), place2[i] = place_of(2, i);
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) row[i] = row_of(place[i]), row1[i] = row_of(place1[i]);
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) ask(now[i], row[i]);
    for (int round = 0; round < rounds; ++round) {
        // Every row of this round has been read when the barrier lets go: arriving there orders a thread's loads before
        // the others' stores behind it.
        if (team > 1) cg::this_cluster().sync();
        else __syncthreads();
        int row2[UNROLL], place3[UNROLL];
#pragma unroll
        for (int i = 0; i < UNROLL; ++i) ask(next[i], row1[i]);
#pragma unroll
        for (int i = 0; i < UNROLL; ++i) row2[i] = row_of(place2[i]), place3[i] = place_of(round + 3, i);
#pragma unroll
        for (int i = 0; i < UNROLL; ++i) {
            if (row[i] < 0) continue;
            const int j = (round * team + rank) * tile + i * per_pass + my_row;
            const int to = out_pages[j / CML_PAGE];
            if (to < 0 || to >= a.n_pages) continue;
            const int out_row = to * head_rows + x.head * CML_PAGE + j % CML_PAGE;
            if (has_v) {
                T* dst = v + (size_t)out_row * a.v_dim;
                *reinterpret_cast<uint4*>(dst) = now[i].v0;
                *reinterpret_cast<uint4*>(dst + v_step) = now[i].v1;
            }
            const unsigned int back = (unsigned int)(place[i] - j);           // places that the row moves down
            if (rotates && back != 0u) {
                float p[N], q[N], sn, cs;
                unpack<T>(now[i].k0, p);
                unpack<T>(now[i].k1, q);
                if (a.interleaved) {
#pragma unroll
                    for (int e = 0; e < N; e += 2) {
                        sine_cosine<T>(back, turns[(d0 + e) / 2], &sn, &cs);
                        turn_back(p[e], p[e + 1], sn, cs);
                        sine_cosine<T>(back, turns[(d1 + e) / 2], &sn, &cs);
                        turn_back(q[e], q[e + 1], sn, cs);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        sine_cosine<T>(back, turns[e * rot_cols + col], &sn, &cs);
                        turn_back(p[e], q[e], sn, cs);
                    }
                }
                now[i].k0 = pack<T>(p);
                now[i].k1 = pack<T>(q);
            }
            if (has_k) {
                T* dst = k + (size_t)out_row * a.k_dim;
                *reinterpret_cast<uint4*>(dst) = now[i].k0;
                *reinterpret_cast<uint4*>(dst + k_step) = now[i].k1;
            }
            if (col == 0) scores[out_row] = now[i].score;
        }
#pragma unroll
        for (int i = 0; i < UNROLL; ++i) {
            now[i] = next[i];
            place[i] = place1[i], row[i] = row1[i];
            place1[i] = place2[i], row1[i] = row2[i];
            place2[i] = place3[i];
        }
    }
}

template <typename T>
static cudaError_t launch_move(const EvictArgs& a, long long units, int team, size_t smem, cudaStream_t s) {
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
    return cudaLaunchKernelEx(&cfg, evict_move_kernel<T>, a);
}

extern "C" int cml_evict_positions(void* k, void* v, float* scores, int dtype, const int* table, int width, const int* out_table,
                                   int out_width, const int* lengths, const int* keeps, int* kept, int cap, int entries,
                                   int n_pages, int n_seqs, int heads, int k_dim, int v_dim, int first, int recent,
                                   const float* inv_freq, int rotary_dim, int interleaved, void* stream) {
    if (dtype != CML_DTYPE_F32 && dtype != CML_DTYPE_BF16) return CML_ERR_BAD_DTYPE;
    if (n_seqs <= 0 || entries <= 0 || cap <= 0) return 0;
    const int n = dtype == CML_DTYPE_F32 ? 4 : 8;
    if (heads <= 0 || n_pages <= 0 || width <= 0 || out_width <= 0 || width > (1 << 24) || out_width > (1 << 24)) return CML_ERR_BAD_SIZE;
    if (k_dim <= 0 || k_dim % 16 || v_dim % 16 || k_dim + v_dim > 1024 || first < 0 || recent < 0) return CML_ERR_BAD_SIZE;
    if (inv_freq != nullptr && (rotary_dim <= 0 || rotary_dim > k_dim || rotary_dim % 16)) return CML_ERR_BAD_SIZE;
    if ((((uintptr_t)k | (uintptr_t)v) & 15) || (((uintptr_t)scores) & 7)) return CML_ERR_BAD_ALIGN;      // scores are read in pairs
    if ((long long)n_pages * heads * CML_PAGE > 0x7fffffffLL) return CML_ERR_BAD_SIZE;       // an entry's rows are counted in 32 bits
    const long long units = (long long)entries * n_seqs * heads;
    if (units * EV_MAX_TEAM > 0x7fffffffLL) return CML_ERR_BAD_SIZE;
    EvictArgs a = {};
    a.k = k; a.v = v; a.scores = scores; a.table = table; a.width = width; a.out_table = out_table; a.out_width = out_width;
    a.lengths = lengths; a.keeps = keeps; a.kept = kept; a.cap = cap; a.entries = entries; a.n_pages = n_pages;
    a.n_seqs = n_seqs; a.heads = heads; a.k_dim = k_dim; a.v_dim = v != nullptr ? v_dim : 0; a.first = first; a.recent = recent;
    a.inv_freq = inv_freq; a.rotary_dim = rotary_dim; a.interleaved = interleaved;
    cudaStream_t s = (cudaStream_t)stream;
    // A unit's scores fit the shared memory up to 48 k places. Short sequences take small blocks, of which many run at once.
    const long long longest = (long long)width * CML_PAGE;
    const int cached = (int)(longest < 49152 ? longest : 49152);
    const size_t select_smem = (2048 + (size_t)cached) * 4;
    cudaError_t e;
    if (longest <= 4096) {
        e = cml_allow_smem<evict_select_kernel<256>>(select_smem);
        if (e == cudaSuccess) e = launch_pdl(evict_select_kernel<256>, dim3((unsigned)units), dim3(256), select_smem, s, a, cached);
    } else {
        e = cml_allow_smem<evict_select_kernel<1024>>(select_smem);
        if (e == cudaSuccess) e = launch_pdl(evict_select_kernel<1024>, dim3((unsigned)units), dim3(1024), select_smem, s, a, cached);
    }
    if (e != cudaSuccess) return (int)e;
    // blocks that share a unit: one for every multiprocessor in all, none without rows to move
    const long long most = out_width * (long long)CML_PAGE < cap ? out_width * (long long)CML_PAGE : cap;
    const int cols = (k_dim > a.v_dim ? k_dim : a.v_dim) / n / 2, tile = EV_MOVE_THREADS / cols * EV_ROWS;
    int team = 1;
    while (team < EV_MAX_TEAM && units * team * 2 <= cml_sm_count() && (long long)team * tile < most) team *= 2;
    const size_t smem = (size_t)rotary_dim / 2 * 8;
    e = dtype == CML_DTYPE_F32 ? launch_move<float>(a, units, team, smem, s) : launch_move<bf16>(a, units, team, smem, s);
    if (e != cudaSuccess) return (int)e;
    return cml_launch_status();
}
