// Attention of a few new tokens per sequence over the paged cache that also keeps what it weighed: the score of every
// cached position gains the attention weight that the step's rows gave it, summed over the query heads of its kv head.
//
//   s = scale q . k      w = exp(s - max s) / sum exp(s - max s)      out = sum w v
//   scores'[place] = (place was cached before ? scores[place] : 0) + sum over rows and heads of w
//
// A step's rows are packed: sequence i owns rows row0[i] .. row0[i] + new[i], its row j stands at place start[i] + j and
// sees the places up to its own. Without an output only the scores are made (what a prompt's last rows look at).
//
// The weights of a key are known only when all keys are seen, so the work is cut in three: (1) blocks take stretches of
// a sequence's keys and keep the running maximum, sum and output of their rows; (2) the stretches are joined, in order;
// (3) every key's weights are summed, in a fixed order of the rows. Steps of few rows (a single token, a drafted step) do all
// three in one launch: the blocks of a cluster share a sequence and kv head, exchange their rows' maxima and sums over distributed
// shared memory, and weigh the products q . k again that they kept (4 bytes a row and key, which stay in L2). More rows make
// the products again in a kernel of their own; without output (a prompt's last rows) on tcgen05 (attention_weights_tc.cuh).
// Products, softmax and sums are float; on the tensor cores a probability is rounded to bfloat16 where it meets a value, as
// the values are: the sum over the keys has half a step of each product (2^-8 of it), beside which the output's own rounding is
// as large (16 sequences of 24,001 to 32,768 keys: 0.0021 from 64 bits in norm, 0.0017 with probabilities in float).
//
// Bound by memory where sequences are long: 16 of 24,001 to 32,768 keys with 8 kv heads of 128 (1.9 GB) take 340 us, 5.6 TB/s
// of 6.6 that a copy reaches; 8 of 300 to 8,191 34.5 us (4.1 TB/s: unequal lengths, and 4 us of joining and weighing at the end);
// short ones by the launch (12 us a call on the host, 6 on the device for 517 keys). In float: 4 sequences of 700 to 2,047 keys, heads of
// 96, 18.2 us for 17 MB (a page is worked on in phases between barriers, and only one is on its way meanwhile).
#include "common.cuh"
#include <cooperative_groups.h>
#include <math_constants.h>
namespace cg = cooperative_groups;

#define AW_THREADS 256
#define AW_ROWS 8               // rows (token, head) a block works on together
#define AW_TEAM 8               // blocks of a cluster at most (sixteen were 7% to 40% slower here)

struct WeightArgs {
    const void* q;
    long long q_stride;
    void* out;                   // null: scores only
    long long out_stride;
    const void* k;
    const void* v;
    const float* scores;
    float* scores_out;
    const int* table;
    int width, n_pages;
    const int* row0;
    const int* start;
    const int* fresh;            // new tokens of each sequence
    const int* cached;           // places of each sequence whose scores count from before (null: those below `start`)
    int n_seqs, n_rows, heads, kv_heads, k_dim, v_dim;
    int max_new, max_len;
    float scale;                 // of the scores, times log2(e): the softmax is taken in powers of two
    int stages;                  // pages of keys and values a block of (1) keeps in shared memory: 2, or 1 where two do not fit
    int split_keys, n_splits;    // keys of a stretch (a multiple of the page), stretches of the longest sequence
    float* stats;                // [seqs * kv heads][splits][rows][2]: maximum and sum of a stretch
    float* joined;               // [seqs * kv heads][rows][2]: maximum and 1 / sum of all
    float* acc;                  // [seqs * kv heads][splits][rows][v_dim]
    float* kept;                 // q . k of steps of few rows: [blocks][rows][64], see kept_of
    int kept_blocks;             // pages of the longest sequence, or 0: the blocks are the cache's own pages
};

// Where the products of a page of keys lie. A sequence's pages in its order need a rectangle, as long as the longest sequence for all;
// where the cache has fewer pages than that, its own pages name the blocks (no page belongs to two sequences), so that the products
// never take more than 4 bytes a row and cached key. A page that is none has no block then: nothing is kept of it or asked.
struct Kept {
    float* base;                 // of place 0 of block 0 of a sequence and kv head
    int stride;                  // floats between blocks: the pages of a kv head, or of all
    bool by_page;
    __device__ __forceinline__ float* at(int p, int page) const { return base + (size_t)(by_page ? page : p) * stride; }
};
__device__ __forceinline__ Kept kept_of(const WeightArgs& a, int pair, int kvh, int rows) {
    Kept k;
    k.by_page = a.kept_blocks == 0;
    k.stride = rows * CML_PAGE * (k.by_page ? a.kv_heads : 1);
    k.base = a.kept + (k.by_page ? (size_t)kvh : (size_t)pair * a.kept_blocks) * (rows * CML_PAGE);
    return k;
}

struct Seq {
    int start, fresh, length, row0, rows;      // rows: (token, head) pairs that share a kv head
    int old;                                   // places below this keep the score they have and gain
};
__device__ __forceinline__ Seq seq_of(const WeightArgs& a, int i) {
    Seq s;
    s.start = max(0, min(a.start[i], 1 << 30));
    s.row0 = a.row0[i];
    s.old = a.cached != nullptr ? min(a.cached[i], s.start) : s.start;
    s.fresh = max(0, min(a.fresh[i], a.max_new));
    if (s.row0 < 0 || s.row0 > a.n_rows - s.fresh) s.fresh = 0;
    s.length = min(min(s.start + s.fresh, a.max_len), a.width * CML_PAGE);
    if (s.fresh == 0) s.length = 0;
    s.rows = s.fresh * (a.heads / a.kv_heads);
    return s;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A page's rows into shared memory, rows of `stride` bytes; rows at and beyond `valid` are zeroed.
template <typename T>
__device__ __forceinline__ void fetch_page(unsigned char* dst, int stride, const T* src, int dim, int valid) {
    const int chunks = dim * (int)sizeof(T) / 16;
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(dst);
    int r = (int)threadIdx.x / chunks, cc = (int)threadIdx.x - r * chunks;    // walked without further divisions
    const int r_step = AW_THREADS / chunks, c_step = AW_THREADS - r_step * chunks;
    while (r < CML_PAGE) {
        if (r < valid) cp_async16(at + (uint32_t)(r * stride + cc * 16), (const unsigned char*)src + ((size_t)r * dim) * sizeof(T) + cc * 16);
        else *reinterpret_cast<uint4*>(dst + r * stride + cc * 16) = make_uint4(0, 0, 0, 0);
        r += r_step, cc += c_step;
        if (cc >= chunks) cc -= chunks, ++r;
    }
}

template <typename T> __device__ __forceinline__ float dot_chunk(const unsigned char* k, const float* q);
template <> __device__ __forceinline__ float dot_chunk<float>(const unsigned char* k, const float* q) {
    const float4 a = *reinterpret_cast<const float4*>(k), b = *reinterpret_cast<const float4*>(q);
    return a.x * b.x + a.y * b.y + a.z * b.z + a.w * b.w;
}
template <> __device__ __forceinline__ float dot_chunk<bf16>(const unsigned char* k, const float* q) {
    const uint4 r = *reinterpret_cast<const uint4*>(k);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        s += __uint_as_float(w[i] << 16) * q[2 * i] + __uint_as_float(w[i] & 0xffff0000u) * q[2 * i + 1];
    return s;
}

// A channel of R rows of q (zero where there is no row); all are asked for at once.
template <typename T, int R>
__device__ __forceinline__ void ask_q(const WeightArgs& a, const Seq& s, int kvh, int m0, int d, float (&x)[R]) {
    const int group = a.heads / a.kv_heads;
#pragma unroll
    for (int m = 0; m < R; ++m) {
        const bool in = m0 + m < s.rows;
        const int j = in ? (m0 + m) / group : 0, h = in ? m0 + m - j * group : 0;
        x[m] = to_f32(((const T*)a.q)[(long long)(s.row0 + j) * a.q_stride + (long long)(kvh * group + h) * a.k_dim + d]);
        if (!in) x[m] = 0.f;
    }
}

// The products of this thread's key (threadIdx.x & 63) with R rows over its quarter (threadIdx.x >> 6) of the 16-byte pieces.
template <typename T, int R>
__device__ __forceinline__ void quarter_products(const WeightArgs& a, const unsigned char* k_row, const float* q_s, float* part_s) {
    constexpr int N = 16 / sizeof(T);
    const int key = threadIdx.x & 63, quarter = threadIdx.x >> 6, chunks = a.k_dim / N;
    float acc[R];
#pragma unroll
    for (int m = 0; m < R; ++m) acc[m] = 0.f;
#pragma unroll 2
    for (int c = quarter; c < chunks; c += 4)
#pragma unroll
        for (int m = 0; m < R; ++m) acc[m] += dot_chunk<T>(k_row + c * 16, q_s + m * a.k_dim + c * N);
#pragma unroll
    for (int m = 0; m < R; ++m) part_s[(quarter * R + m) * CML_PAGE + key] = acc[m];
}
// The four quarters' sum for a row and key.
template <int R>
__device__ __forceinline__ float product_of(const float* part_s, int m, int key) {
    const float* const from = part_s + m * CML_PAGE + key;
    return (from[0] + from[R * CML_PAGE]) + (from[2 * R * CML_PAGE] + from[3 * R * CML_PAGE]);
}

template <typename T> __device__ __forceinline__ void four_of(const T* p, float (&v)[4]);
template <> __device__ __forceinline__ void four_of<float>(const float* p, float (&v)[4]) {
    const float4 x = *reinterpret_cast<const float4*>(p);
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
}
template <> __device__ __forceinline__ void four_of<bf16>(const bf16* p, float (&v)[4]) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    v[0] = __uint_as_float(x.x << 16), v[1] = __uint_as_float(x.x & 0xffff0000u), v[2] = __uint_as_float(x.y << 16), v[3] = __uint_as_float(x.y & 0xffff0000u);
}

// R rows and a stretch of keys, in float on the CUDA cores, a page of keys and values at a time. For the scores a thread has a key, all
// rows and a quarter of the channels, so that a key is read from shared memory once; for the output four channels of the keys that its
// group of v_dim / 4 threads takes in turn with the others, so that no thread is idle; the groups meet once, behind the keys. (With a
// row a thread over all channels, and a channel a thread over half of the keys, 4 sequences of 700 to 2,047 keys took 20.8 us for 18.2
// with heads of 96, two of 4,000 68 for 50 with heads of 256; rings of four pages leave room for one block and took 23.6.)
// ALL (grid: cluster, pairs; for steps of at most R rows): the blocks of a cluster share all keys of a sequence and finish by
// themselves, as on the tensor cores below. Otherwise (grid: stretches, pairs, row tiles) this is step (1).
template <typename T, int R, bool ALL>
__global__ void __launch_bounds__(AW_THREADS) weights_part_kernel(WeightArgs a) {
    extern __shared__ __align__(16) unsigned char raw[];
    __shared__ float2 stat_s[ALL ? AW_TEAM * R : 1];              // ALL: [blocks][rows] maximum and sum, of the whole cluster
    __shared__ float2 join_s[ALL ? R : 1];                        // ALL: [rows] maximum and 1 / sum of all keys
    const int split = blockIdx.x, seq = blockIdx.y / a.kv_heads, kvh = blockIdx.y % a.kv_heads, m0 = blockIdx.z * R;
    pdl_wait();
    const Seq s = seq_of(a, seq);
    if (m0 >= s.rows) return;                                     // the same for a whole cluster
    const int team = ALL ? (int)gridDim.x : 1;
    const int share = ALL ? (s.length + team * CML_PAGE - 1) / (team * CML_PAGE) * CML_PAGE : a.split_keys;
    const int first = split * share, last = min(s.length, first + share);
    if (ALL) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");        // started: waited for before remote stores
    else if (first >= last) return;
    const int k_stride = a.k_dim * (int)sizeof(T) + 16, v_stride = a.out ? a.v_dim * (int)sizeof(T) : 0;
    const int page_bytes = CML_PAGE * (k_stride + v_stride);
    // (the ring's room holds the output of all groups of threads in the end, so it is as large as that at least)
    float* q_s = reinterpret_cast<float*>(raw + max(a.stages * page_bytes, a.out ? R * AW_THREADS * 16 : 0));
    float* p_s = q_s + R * a.k_dim;                               // [page][rows]
    float* part_s = p_s + R * CML_PAGE;                           // [quarters][rows][page] the quarters' products
    float* m_s = part_s + 4 * R * CML_PAGE;
    float* l_s = m_s + R;
    float* c_s = l_s + R;
    float* own = c_s + R;                                         // [rows][v_dim], the block's output
    const int* pages = a.table + (size_t)seq * a.width;
    const int p_first = first / CML_PAGE, p_last = (last + CML_PAGE - 1) / CML_PAGE;
    const int group_rows = a.max_new * (a.heads / a.kv_heads);
    const Kept products = kept_of(a, blockIdx.y, kvh, group_rows);
    auto valid_of = [&](int p) {
        const int page = p < p_last ? pages[p] : -1;
        return page < 0 || page >= a.n_pages ? 0 : min(CML_PAGE, last - p * CML_PAGE);
    };
    auto fetch = [&](int p) {
        if (p < p_last) {
            const int valid = valid_of(p);
            const size_t at = valid ? ((size_t)pages[p] * a.kv_heads + kvh) * CML_PAGE : 0;
            unsigned char* dst = raw + (size_t)((p - p_first) & (a.stages - 1)) * page_bytes;
            fetch_page<T>(dst, k_stride, (const T*)a.k + at * a.k_dim, a.k_dim, valid);
            if (a.out) fetch_page<T>(dst + CML_PAGE * k_stride, v_stride, (const T*)a.v + at * a.v_dim, a.v_dim, valid);
        }
        cp_async_commit();
    };
    fetch(p_first);
    for (int d = threadIdx.x; d < a.k_dim; d += AW_THREADS) {
        float x[R];
        ask_q<T, R>(a, s, kvh, m0, d, x);
#pragma unroll
        for (int m = 0; m < R; ++m) q_s[m * a.k_dim + d] = x[m];
    }
    if (threadIdx.x < R) m_s[threadIdx.x] = -CUDART_INF_F, l_s[threadIdx.x] = 0.f;
    float o[R][4];
#pragma unroll
    for (int m = 0; m < R; ++m) o[m][0] = o[m][1] = o[m][2] = o[m][3] = 0.f;
    const int quads = a.out ? a.v_dim / 4 : AW_THREADS, groups = AW_THREADS / quads;          // groups of threads that share the keys
    const int kk_first = threadIdx.x / quads, d = (threadIdx.x - kk_first * quads) * 4;       // (a thread behind the groups has no keys)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rows = min(R, s.rows - m0), group = a.heads / a.kv_heads;
    for (int p = p_first; p < p_last; ++p) {
        if (a.stages > 1) fetch(p + 1);
        else if (p > p_first) fetch(p);
        if (a.stages > 1) cp_async_wait<1>();
        else cp_async_wait<0>();
        __syncthreads();
        const unsigned char* ks = raw + (size_t)((p - p_first) & (a.stages - 1)) * page_bytes;
        quarter_products<T, R>(a, ks + (threadIdx.x & 63) * k_stride, q_s, part_s);
        __syncthreads();
        const int valid = valid_of(p);
        float* const kept = ALL && valid > 0 ? products.at(p, pages[p]) : nullptr;
        for (int m = warp; m < rows; m += AW_THREADS / 32) {
            const int sees = min(valid - 1, s.start + (m0 + m) / group - p * CML_PAGE);       // the last key of the page that the row sees
            float x[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                x[h] = product_of<R>(part_s, m, lane + 32 * h) * a.scale;
                if (lane + 32 * h > sees) x[h] = -CUDART_INF_F;
                if (ALL && valid > 0) kept[m * CML_PAGE + lane + 32 * h] = x[h];
            }
            const float a0 = x[0], a1 = x[1];
            const float old = m_s[m], now = fmaxf(old, warp_max(fmaxf(a0, a1)));
            const float e0 = a0 == -CUDART_INF_F ? 0.f : exp2f(a0 - now), e1 = a1 == -CUDART_INF_F ? 0.f : exp2f(a1 - now);
            const float corr = old == -CUDART_INF_F ? 0.f : exp2f(old - now);
            const float sum = warp_sum(e0 + e1);
            p_s[lane * R + m] = e0;
            p_s[(lane + 32) * R + m] = e1;
            __syncwarp();
            if (lane == 0) m_s[m] = now, l_s[m] = l_s[m] * corr + sum, c_s[m] = corr;
        }
        __syncthreads();
        if (a.out && kk_first < groups) {
            const T* vs = reinterpret_cast<const T*>(ks + CML_PAGE * k_stride) + d;
            // where rows do not all see the same places, one that a row does not see adds nothing, whatever it holds
            const bool careful = s.fresh > 1 && (p + 1) * CML_PAGE > s.start + 1;
#pragma unroll
            for (int m = 0; m < R; ++m) {
                const float f = m < rows ? c_s[m] : 1.f;
                o[m][0] *= f, o[m][1] *= f, o[m][2] *= f, o[m][3] *= f;
            }
            auto add = [&](int kk, bool zero) {
                float v[4];
                four_of<T>(vs + kk * a.v_dim, v);
#pragma unroll
                for (int m = 0; m < R; m += 4) {
                    const float4 w4 = *reinterpret_cast<const float4*>(p_s + kk * R + m);
                    const float w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                    for (int u = 0; u < 4; ++u)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[m + u][i] = fmaf(w[u], zero && w[u] == 0.f ? 0.f : v[i], o[m + u][i]);
                }
            };
            if (careful)
                for (int kk = kk_first; kk < CML_PAGE; kk += groups) add(kk, true);
            else {
#pragma unroll 4
                for (int kk = kk_first; kk < CML_PAGE; kk += groups) add(kk, false);
            }
        }
        __syncthreads();
    }
    cp_async_wait<0>();
    __syncthreads();
    pdl_launch_dependents();
    if (a.out) {                                                  // the groups' sums meet in the ring's room, in their order
        float* const red = reinterpret_cast<float*>(raw);         // [groups][rows][v_dim]
        if (kk_first < groups) {
#pragma unroll
            for (int m = 0; m < R; ++m) *reinterpret_cast<float4*>(red + (kk_first * R + m) * a.v_dim + d) = make_float4(o[m][0], o[m][1], o[m][2], o[m][3]);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < R * a.v_dim; i += AW_THREADS) {
            float x = 0.f;
#pragma unroll 4
            for (int g = 0; g < groups; ++g) x += red[g * R * a.v_dim + i];
            own[i] = x;
        }
    }
    __syncthreads();
    if (!ALL) {
        const size_t base = ((size_t)blockIdx.y * a.n_splits + split) * group_rows + m0;
        if ((int)threadIdx.x < rows) {
            a.stats[(base + threadIdx.x) * 2] = m_s[threadIdx.x];
            a.stats[(base + threadIdx.x) * 2 + 1] = l_s[threadIdx.x];
        }
        __syncthreads();
        if (a.out)
            for (int i = threadIdx.x; i < rows * a.v_dim; i += AW_THREADS) a.acc[base * a.v_dim + i] = own[i];
        return;
    }
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if ((int)threadIdx.x < rows)
        for (int c = 0; c < team; ++c) cg::this_cluster().map_shared_rank(&stat_s[0], c)[split * R + threadIdx.x] = make_float2(m_s[threadIdx.x], l_s[threadIdx.x]);
    cg::this_cluster().sync();
    if ((int)threadIdx.x < rows) {
        const int m = threadIdx.x;
        float most = -CUDART_INF_F, l = 0.f;
        for (int c = 0; c < team; ++c) most = fmaxf(most, stat_s[c * R + m].x);
        for (int c = 0; c < team; ++c) {
            const float2 t = stat_s[c * R + m];
            const float f = t.x == -CUDART_INF_F ? 0.f : exp2f(t.x - most);
            stat_s[c * R + m].x = f;                              // from here on: what a block's output counts in the joined one
            l += f * t.y;
        }
        join_s[m] = most == -CUDART_INF_F ? make_float2(0.f, 0.f) : make_float2(most, 1.f / l);
    }
    __syncthreads();
    if (a.out) {                                                  // the output's elements in equal shares, the blocks in their order
        for (int i = split * AW_THREADS + threadIdx.x; i < rows * a.v_dim; i += team * AW_THREADS) {
            const int m = i / a.v_dim, d = i - m * a.v_dim;
            float x = 0.f;
#pragma unroll 4
            for (int c = 0; c < team; ++c) x += stat_s[c * R + m].x * cg::this_cluster().map_shared_rank(own, c)[m * a.v_dim + d];
            ((T*)a.out)[(long long)(s.row0 + m / group) * a.out_stride + (long long)(kvh * group + m % group) * a.v_dim + d] = from_f32<T>(x * join_s[m].y);
        }
    }
    // the weights of this block's keys
    for (int place = first + (int)threadIdx.x; place < last; place += AW_THREADS) {
        const int page = pages[place / CML_PAGE];
        if (page < 0 || page >= a.n_pages) continue;
        const size_t at = ((size_t)page * a.kv_heads + kvh) * CML_PAGE + place % CML_PAGE;
        const float* const kept = products.at(place / CML_PAGE, page) + place % CML_PAGE;
        float gained = 0.f;
        const float old = a.scores[at];
#pragma unroll
        for (int m = 0; m < R; ++m)
            if (m < rows) gained += exp2f(kept[m * CML_PAGE] - join_s[m].x) * join_s[m].y;
        a.scores_out[at] = (place < s.old ? old : 0.f) + gained;
    }
    if (a.out) cg::this_cluster().sync();                         // a block's output stays until every block has read it
}

// (2) the stretches of a row joined in their order: grid (rows that share a kv head, sequences * kv heads)
template <typename T>
__global__ void __launch_bounds__(AW_THREADS) weights_join_kernel(WeightArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    const int m = blockIdx.x, seq = blockIdx.y / a.kv_heads, kvh = blockIdx.y % a.kv_heads;
    const Seq s = seq_of(a, seq);
    if (m >= s.rows) return;
    const int group = a.heads / a.kv_heads, group_rows = a.max_new * group;
    const int splits = (s.length + a.split_keys - 1) / a.split_keys;
    const size_t base = (size_t)blockIdx.y * a.n_splits * group_rows + m;
    float top = -CUDART_INF_F, sum = 0.f;
    for (int i = 0; i < splits; ++i) top = fmaxf(top, a.stats[(base + (size_t)i * group_rows) * 2]);
    for (int i = 0; i < splits; ++i) {
        const float t = a.stats[(base + (size_t)i * group_rows) * 2];
        if (t != -CUDART_INF_F) sum += exp2f(t - top) * a.stats[(base + (size_t)i * group_rows) * 2 + 1];
    }
    const float inv = top == -CUDART_INF_F ? 0.f : 1.f / sum;
    if (threadIdx.x == 0) {
        float* j = a.joined + ((size_t)blockIdx.y * group_rows + m) * 2;
        j[0] = top == -CUDART_INF_F ? 0.f : top;
        j[1] = inv;
    }
    if (a.out == nullptr) return;
    T* out = (T*)a.out + (long long)(s.row0 + m / group) * a.out_stride + (long long)(kvh * group + m % group) * a.v_dim;
    for (int d = threadIdx.x; d < a.v_dim; d += AW_THREADS) {
        float x = 0.f;
        for (int i = 0; i < splits; ++i) {
            const float t = a.stats[(base + (size_t)i * group_rows) * 2];
            if (t != -CUDART_INF_F) x += exp2f(t - top) * a.acc[(base + (size_t)i * group_rows) * a.v_dim + d];
        }
        out[d] = from_f32<T>(x * inv);
    }
}

// (3) the weights of a page of keys: grid (pages of the longest sequence, sequences * kv heads)
template <typename T>
__global__ void __launch_bounds__(AW_THREADS) weights_sum_kernel(WeightArgs a) {
    extern __shared__ __align__(16) unsigned char raw[];
    __shared__ float other[3][CML_PAGE];
    pdl_wait();
    pdl_launch_dependents();
    const int p = blockIdx.x, seq = blockIdx.y / a.kv_heads, kvh = blockIdx.y % a.kv_heads;
    const Seq s = seq_of(a, seq);
    const int valid = min(CML_PAGE, s.length - p * CML_PAGE);
    if (valid <= 0) return;
    const int page = a.table[(size_t)seq * a.width + p];
    if (page < 0 || page >= a.n_pages) return;
    const int k_stride = a.k_dim * (int)sizeof(T) + 16;
    float* q_s = reinterpret_cast<float*>(raw + CML_PAGE * k_stride);
    const size_t at = ((size_t)page * a.kv_heads + kvh) * CML_PAGE;
    fetch_page<T>(raw, k_stride, (const T*)a.k + at * a.k_dim, a.k_dim, valid);
    cp_async_commit();
    const int key = threadIdx.x & 63, quarter = threadIdx.x >> 6, place = p * CML_PAGE + key;
    const int group = a.heads / a.kv_heads, group_rows = a.max_new * group;
    float* const part_s = q_s + AW_ROWS * a.k_dim;                // [quarters][rows][page]
    const bool has = (int)threadIdx.x < a.k_dim;                  // (256 channels at most, as many as threads)
    float next[AW_ROWS];
    if (has) ask_q<T, AW_ROWS>(a, s, kvh, 0, threadIdx.x, next);
    cp_async_wait<0>();
    float gained = 0.f;
    for (int m0 = 0; m0 < s.rows; m0 += AW_ROWS) {
        if (has) {
#pragma unroll
            for (int m = 0; m < AW_ROWS; ++m) q_s[m * a.k_dim + threadIdx.x] = next[m];
        }
        __syncthreads();
        if (has && m0 + AW_ROWS < s.rows) ask_q<T, AW_ROWS>(a, s, kvh, m0 + AW_ROWS, threadIdx.x, next);      // beside the products of these
        quarter_products<T, AW_ROWS>(a, raw + key * k_stride, q_s, part_s);
        __syncthreads();
#pragma unroll
        for (int u = 0; u < AW_ROWS / 4; ++u) {                   // a quarter of the rows each
            const int m = quarter * (AW_ROWS / 4) + u, r = m0 + m;
            if (r >= s.rows || place > s.start + r / group) continue;
            const float2 j = *reinterpret_cast<const float2*>(a.joined + ((size_t)blockIdx.y * group_rows + r) * 2);
            gained += exp2f(product_of<AW_ROWS>(part_s, m, key) * a.scale - j.x) * j.y;
        }
    }
    if (quarter > 0) other[quarter - 1][key] = gained;
    __syncthreads();
    if (quarter == 0 && key < valid) {
        a.scores_out[at + key] = (place < s.old ? a.scores[at + key] : 0.f) + (((gained + other[0][key]) + other[1][key]) + other[2][key]);
    }
}

// ------------------------------------------------------------------------------------------------------------------
// bfloat16 with head sizes 64 and 128 on the tensor cores (mma.sync m16n8k16: what bounds these kernels is memory, or the
// exponentials of many rows, not the products). Shared-memory rows are padded by 16 bytes, so ldmatrix meets no bank twice.

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ float fast_exp2(float x) {            // 2^x to 2^-22 of itself; 0 for -inf
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool there) {
    const int n = there ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

#define AM_WARPS 4
#define AM_STAGES 3
// Keys of a tile: with heads of 64, 32 where 17 to 32 rows share them (8 sequences of 1,500 to 4,100 keys 27.7 us for 28.7 with 16), 16
// where fewer do (8 sequences of 300 to 8,191 keys 22.1 us for 24.7 with 32: four blocks fit a multiprocessor, not two).
template <int HD, int MT> constexpr int few_tile = HD == 128 || MT == 1 ? 16 : 32;

// Up to 16 * MT rows of a (sequence, kv head). A warp takes every fourth tile of TILE keys of the block's stretch with a ring of
// its own in shared memory, and the warps' ranges are joined at the end in their order. OUT: with values and output.
// ALL (grid: cluster, pairs): the blocks of a cluster share all keys of a sequence, exchange their rows' maxima and sums over
// distributed shared memory, join the output and sum the weights of their own keys, whose products they kept: one
// launch does it all. Otherwise (grid: stretches, pairs, row chunks) this is step (1).
template <int HD, int MT, bool OUT, bool ALL>
__global__ void __launch_bounds__(AM_WARPS * 32) weights_part_mma_kernel(WeightArgs a) {
    constexpr int TILE = few_tile<HD, MT>;
    constexpr int LDS = HD + 8, KS = HD / 16, DT = HD / 8, NT = TILE / 8, KK = TILE / 16, CH = HD / 8;
    constexpr int HALF = TILE * LDS * 2, STAGE = HALF * (OUT ? 2 : 1);        // bytes
    constexpr int TEAM = MT == 1 ? 16 : 8;                                    // blocks of a cluster at most
    extern __shared__ __align__(16) unsigned char raw[];
    pdl_wait();
    const int split = blockIdx.x, seq = blockIdx.y / a.kv_heads, kvh = blockIdx.y % a.kv_heads, m0 = blockIdx.z * 16 * MT;
    const Seq s = seq_of(a, seq);
    if (m0 >= s.rows) return;                                                 // the same for a whole cluster
    const int team = ALL ? (int)gridDim.x : 1;
    const int share = ALL ? (s.length + team * TILE - 1) / (team * TILE) * TILE : a.split_keys;
    const int first = split * share, last = min(s.length, first + share);
    if (ALL) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");        // started: waited for before remote stores
    else if (first >= last) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = a.heads / a.kv_heads;
    const int* pages = a.table + (size_t)seq * a.width;
    const bf16* kp = (const bf16*)a.k;
    const bf16* vp = (const bf16*)a.v;
    unsigned char* mine = raw + (size_t)warp * AM_STAGES * STAGE;
    const uint32_t mine32 = (uint32_t)__cvta_generic_to_shared(mine);
    const int t_first = first / TILE, t_last = (last + TILE - 1) / TILE;
    const int n_mine = max(0, t_last - t_first - warp + AM_WARPS - 1) / AM_WARPS;
    auto there = [&](int page) { return page >= 0 && page < a.n_pages; };
    int page_next = 0 < n_mine ? pages[(t_first + warp) * TILE / CML_PAGE] : -1;         // a tile's page is looked up a tile ahead
    int ahead[AM_STAGES - 1];                                                 // the pages of the tiles in flight, -1: none
    // this lane's 16 bytes of a tile's first rows, in the page and in the stage; the others lie at constant distances
    const int lane_row = lane / CH, lane_in = lane_row * HD + lane % CH * 8;
    const uint32_t lane_out = mine32 + (uint32_t)(lane_row * LDS + lane % CH * 8) * 2;
    const bf16* const k_lane = kp + (size_t)kvh * CML_PAGE * HD + lane_in;
    const bf16* const v_lane = OUT ? vp + (size_t)kvh * CML_PAGE * HD + lane_in : nullptr;
    const size_t page_elems = (size_t)a.kv_heads * CML_PAGE * HD;
    int next_tile = t_first + warp, next_stage = 0, to_issue = n_mine;
    auto issue = [&]() {
        int follow = -1;
        if (to_issue > 0) {
            const int t = next_tile, page = page_next;
            next_tile += AM_WARPS;
            if (--to_issue > 0) page_next = pages[next_tile * TILE / CML_PAGE];
            const bool ok = there(page);
            const size_t at = (size_t)(ok ? page : 0) * page_elems + (size_t)(t * TILE % CML_PAGE) * HD;
            const uint32_t dst = lane_out + (uint32_t)next_stage * STAGE;
            const int valid = ok ? last - t * TILE : 0;
            follow = ok ? page : -1;
            if (valid >= TILE) {
#pragma unroll
                for (int c = 0; c < TILE * CH / 32; ++c) {
                    cp_async16(dst + c * (32 / CH) * LDS * 2, k_lane + at + c * (32 / CH) * HD);
                    if (OUT) cp_async16(dst + HALF + c * (32 / CH) * LDS * 2, v_lane + at + c * (32 / CH) * HD);
                }
            } else {
#pragma unroll
                for (int c = 0; c < TILE * CH / 32; ++c) {
                    const bool in = lane_row + c * (32 / CH) < valid;
                    cp_async16_or_zero(dst + c * (32 / CH) * LDS * 2, k_lane + at + c * (32 / CH) * HD, in);
                    if (OUT) cp_async16_or_zero(dst + HALF + c * (32 / CH) * LDS * 2, v_lane + at + c * (32 / CH) * HD, in);
                }
            }
            next_stage = next_stage + 1 == AM_STAGES ? 0 : next_stage + 1;
        }
#pragma unroll
        for (int i = 0; i < AM_STAGES - 2; ++i) ahead[i] = ahead[i + 1];
        ahead[AM_STAGES - 2] = follow;
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < AM_STAGES - 1; ++i) issue();
    // the rows of q as A fragments (zero where there is no row); a thread holds rows lane / 4 and + 8 of each 16
    uint32_t qa[MT][KS][4];
    int pos[MT][2];                                                           // the last place a row sees, -1: no row
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int m = m0 + mt * 16 + (lane >> 2) + 8 * h;
            const bool in = m < s.rows;
            const int j = in ? m / group : 0;
            pos[mt][h] = in ? s.start + j : -1;
            const bf16* qr = (const bf16*)a.q + (long long)(s.row0 + j) * a.q_stride + (long long)(kvh * group + (in ? m % group : 0)) * HD + 2 * (lane & 3);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                qa[mt][ks][h] = in ? *reinterpret_cast<const uint32_t*>(qr + ks * 16) : 0u;
                qa[mt][ks][h + 2] = in ? *reinterpret_cast<const uint32_t*>(qr + ks * 16 + 8) : 0u;
            }
        }
    float top[MT][2], sum[MT][2];
    float o[MT][OUT ? DT : 1][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        top[mt][0] = top[mt][1] = -CUDART_INF_F;
        sum[mt][0] = sum[mt][1] = 0.f;
#pragma unroll
        for (int d = 0; d < (OUT ? DT : 1); ++d) o[mt][d][0] = o[mt][d][1] = o[mt][d][2] = o[mt][d][3] = 0.f;
    }
    const int mat = lane >> 3, rr = lane & 7;
    const int group_rows = a.max_new * group;
    const Kept products = kept_of(a, blockIdx.y, kvh, group_rows);
    int stage = 0;
    const uint32_t k_frag = mine32 + (uint32_t)(((mat >> 1) * 8 + rr) * LDS + (mat & 1) * 8) * 2;
    const uint32_t v_frag = mine32 + HALF + (uint32_t)(((mat & 1) * 8 + rr) * LDS + (mat >> 1) * 8) * 2;
    for (int place0 = (t_first + warp) * TILE; place0 < last; place0 += AM_WARPS * TILE) {
        cp_async_wait<AM_STAGES - 2>();
        __syncwarp();
        const int page = ahead[0];
        const bool ok = page >= 0;
        issue();
        const uint32_t k32 = k_frag + (uint32_t)stage * STAGE, v32 = v_frag + (uint32_t)stage * STAGE;
        unsigned char* const here = mine + (size_t)stage * STAGE;
        stage = stage + 1 == AM_STAGES ? 0 : stage + 1;
        float x[MT][NT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int n = 0; n < NT; ++n) x[mt][n][0] = x[mt][n][1] = x[mt][n][2] = x[mt][n][3] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int np = 0; np < NT / 2; ++np) {
                uint32_t b0, b1, b2, b3;
                ldsm_x4(k32 + (np * 16 * LDS + ks * 16) * 2, b0, b1, b2, b3);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    mma_bf16(x[mt][np * 2], qa[mt][ks], b0, b1);
                    mma_bf16(x[mt][np * 2 + 1], qa[mt][ks], b2, b3);
                }
            }
        // mask; the products are kept
        const int key0 = place0 + 2 * (lane & 3);
        const bool whole = ok && place0 + TILE - 1 <= s.start && place0 + TILE <= last;     // every row sees every key
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            if (!whole) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = key0 + n * 8 + (i & 1);
                        if (!(ok && key < last && key <= pos[mt][i >> 1])) x[mt][n][i] = -CUDART_INF_F;
                    }
            }
            if (ALL && ok) {
                float* const kept = products.at(place0 / CML_PAGE, page) + key0 % CML_PAGE;
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (pos[mt][h] >= 0) {
                        float* row = kept + (mt * 16 + (lane >> 2) + 8 * h) * CML_PAGE;
#pragma unroll
                        for (int n = 0; n < NT; ++n) *reinterpret_cast<float2*>(row + n * 8) = make_float2(x[mt][n][2 * h], x[mt][n][2 * h + 1]);
                    }
            }
        }
        // The reference of the exponentials moves only when a row passes it by a factor of 2^6: a vote, seldom more.
        float now[MT][2];
        bool passed = false;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                now[mt][h] = x[mt][0][2 * h];
#pragma unroll
                for (int n = 0; n < NT; ++n) now[mt][h] = fmaxf(now[mt][h], fmaxf(x[mt][n][2 * h], x[mt][n][2 * h + 1]));
                now[mt][h] *= a.scale;
                passed = passed || now[mt][h] > top[mt][h] + 6.f;
            }
        if (__any_sync(0xffffffffu, passed)) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float next = fmaxf(now[mt][h], __shfl_xor_sync(0xffffffffu, now[mt][h], 1));
                    next = fmaxf(top[mt][h], fmaxf(next, __shfl_xor_sync(0xffffffffu, next, 2)));
                    const float corr = top[mt][h] == -CUDART_INF_F ? 0.f : fast_exp2(top[mt][h] - next);
                    top[mt][h] = next;
                    sum[mt][h] *= corr;
#pragma unroll
                    for (int d = 0; d < (OUT ? DT : 1); ++d) o[mt][d][2 * h] *= corr, o[mt][d][2 * h + 1] *= corr;
                }
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float ref = top[mt][h] == -CUDART_INF_F ? 0.f : top[mt][h];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        x[mt][n][2 * h + i] = fast_exp2(fmaf(x[mt][n][2 * h + i], a.scale, -ref));
                        sum[mt][h] += x[mt][n][2 * h + i];
                    }
            }
        if (OUT) {
            bf16* vs = reinterpret_cast<bf16*>(here + HALF);
            if (s.fresh > 1 && place0 + TILE > s.start + 1) {
                // New places that not every row sees: a probability of zero times what such a place holds must stay zero even
                // where that is infinite, so their products are made apart, and the tensor cores get zeros.
                // The probabilities pass through the room of the tile's keys, which are done.
                float* ps = reinterpret_cast<float*>(here);                   // [16 * MT rows][TILE]
                __syncwarp();
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            *reinterpret_cast<float2*>(ps + (mt * 16 + (lane >> 2) + 8 * h) * TILE + n * 8 + 2 * (lane & 3)) =
                                make_float2(x[mt][n][2 * h], x[mt][n][2 * h + 1]);
                __syncwarp();
#pragma unroll 1
                for (int kk = max(0, s.start + 1 - place0); kk < TILE && place0 + kk < last; ++kk) {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float p = ps[(mt * 16 + (lane >> 2) + 8 * h) * TILE + kk];
                            if (p != 0.f) {
#pragma unroll
                                for (int d = 0; d < DT; ++d) {
                                    const uint32_t w = *reinterpret_cast<const uint32_t*>(vs + kk * LDS + d * 8 + 2 * (lane & 3));
                                    o[mt][d][2 * h] = fmaf(p, __uint_as_float(w << 16), o[mt][d][2 * h]);
                                    o[mt][d][2 * h + 1] = fmaf(p, __uint_as_float(w & 0xffff0000u), o[mt][d][2 * h + 1]);
                                }
                            }
                        }
                }
                __syncwarp();
                const int from = max(0, s.start + 1 - place0);
                for (int c = lane; c < (TILE - from) * CH; c += 32)
                    *reinterpret_cast<uint4*>(vs + (from + c / CH) * LDS + (c % CH) * 8) = make_uint4(0, 0, 0, 0);
                __syncwarp();
            }
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                uint32_t pa[MT][4];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    pa[mt][0] = pack_bf16(x[mt][2 * kk][0], x[mt][2 * kk][1]);
                    pa[mt][1] = pack_bf16(x[mt][2 * kk][2], x[mt][2 * kk][3]);
                    pa[mt][2] = pack_bf16(x[mt][2 * kk + 1][0], x[mt][2 * kk + 1][1]);
                    pa[mt][3] = pack_bf16(x[mt][2 * kk + 1][2], x[mt][2 * kk + 1][3]);
                }
#pragma unroll
                for (int dp = 0; dp < DT / 2; ++dp) {
                    uint32_t b0, b1, b2, b3;
                    ldsm_x4_t(v32 + (kk * 16 * LDS + dp * 16) * 2, b0, b1, b2, b3);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        mma_bf16(o[mt][dp * 2], pa[mt], b0, b1);
                        mma_bf16(o[mt][dp * 2 + 1], pa[mt], b2, b3);
                    }
                }
            }
        }
    }
    cp_async_wait<0>();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            sum[mt][h] += __shfl_xor_sync(0xffffffffu, sum[mt][h], 1);
            sum[mt][h] += __shfl_xor_sync(0xffffffffu, sum[mt][h], 2);
        }
    __syncthreads();                                                          // every warp is done with its ring
    // The next kernel may begin beside what is left: earlier it only took room (16 long sequences 348 us for 345).
    pdl_launch_dependents();
    // the warps' ranges: [warp][16 * MT rows][maximum, sum, output]
    constexpr int RW = OUT ? HD + 4 : 4;
    static_assert(AM_WARPS * 16 * MT * RW * 4 + (OUT ? 16 * MT * HD * 4 : 0) <= AM_WARPS * AM_STAGES * STAGE, "the results take the ring's room");
    static_assert(!OUT || 16 * MT * TILE * 4 <= HALF, "the probabilities take the room of a tile's keys");
    float* red = reinterpret_cast<float*>(raw);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float* dst = red + ((size_t)warp * 16 * MT + mt * 16 + (lane >> 2) + 8 * h) * RW;
            if ((lane & 3) == 0) dst[0] = top[mt][h], dst[1] = sum[mt][h];
            if (OUT) {
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    dst[4 + d * 8 + 2 * (lane & 3)] = o[mt][d][2 * h];
                    dst[4 + d * 8 + 2 * (lane & 3) + 1] = o[mt][d][2 * h + 1];
                }
            }
        }
    __syncthreads();
    const size_t base = ((size_t)blockIdx.y * a.n_splits + split) * group_rows + m0;
    const int rows = min(16 * MT, s.rows - m0);
    constexpr int PER = OUT ? HD / 4 : 1;
    float* const own = red + (size_t)AM_WARPS * 16 * MT * RW;                 // ALL: [16 * MT rows][HD], the block's output
    __shared__ float2 stat_s[ALL ? TEAM * 16 * MT : 1];                // ALL: [blocks][rows] maximum and sum, of the whole cluster
    __shared__ float factor_s[ALL ? TEAM * 16 * MT : 1];               // ALL: what a block's output counts in the joined one
    __shared__ float2 join_s[ALL ? 16 * MT : 1];                              // ALL: [rows] maximum and 1 / sum of all keys
    if (ALL) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    for (int i = threadIdx.x; i < rows * PER; i += AM_WARPS * 32) {
        const int m = i / PER, d = i % PER * 4;
        float most = -CUDART_INF_F, f[AM_WARPS], l = 0.f;
#pragma unroll
        for (int w = 0; w < AM_WARPS; ++w) most = fmaxf(most, red[((size_t)w * 16 * MT + m) * RW]);
#pragma unroll
        for (int w = 0; w < AM_WARPS; ++w) {
            const float* src = red + ((size_t)w * 16 * MT + m) * RW;
            f[w] = src[0] == -CUDART_INF_F ? 0.f : fast_exp2(src[0] - most);
            l += f[w] * src[1];
        }
        if (OUT) {
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < AM_WARPS; ++w) {
                const float4 t = *reinterpret_cast<const float4*>(red + ((size_t)w * 16 * MT + m) * RW + 4 + d);
                v.x += f[w] * t.x; v.y += f[w] * t.y; v.z += f[w] * t.z; v.w += f[w] * t.w;
            }
            *reinterpret_cast<float4*>(ALL ? own + m * HD + d : a.acc + (base + m) * HD + d) = v;
        }
        if (d == 0) {
            if (ALL) {
                for (int c = 0; c < team; ++c) cg::this_cluster().map_shared_rank(&stat_s[0], c)[split * 16 * MT + m] = make_float2(most, l);
            } else {
                a.stats[(base + m) * 2] = most;
                a.stats[(base + m) * 2 + 1] = l;
            }
        }
    }
    if (!ALL) return;
    cg::this_cluster().sync();
    if ((int)threadIdx.x < rows) {
        const int m = threadIdx.x;
        float most = -CUDART_INF_F, l = 0.f;
        for (int c = 0; c < team; ++c) most = fmaxf(most, stat_s[c * 16 * MT + m].x);
        for (int c = 0; c < team; ++c) {
            const float2 t = stat_s[c * 16 * MT + m];
            const float f = t.x == -CUDART_INF_F ? 0.f : fast_exp2(t.x - most);
            factor_s[c * 16 * MT + m] = f;
            l += f * t.y;
        }
        join_s[m] = most == -CUDART_INF_F ? make_float2(0.f, 0.f) : make_float2(most, 1.f / l);
    }
    __syncthreads();
    if (OUT) {                                                                // the output's elements in equal shares, the blocks in their order
        const int pairs2 = rows * HD / 2;
        for (int i = split * AM_WARPS * 32 + threadIdx.x; i < pairs2; i += team * AM_WARPS * 32) {
            const int m = i / (HD / 2), d = i % (HD / 2) * 2;
            float x = 0.f, y = 0.f;
#pragma unroll 4
            for (int c = 0; c < team; ++c) {
                const float2 t = *reinterpret_cast<const float2*>(cg::this_cluster().map_shared_rank(own, c) + m * HD + d);
                const float f = factor_s[c * 16 * MT + m];
                x += f * t.x, y += f * t.y;
            }
            const float inv = join_s[m].y;
            bf16* dst = (bf16*)a.out + (long long)(s.row0 + m / group) * a.out_stride + (long long)(kvh * group + m % group) * HD + d;
            if ((a.out_stride & 1) == 0 && (((uintptr_t)a.out) & 3) == 0) *reinterpret_cast<uint32_t*>(dst) = pack_bf16(x * inv, y * inv);
            else dst[0] = __float2bfloat16_rn(x * inv), dst[1] = __float2bfloat16_rn(y * inv);
        }
    }
    // the weights of this block's keys, two groups of four keys a thread in flight
    for (int group0 = first + 4 * (int)threadIdx.x; group0 < last; group0 += 2 * AM_WARPS * 128) {
        float g[2][4], old[2][4];
        size_t at[2];
        bool has[2];
        const float* x[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int place = group0 + u * AM_WARPS * 128;
            const int page = place < last ? pages[place / CML_PAGE] : -1;
            has[u] = there(page);
            at[u] = ((size_t)(has[u] ? page : 0) * a.kv_heads + kvh) * CML_PAGE + place % CML_PAGE;
            const float4 t = *reinterpret_cast<const float4*>(a.scores + at[u]);
            old[u][0] = t.x, old[u][1] = t.y, old[u][2] = t.z, old[u][3] = t.w;
            // (no place: any products that are there; what comes of them goes nowhere)
            x[u] = has[u] ? products.at(place / CML_PAGE, page) + place % CML_PAGE : a.kept;
            g[u][0] = g[u][1] = g[u][2] = g[u][3] = 0.f;
        }
#pragma unroll 4
        for (int m = 0; m < rows; ++m) {
            const float2 j = join_s[m];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float4 t = *reinterpret_cast<const float4*>(x[u] + m * CML_PAGE);
                g[u][0] = fmaf(fast_exp2(fmaf(t.x, a.scale, -j.x)), j.y, g[u][0]);
                g[u][1] = fmaf(fast_exp2(fmaf(t.y, a.scale, -j.x)), j.y, g[u][1]);
                g[u][2] = fmaf(fast_exp2(fmaf(t.z, a.scale, -j.x)), j.y, g[u][2]);
                g[u][3] = fmaf(fast_exp2(fmaf(t.w, a.scale, -j.x)), j.y, g[u][3]);
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if (!has[u]) continue;
            const int place = group0 + u * AM_WARPS * 128;
#pragma unroll
            for (int k = 0; k < 4; ++k) g[u][k] += place + k < s.old ? old[u][k] : 0.f;
            if (place + 4 <= last) *reinterpret_cast<float4*>(a.scores_out + at[u]) = make_float4(g[u][0], g[u][1], g[u][2], g[u][3]);
            else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (place + k < last) a.scores_out[at[u] + k] = g[u][k];
            }
        }
    }
    if (OUT) cg::this_cluster().sync();                                       // a block's output stays until every block has read it
}

#define AR_WARPS 4
// (3) for more than 32 rows with output: a warp keeps 64 keys in registers as the operand of 16 rows and lets the rows of q pass, so that a
// key's sum over the rows stays in one quad of lanes, in the order of the rows. Grid (256 keys, pairs).
#define AC_ROWS 32              // rows of q in a stage
#define AC_STAGES 4
template <int HD>
__global__ void __launch_bounds__(AR_WARPS * 32, 2) weights_keys_mma_kernel(WeightArgs a) {
    constexpr int LDS = HD + 8, KS = HD / 16, CH = HD / 8, KEYS = AR_WARPS * 64;
    constexpr int QSTAGE = AC_ROWS * LDS * 2 + AC_ROWS * 16;                  // rows, then (maximum, 1 / sum, last place) of each
    extern __shared__ __align__(16) unsigned char raw[];
    pdl_wait();
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int seq = blockIdx.y / a.kv_heads, kvh = blockIdx.y % a.kv_heads, key0 = blockIdx.x * KEYS;
    const Seq s = seq_of(a, seq);
    if (key0 >= s.length) return;
    const int group = a.heads / a.kv_heads, group_rows = a.max_new * group;
    const int* pages = a.table + (size_t)seq * a.width;
    const uint32_t raw32 = (uint32_t)__cvta_generic_to_shared(raw);
    // this warp's page of keys
    const int place0 = key0 + warp * 64;
    int page = place0 < s.length ? pages[place0 / CML_PAGE] : -1;
    if (page >= a.n_pages) page = -1;
    const int valid = page < 0 ? 0 : min(64, s.length - place0);
    {
        const bf16* src = (const bf16*)a.k + ((size_t)max(page, 0) * a.kv_heads + kvh) * CML_PAGE * HD;
        const uint32_t dst = raw32 + (uint32_t)(warp * 64 * LDS) * 2;
#pragma unroll
        for (int c0 = 0; c0 < 64 * CH; c0 += 32) {
            const int c = c0 + lane, r = c / CH, cc = c % CH;
            cp_async16_or_zero(dst + (uint32_t)(r * LDS + cc * 8) * 2, src + (size_t)r * HD + cc * 8, r < valid);
        }
        cp_async_commit();
        cp_async_wait<0>();
        __syncwarp();
    }
    const int mat = lane >> 3, rr = lane & 7;
    uint32_t ka[4][KS][4];
#pragma unroll
    for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
            ldsm_x4(raw32 + (uint32_t)((warp * 64 + mt * 16 + (mat & 1) * 8 + rr) * LDS + ks * 16 + (mat >> 1) * 8) * 2, ka[mt][ks][0], ka[mt][ks][1],
                    ka[mt][ks][2], ka[mt][ks][3]);
    __syncthreads();                                                          // the keys are in registers: their room holds the rows of q now
    const int chunks = (s.rows + AC_ROWS - 1) / AC_ROWS;
    auto issue = [&](int c) {
        if (c < chunks) {
            unsigned char* st = raw + (size_t)(c % AC_STAGES) * QSTAGE;
            const uint32_t dst = raw32 + (uint32_t)(c % AC_STAGES) * QSTAGE;
#pragma unroll
            for (int c0 = 0; c0 < AC_ROWS * CH; c0 += AR_WARPS * 32) {
                const int i = c0 + threadIdx.x, r = i / CH, cc = i % CH, m = c * AC_ROWS + r;
                const bool in = m < s.rows;
                const bf16* src = (const bf16*)a.q + (long long)(s.row0 + (in ? m / group : 0)) * a.q_stride + (long long)(kvh * group + (in ? m % group : 0)) * HD + cc * 8;
                cp_async16_or_zero(dst + (uint32_t)(r * LDS + cc * 8) * 2, src, in);
            }
            if (threadIdx.x < AC_ROWS) {
                const int m = c * AC_ROWS + threadIdx.x;
                float2 j = make_float2(0.f, 0.f);
                if (m < s.rows) j = *reinterpret_cast<const float2*>(a.joined + ((size_t)blockIdx.y * group_rows + m) * 2);
                float4* tail = reinterpret_cast<float4*>(st + AC_ROWS * LDS * 2);
                tail[threadIdx.x] = make_float4(j.x, j.y, __int_as_float(m < s.rows ? s.start + m / group : -1), 0.f);
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < AC_STAGES - 1; ++i) issue(i);
    float gained[4][2];
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) gained[mt][0] = gained[mt][1] = 0.f;
    const bool whole = place0 + 63 <= s.start;                                // every row sees every key of this warp
    for (int c = 0; c < chunks; ++c) {
        cp_async_wait<AC_STAGES - 2>();
        __syncthreads();
        issue(c + AC_STAGES - 1);
        if (valid == 0) continue;
        const uint32_t q32 = raw32 + (uint32_t)(c % AC_STAGES) * QSTAGE;
        const float4* tail = reinterpret_cast<const float4*>(raw + (size_t)(c % AC_STAGES) * QSTAGE + AC_ROWS * LDS * 2);
#pragma unroll 1
        for (int half = 0; half < AC_ROWS / 16; ++half) {
            float x[4][2][4];
#pragma unroll
            for (int mt = 0; mt < 4; ++mt)
#pragma unroll
                for (int n = 0; n < 2; ++n) x[mt][n][0] = x[mt][n][1] = x[mt][n][2] = x[mt][n][3] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                uint32_t b0, b1, b2, b3;
                ldsm_x4(q32 + (uint32_t)((half * 16 + (mat >> 1) * 8 + rr) * LDS + ks * 16 + (mat & 1) * 8) * 2, b0, b1, b2, b3);
#pragma unroll
                for (int mt = 0; mt < 4; ++mt) {
                    mma_bf16(x[mt][0], ka[mt][ks], b0, b1);
                    mma_bf16(x[mt][1], ka[mt][ks], b2, b3);
                }
            }
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float4 row = tail[half * 16 + n * 8 + 2 * (lane & 3) + i];
                    if (whole && c * AC_ROWS + AC_ROWS <= s.rows) {           // (rows that are none: zero times an infinite key is no zero)
#pragma unroll
                        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
                            for (int h = 0; h < 2; ++h) gained[mt][h] = fmaf(fast_exp2(fmaf(x[mt][n][2 * h + i], a.scale, -row.x)), row.y, gained[mt][h]);
                    } else {
                        const int sees = __float_as_int(row.z) - place0;
#pragma unroll
                        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
                            for (int h = 0; h < 2; ++h)
                                if (mt * 16 + (lane >> 2) + 8 * h <= sees)
                                    gained[mt][h] = fmaf(fast_exp2(fmaf(x[mt][n][2 * h + i], a.scale, -row.x)), row.y, gained[mt][h]);
                    }
                }
        }
    }
    cp_async_wait<0>();
    const size_t at = ((size_t)max(page, 0) * a.kv_heads + kvh) * CML_PAGE;
#pragma unroll
    for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float g = gained[mt][h];
            g += __shfl_xor_sync(0xffffffffu, g, 1);
            g += __shfl_xor_sync(0xffffffffu, g, 2);
            const int key = mt * 16 + (lane >> 2) + 8 * h;
            if ((lane & 3) == 0 && key < valid) a.scores_out[at + key] = (place0 + key < s.old ? a.scores[at + key] : 0.f) + g;
        }
}

// A launch of clusters of `team` blocks, one for each pair.
template <typename K>
static cudaError_t launch_team(K kernel, const WeightArgs& a, unsigned pairs, int team, int threads, size_t smem, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)team, pairs);
    cfg.blockDim = dim3((unsigned)threads);
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
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <typename T, int R>
static cudaError_t launch_plain_all(const WeightArgs& a, unsigned pairs, size_t smem, cudaStream_t s) {
    const cudaError_t e = cml_allow_smem<weights_part_kernel<T, R, true>>(smem);
    if (e != cudaSuccess) return e;
    int team = 1;                                                 // two blocks for every multiprocessor, none without a page of keys
    while (team < AW_TEAM && (long long)pairs * team < 2ll * cml_sm_count() && team * CML_PAGE < a.max_len) team *= 2;
    return launch_team(weights_part_kernel<T, R, true>, a, pairs, team, AW_THREADS, smem, s);
}

template <typename T>
static cudaError_t launch_plain(WeightArgs& a, cudaStream_t s) {
    const unsigned pairs = (unsigned)a.n_seqs * (unsigned)a.kv_heads;
    const int group_rows = a.max_new * (a.heads / a.kv_heads);
    const size_t k_page = (size_t)CML_PAGE * (a.k_dim * sizeof(T) + 16), v_page = a.out ? (size_t)CML_PAGE * a.v_dim * sizeof(T) : 0;
    auto rest = [&](int rows) { return (size_t)rows * (a.k_dim + 5 * CML_PAGE + 4 + (a.out ? a.v_dim : 0)) * 4; };
    a.stages = 2 * (k_page + v_page) + rest(AW_ROWS) <= 220 * 1024 ? 2 : 1;
    const size_t groups = (size_t)AW_ROWS * AW_THREADS * 4 * 4;               // the output of all groups of threads, where the ring was
    const size_t ring = a.stages * (k_page + v_page) > groups ? a.stages * (k_page + v_page) : groups;
    if (group_rows <= 4) return launch_plain_all<T, 4>(a, pairs, ring + rest(4), s);
    if (group_rows <= AW_ROWS) return launch_plain_all<T, AW_ROWS>(a, pairs, ring + rest(AW_ROWS), s);
    const size_t smem1 = ring + rest(AW_ROWS), smem3 = k_page + (size_t)AW_ROWS * (a.k_dim + 4 * CML_PAGE) * 4;
    cudaError_t e = cml_allow_smem<weights_part_kernel<T, AW_ROWS, false>>(smem1);
    if (e == cudaSuccess) e = cml_allow_smem<weights_sum_kernel<T>>(smem3);
    if (e != cudaSuccess) return e;
    e = launch_pdl(weights_part_kernel<T, AW_ROWS, false>, dim3((unsigned)a.n_splits, pairs, (unsigned)((group_rows + AW_ROWS - 1) / AW_ROWS)), dim3(AW_THREADS),
                   smem1, s, a);
    if (e != cudaSuccess) return e;
    e = launch_pdl(weights_join_kernel<T>, dim3((unsigned)group_rows, pairs), dim3(AW_THREADS), 0, s, a);
    if (e != cudaSuccess) return e;
    return launch_pdl(weights_sum_kernel<T>, dim3((unsigned)((a.max_len + CML_PAGE - 1) / CML_PAGE), pairs), dim3(AW_THREADS), smem3, s, a);
}

template <int HD, int MT, bool OUT>
static cudaError_t launch_all(const WeightArgs& a, unsigned pairs, int team, size_t smem, cudaStream_t s) {
    const auto kernel = weights_part_mma_kernel<HD, MT, OUT, true>;
    cudaError_t e = cml_allow_smem<weights_part_mma_kernel<HD, MT, OUT, true>>(smem);
    if (e == cudaSuccess && team > 8) e = cml_allow_wide_clusters<weights_part_mma_kernel<HD, MT, OUT, true>>();
    if (e != cudaSuccess) return e;
    return launch_team(kernel, a, pairs, team, AM_WARPS * 32, smem, s);
}

#include "attention_weights_tc.cuh"

template <int HD>
static cudaError_t launch_mma(const WeightArgs& a, int* err, cudaStream_t s) {
    const unsigned pairs = (unsigned)a.n_seqs * (unsigned)a.kv_heads;
    const int rows = a.max_new * (a.heads / a.kv_heads);
    constexpr size_t ring1 = (size_t)AM_WARPS * AM_STAGES * few_tile<HD, 1> * (HD + 8) * 2, ring2 = ring1 / few_tile<HD, 1> * few_tile<HD, 2>;
    cudaError_t e;
    if (rows <= 32) {
        // Where the blocks of all sequences run at the same time, more of them; beyond that up to twice as many, for sequences of
        // unequal lengths, while a block has 768 keys (8 sequences of up to 8,191 keys: 34.6 us with eight blocks, 43 with four;
        // 64 of up to 1,047: 24.0 with one, 35 with two); none without a tile of keys for each warp. Long sequences of which there are
        // few take clusters of sixteen (one of 32,001 keys and eight kv heads: 41.6 us for 52.4; at 2,047 keys they are equal).
        const long long slots = 2ll * cml_sm_count();
        int team = 1;
        while (team < 8 && (pairs * team * 2 <= slots || (pairs * team * 2 <= 2 * slots && a.max_len >= team * 2 * 768)) && team * 128 < a.max_len) team *= 2;
        if (rows <= 16 && team == 8 && pairs * 16 <= (unsigned)cml_sm_count() && a.max_len >= 4096) team = 16;
        if (rows <= 16) return a.out ? launch_all<HD, 1, true>(a, pairs, team, 2 * ring1, s) : launch_all<HD, 1, false>(a, pairs, team, ring1, s);
        return a.out ? launch_all<HD, 2, true>(a, pairs, team, 2 * ring2, s) : launch_all<HD, 2, false>(a, pairs, team, ring2, s);
    }
    // Without output and beyond the rows whose products are kept: tcgen05, in two launches (four sequences of 4,000 keys, 8 kv heads of
    // 128: 27.9 us whatever the rows up to 128; the one launch above takes 26.2 with 32 rows, 14.3 with 8, and its split form, which
    // stood here, 56 with 36 and 94 with 128).
    if (a.out == nullptr) return launch_tc<HD>(a, err, s);
    e = cml_allow_smem<weights_part_mma_kernel<HD, 2, true, false>>(2 * ring2);
    if (e == cudaSuccess)
        e = launch_pdl(weights_part_mma_kernel<HD, 2, true, false>, dim3((unsigned)a.n_splits, pairs, (unsigned)((rows + 31) / 32)), dim3(AM_WARPS * 32),
                       2 * ring2, s, a);
    if (e != cudaSuccess) return e;
    e = launch_pdl(weights_join_kernel<bf16>, dim3((unsigned)rows, pairs), dim3(AW_THREADS), 0, s, a);
    if (e != cudaSuccess) return e;
    constexpr size_t keys = (size_t)AR_WARPS * 64 * (HD + 8) * 2, stages = (size_t)AC_STAGES * AC_ROWS * ((HD + 8) * 2 + 16);
    constexpr size_t smem = keys > stages ? keys : stages;
    e = cml_allow_smem<weights_keys_mma_kernel<HD>>(smem);
    if (e != cudaSuccess) return e;
    return launch_pdl(weights_keys_mma_kernel<HD>, dim3((unsigned)((a.max_len + AR_WARPS * 64 - 1) / (AR_WARPS * 64)), pairs), dim3(AR_WARPS * 32), smem, s, a);
}

extern "C" int cml_attn_paged_weights(const void* q, int dtype, long long q_stride, void* out, long long out_stride, const void* k,
                                      const void* v, const float* scores, float* scores_out, const int* table, int width, int n_pages,
                                      const int* row0, const int* start, const int* fresh, const int* cached, int n_seqs, int n_rows, int heads,
                                      int kv_heads, int k_dim, int v_dim, int max_new, int max_len, float scale, int split_keys,
                                      float* scratch, int* err, void* stream) {
    if (dtype != CML_DTYPE_F32 && dtype != CML_DTYPE_BF16) return CML_ERR_BAD_DTYPE;
    if (n_seqs <= 0 || n_rows <= 0) return 0;
    if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || k_dim < 16 || k_dim > 256 || k_dim % 16 || v_dim < 16 || v_dim > 256 || v_dim % 16)
        return CML_ERR_BAD_SIZE;
    if (!(scale > 0.f) || !(scale < __builtin_inff())) return CML_ERR_BAD_SIZE;
    if (width <= 0 || n_pages <= 0 || max_new <= 0 || max_len <= 0 || split_keys <= 0 || split_keys % CML_PAGE) return CML_ERR_BAD_SIZE;
    const long long pairs = (long long)n_seqs * kv_heads, rows = (long long)max_new * (heads / kv_heads);
    if (pairs > 65535 || rows > 65535ll * AW_ROWS || max_len > (1 << 28) || width > (1 << 24)) return CML_ERR_BAD_SIZE;
    if (((uintptr_t)k | (uintptr_t)(out ? v : nullptr)) & 15) return CML_ERR_BAD_ALIGN;
    WeightArgs a = {};
    a.q = q; a.q_stride = q_stride; a.out = out; a.out_stride = out_stride; a.k = k; a.v = v; a.scores = scores; a.scores_out = scores_out;
    a.table = table; a.width = width; a.n_pages = n_pages; a.row0 = row0; a.start = start; a.fresh = fresh; a.cached = cached; a.n_seqs = n_seqs;
    a.n_rows = n_rows; a.heads = heads; a.kv_heads = kv_heads; a.k_dim = k_dim; a.v_dim = v_dim; a.max_new = max_new; a.max_len = max_len;
    a.scale = scale * 1.4426950408889634f; a.split_keys = split_keys;
    a.n_splits = (max_len + split_keys - 1) / split_keys;
    auto room = [](long long n) { return (n + 31) / 32 * 32; };               // every part on a boundary of 128 bytes
    a.joined = scratch;
    a.stats = a.joined + room(pairs * rows * 2);
    a.acc = a.stats + room(pairs * rows * 2 * a.n_splits);
    a.kept = scratch;                                                         // (one launch keeps products, several keep the parts above)
    const int blocks = (max_len + CML_PAGE - 1) / CML_PAGE;                   // ops.attn_weights_plan has the same rule
    a.kept_blocks = (long long)n_seqs * blocks <= n_pages ? blocks : 0;
    if ((((uintptr_t)scratch) & 15) || (((uintptr_t)scores | (uintptr_t)scores_out) & 15)) return CML_ERR_BAD_ALIGN;
    // the tensor cores take rows of q that begin on 16 bytes
    const bool mma = dtype == CML_DTYPE_BF16 && (k_dim == 64 || k_dim == 128) && (out == nullptr || v_dim == k_dim) &&
                     (((uintptr_t)q) & 15) == 0 && q_stride % 8 == 0;
    if (mma && out == nullptr && (err == nullptr || (long long)n_pages * kv_heads * CML_PAGE > 0x7fffffffLL)) return CML_ERR_BAD_SIZE;      // rows of TMA's matrix
    cudaStream_t s = (cudaStream_t)stream;
    const cudaError_t e = mma ? (k_dim == 64 ? launch_mma<64>(a, err, s) : launch_mma<128>(a, err, s))
                              : (dtype == CML_DTYPE_F32 ? launch_plain<float>(a, s) : launch_plain<bf16>(a, s));
    if (e != cudaSuccess) return (int)e;
    return cml_launch_status();
}
