// Attention of a few new tokens per sequence over the paged cache that also keeps what it weighed: the score of every
// cached position gains the attention weight that the step's rows gave it, summed over the query heads of its kv head.
//
//   s = scale q . k      w = exp(s - max s) / sum exp(s - max s)      out = sum w v
//   scores'[place] = (place was cached before the step ? scores[place] : 0) + sum over rows and heads of w
//
// A step's rows are packed: sequence i owns rows row0[i] .. row0[i] + new[i], its row j stands at place start[i] + j and
// sees the places up to its own. Without an output only the scores are made (what a prompt's last rows look at).
//
// The weights of a key are known only when all keys are seen, so the work is cut in three: (1) blocks take stretches of
// a sequence's keys and keep the running maximum, sum and output of their rows; (2) the stretches are joined, in order;
// (3) the products q . k are made again and every key's weights summed, in a fixed order of the rows. Products,
// softmax and sums are float.
#include "common.cuh"
#include <math_constants.h>

#define AW_THREADS 128
#define AW_ROWS 8               // rows (token, head) a block works on together

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
    int n_seqs, n_rows, heads, kv_heads, k_dim, v_dim;
    int max_new, max_len;
    float scale;
    int stages;                  // pages of keys and values a block of (1) keeps in shared memory: 2, or 1 where two do not fit
    int split_keys, n_splits;    // keys of a stretch (a multiple of the page), stretches of the longest sequence
    float* stats;                // [seqs * kv heads][splits][rows][2]: maximum and sum of a stretch
    float* joined;               // [seqs * kv heads][rows][2]: maximum and 1 / sum of all
    float* acc;                  // [seqs * kv heads][splits][rows][v_dim]
};

struct Seq {
    int start, fresh, length, row0, rows;      // rows: (token, head) pairs that share a kv head
};
__device__ __forceinline__ Seq seq_of(const WeightArgs& a, int i) {
    Seq s;
    s.start = max(0, min(a.start[i], 1 << 30));
    s.row0 = a.row0[i];
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
    for (int c = threadIdx.x; c < CML_PAGE * chunks; c += AW_THREADS) {
        const int r = c / chunks, cc = c - r * chunks;
        if (r < valid) cp_async16(at + (uint32_t)(r * stride + cc * 16), (const unsigned char*)src + ((size_t)r * dim) * sizeof(T) + cc * 16);
        else *reinterpret_cast<uint4*>(dst + r * stride + cc * 16) = make_uint4(0, 0, 0, 0);
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

// q of AW_ROWS rows as float into shared memory (zeros where there is no row).
template <typename T>
__device__ __forceinline__ void load_q(const WeightArgs& a, const Seq& s, int kvh, int m0, float* q_s) {
    const int group = a.heads / a.kv_heads;
    for (int c = threadIdx.x; c < AW_ROWS * a.k_dim; c += AW_THREADS) {
        const int m = m0 + c / a.k_dim, d = c % a.k_dim;
        float x = 0.f;
        if (m < s.rows) x = to_f32(((const T*)a.q)[(long long)(s.row0 + m / group) * a.q_stride + (long long)(kvh * group + m % group) * a.k_dim + d]);
        q_s[c] = x;
    }
}

// The scores of this thread's key (threadIdx.x & 63) for four of the block's rows (threadIdx.x >> 6), scaled and masked.
template <typename T>
__device__ __forceinline__ void score4(const WeightArgs& a, const Seq& s, int m0, int place, bool there, const unsigned char* k_row,
                                       const float* q_s, float (&out)[4]) {
    constexpr int N = 16 / sizeof(T);
    const int group = a.heads / a.kv_heads, half = threadIdx.x >> 6;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    const float* q = q_s + half * 4 * a.k_dim;
    for (int d = 0; d < a.k_dim; d += N)
#pragma unroll
        for (int m = 0; m < 4; ++m) acc[m] += dot_chunk<T>(k_row + d * sizeof(T), q + m * a.k_dim + d);
#pragma unroll
    for (int m = 0; m < 4; ++m) {
        const int r = m0 + half * 4 + m;
        out[m] = there && r < s.rows && place <= s.start + r / group ? acc[m] * a.scale : -CUDART_INF_F;
    }
}

// (1) a stretch of keys: grid (stretches, sequences * kv heads, row tiles)
template <typename T>
__global__ void __launch_bounds__(AW_THREADS) weights_part_kernel(WeightArgs a) {
    extern __shared__ __align__(16) unsigned char raw[];
    const int split = blockIdx.x, seq = blockIdx.y / a.kv_heads, kvh = blockIdx.y % a.kv_heads, m0 = blockIdx.z * AW_ROWS;
    pdl_wait();
    pdl_launch_dependents();
    const Seq s = seq_of(a, seq);
    const int first = split * a.split_keys, last = min(s.length, first + a.split_keys);
    if (first >= last || m0 >= s.rows) return;
    const int k_stride = a.k_dim * (int)sizeof(T) + 16, v_stride = a.out ? a.v_dim * (int)sizeof(T) : 0;
    const int page_bytes = CML_PAGE * (k_stride + v_stride);
    float* q_s = reinterpret_cast<float*>(raw + a.stages * page_bytes);
    float* p_s = q_s + AW_ROWS * a.k_dim;                          // [rows][page]
    float* m_s = p_s + AW_ROWS * CML_PAGE;
    float* l_s = m_s + AW_ROWS;
    float* c_s = l_s + AW_ROWS;
    const int* pages = a.table + (size_t)seq * a.width;
    const int p_first = first / CML_PAGE, p_last = (last + CML_PAGE - 1) / CML_PAGE;
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
    load_q<T>(a, s, kvh, m0, q_s);
    if (threadIdx.x < AW_ROWS) m_s[threadIdx.x] = -CUDART_INF_F, l_s[threadIdx.x] = 0.f;
    float o[AW_ROWS][2];
#pragma unroll
    for (int m = 0; m < AW_ROWS; ++m) o[m][0] = o[m][1] = 0.f;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int p = p_first; p < p_last; ++p) {
        if (a.stages > 1) fetch(p + 1);
        else if (p > p_first) fetch(p);
        if (a.stages > 1) cp_async_wait<1>();
        else cp_async_wait<0>();
        __syncthreads();
        const unsigned char* ks = raw + (size_t)((p - p_first) & (a.stages - 1)) * page_bytes;
        const int key = threadIdx.x & 63;
        float sc[4];
        score4<T>(a, s, m0, p * CML_PAGE + key, key < valid_of(p), ks + key * k_stride, q_s, sc);
#pragma unroll
        for (int m = 0; m < 4; ++m) p_s[((threadIdx.x >> 6) * 4 + m) * CML_PAGE + key] = sc[m];
        __syncthreads();
#pragma unroll
        for (int mm = 0; mm < 2; ++mm) {
            const int m = warp * 2 + mm;
            const float a0 = p_s[m * CML_PAGE + lane], a1 = p_s[m * CML_PAGE + lane + 32];
            const float old = m_s[m], now = fmaxf(old, warp_max(fmaxf(a0, a1)));
            const float e0 = a0 == -CUDART_INF_F ? 0.f : expf(a0 - now), e1 = a1 == -CUDART_INF_F ? 0.f : expf(a1 - now);
            const float corr = old == -CUDART_INF_F ? 0.f : expf(old - now);
            const float sum = warp_sum(e0 + e1);
            p_s[m * CML_PAGE + lane] = e0;
            p_s[m * CML_PAGE + lane + 32] = e1;
            __syncwarp();
            if (lane == 0) m_s[m] = now, l_s[m] = l_s[m] * corr + sum, c_s[m] = corr;
        }
        __syncthreads();
        if (a.out) {
            const T* vs = reinterpret_cast<const T*>(ks + CML_PAGE * k_stride);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int d = threadIdx.x + h * AW_THREADS;
                if (d >= a.v_dim) break;
                float t[AW_ROWS];
#pragma unroll
                for (int m = 0; m < AW_ROWS; ++m) t[m] = 0.f;
                for (int kk = 0; kk < CML_PAGE; ++kk) {
                    const float val = to_f32(vs[kk * a.v_dim + d]);
#pragma unroll
                    for (int m = 0; m < AW_ROWS; ++m) {
                        const float w = p_s[m * CML_PAGE + kk];
                        if (w != 0.f) t[m] += w * val;             // a place that a row does not see adds nothing, whatever it holds
                    }
                }
#pragma unroll
                for (int m = 0; m < AW_ROWS; ++m) o[m][h] = o[m][h] * c_s[m] + t[m];
            }
        }
        __syncthreads();
    }
    cp_async_wait<0>();
    const int group_rows = a.max_new * (a.heads / a.kv_heads);
    const size_t base = ((size_t)blockIdx.y * a.n_splits + split) * group_rows;
    if (threadIdx.x < AW_ROWS && m0 + threadIdx.x < s.rows) {
        a.stats[(base + m0 + threadIdx.x) * 2] = m_s[threadIdx.x];
        a.stats[(base + m0 + threadIdx.x) * 2 + 1] = l_s[threadIdx.x];
    }
    if (a.out) {
#pragma unroll
        for (int m = 0; m < AW_ROWS; ++m) {
            if (m0 + m >= s.rows) break;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int d = threadIdx.x + h * AW_THREADS;
                if (d < a.v_dim) a.acc[(base + m0 + m) * a.v_dim + d] = o[m][h];
            }
        }
    }
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
        if (t != -CUDART_INF_F) sum += expf(t - top) * a.stats[(base + (size_t)i * group_rows) * 2 + 1];
    }
    const float inv = top == -CUDART_INF_F ? 0.f : 1.f / sum;
    if (threadIdx.x == 0) {
        float* j = a.joined + ((size_t)blockIdx.y * group_rows + m) * 2;
        j[0] = top;
        j[1] = inv;
    }
    if (a.out == nullptr) return;
    T* out = (T*)a.out + (long long)(s.row0 + m / group) * a.out_stride + (long long)(kvh * group + m % group) * a.v_dim;
    for (int d = threadIdx.x; d < a.v_dim; d += AW_THREADS) {
        float x = 0.f;
        for (int i = 0; i < splits; ++i) {
            const float t = a.stats[(base + (size_t)i * group_rows) * 2];
            if (t != -CUDART_INF_F) x += expf(t - top) * a.acc[(base + (size_t)i * group_rows) * a.v_dim + d];
        }
        out[d] = from_f32<T>(x * inv);
    }
}

// (3) the weights of a page of keys: grid (pages of the longest sequence, sequences * kv heads)
template <typename T>
__global__ void __launch_bounds__(AW_THREADS) weights_sum_kernel(WeightArgs a) {
    extern __shared__ __align__(16) unsigned char raw[];
    __shared__ float other[CML_PAGE];
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
    const int key = threadIdx.x & 63, half = threadIdx.x >> 6;
    const int group_rows = a.max_new * (a.heads / a.kv_heads);
    float gained = 0.f;
    for (int m0 = 0; m0 < s.rows; m0 += AW_ROWS) {
        __syncthreads();
        load_q<T>(a, s, kvh, m0, q_s);
        cp_async_wait<0>();
        __syncthreads();
        float sc[4];
        score4<T>(a, s, m0, p * CML_PAGE + key, key < valid, raw + key * k_stride, q_s, sc);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const int r = m0 + half * 4 + m;
            if (r >= s.rows || sc[m] == -CUDART_INF_F) continue;
            const float* j = a.joined + ((size_t)blockIdx.y * group_rows + r) * 2;
            gained += expf(sc[m] - j[0]) * j[1];
        }
    }
    if (half == 1) other[key] = gained;
    __syncthreads();
    if (half == 0 && key < valid) {
        const int place = p * CML_PAGE + key;
        a.scores_out[at + key] = (place < s.start ? a.scores[at + key] : 0.f) + (gained + other[key]);
    }
}

template <typename T>
static cudaError_t launch_plain(WeightArgs& a, cudaStream_t s) {
    const unsigned pairs = (unsigned)a.n_seqs * (unsigned)a.kv_heads;
    const int group_rows = a.max_new * (a.heads / a.kv_heads);
    const size_t k_page = (size_t)CML_PAGE * (a.k_dim * sizeof(T) + 16), v_page = a.out ? (size_t)CML_PAGE * a.v_dim * sizeof(T) : 0;
    const size_t rows = (size_t)AW_ROWS * a.k_dim * 4;
    const size_t rest = rows + AW_ROWS * CML_PAGE * 4 + 3 * AW_ROWS * 4, smem3 = k_page + rows;
    a.stages = 2 * (k_page + v_page) + rest <= 227 * 1024 ? 2 : 1;
    const size_t smem1 = a.stages * (k_page + v_page) + rest;
    cudaError_t e = cml_allow_smem<weights_part_kernel<T>>(smem1);
    if (e == cudaSuccess) e = cml_allow_smem<weights_sum_kernel<T>>(smem3);
    if (e != cudaSuccess) return e;
    e = launch_pdl(weights_part_kernel<T>, dim3((unsigned)a.n_splits, pairs, (unsigned)((group_rows + AW_ROWS - 1) / AW_ROWS)), dim3(AW_THREADS),
                   smem1, s, a);
    if (e != cudaSuccess) return e;
    e = launch_pdl(weights_join_kernel<T>, dim3((unsigned)group_rows, pairs), dim3(AW_THREADS), 0, s, a);
    if (e != cudaSuccess) return e;
    return launch_pdl(weights_sum_kernel<T>, dim3((unsigned)((a.max_len + CML_PAGE - 1) / CML_PAGE), pairs), dim3(AW_THREADS), smem3, s, a);
}

extern "C" int cml_attn_paged_weights(const void* q, int dtype, long long q_stride, void* out, long long out_stride, const void* k,
                                      const void* v, const float* scores, float* scores_out, const int* table, int width, int n_pages,
                                      const int* row0, const int* start, const int* fresh, int n_seqs, int n_rows, int heads,
                                      int kv_heads, int k_dim, int v_dim, int max_new, int max_len, float scale, int split_keys,
                                      float* scratch, void* stream) {
    if (dtype != CML_DTYPE_F32 && dtype != CML_DTYPE_BF16) return CML_ERR_BAD_DTYPE;
    if (n_seqs <= 0 || n_rows <= 0) return 0;
    if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || k_dim < 16 || k_dim > 256 || k_dim % 16 || v_dim < 16 || v_dim > 256 || v_dim % 16)
        return CML_ERR_BAD_SIZE;
    if (width <= 0 || n_pages <= 0 || max_new <= 0 || max_len <= 0 || split_keys <= 0 || split_keys % CML_PAGE) return CML_ERR_BAD_SIZE;
    const long long pairs = (long long)n_seqs * kv_heads, rows = (long long)max_new * (heads / kv_heads);
    if (pairs > 65535 || rows > 65535ll * AW_ROWS || max_len > (1 << 28) || width > (1 << 24)) return CML_ERR_BAD_SIZE;
    if (((uintptr_t)k | (uintptr_t)(out ? v : nullptr)) & 15) return CML_ERR_BAD_ALIGN;
    WeightArgs a = {};
    a.q = q; a.q_stride = q_stride; a.out = out; a.out_stride = out_stride; a.k = k; a.v = v; a.scores = scores; a.scores_out = scores_out;
    a.table = table; a.width = width; a.n_pages = n_pages; a.row0 = row0; a.start = start; a.fresh = fresh; a.n_seqs = n_seqs;
    a.n_rows = n_rows; a.heads = heads; a.kv_heads = kv_heads; a.k_dim = k_dim; a.v_dim = v_dim; a.max_new = max_new; a.max_len = max_len;
    a.scale = scale; a.split_keys = split_keys;
    a.n_splits = (max_len + split_keys - 1) / split_keys;
    a.joined = scratch;
    a.stats = a.joined + pairs * rows * 2;
    a.acc = a.stats + pairs * rows * 2 * a.n_splits;
    const cudaError_t e = dtype == CML_DTYPE_F32 ? launch_plain<float>(a, (cudaStream_t)stream) : launch_plain<bf16>(a, (cudaStream_t)stream);
    if (e != cudaSuccess) return (int)e;
    return cml_launch_status();
}
