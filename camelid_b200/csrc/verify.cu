// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Sequence i drafted len[i] tokens x_0 .. and owns the rows row0[i] .. row0[i] + len[i] of the target's logits: row j
// holds the logits of the place where x_j would stand, the last one those of the place behind all of them. With the
// target's distribution p_j = softmax(logits / T) (after the sampler's top_k, min_p and top_p) and the drafter's q_j:
//
//   x_j is accepted while  u_j q_j(x_j) < p_j(x_j)
//   at the first rejection the next token is drawn from max(p_j - q_j, 0) normalised, with all accepted from p_len
//
// which makes every token distributed as the target's own. A drafter without probabilities is certain of its tokens
// (q = 1 there, 0 elsewhere). The draw walks the tokens in ascending order of their ids: the next token is the first at
// which the cumulative weight exceeds draw * total. Temperature 0 is the greedy target: p = 1 at the largest logit,
// the lowest id among equals.
//
// Everything that a decision rests on is computed in double, because a rounding of 2^-24 in a sum over 128,256 tokens
// would move one draw in a hundred to a neighbouring token: exp((l - max) / T), its sums, the thresholds.
//
// Two launches: (1) the maximum and the sum of every row, in parts of 1,024 columns, or, with
// filters, the same of the candidates, by a cluster per row (row_select.cuh); (2) a cluster per sequence decides how
// many tokens stay, adds up the one row that the next token is drawn from, warp by warp, and walks the warp's stretch
// in which the crossing lies.
//
// 64 sequences of 7 drafts over 128,256 tokens (263 MB of logits, 33 MB of the drafter's probabilities): 96 us, of which the sums take 70
// (3.8 TB/s: the double operations of the exponentials, half of that unit's rate, and their chain) and the decisions 32 (two
// steps of loads, the same exponentials over one row, three exchanges). One sequence of 4 drafts: 13.2 us, the two launches' time on the
// host; 4 and 9 us on the device. With a min_p and a top_p, 8 sequences of 4 drafts: 31 us, 18 of them the candidates (two passes over
// a row by three blocks, maximum and listing, the sort and their exchanges); a top_k of 40 33 us, one of 1,000 44.
#include "row_select.cuh"

#define VF_PART 1024            // columns of a row that one warp adds up
#define VF_PART_THREADS 256
#define VF_PART_BLOCKS 3        // a multiprocessor: two (127 registers) are 8% slower over 449 rows, four (64) 3%
#define VF_THREADS 512          // threads of a block that decides
#define VF_WARPS (VF_THREADS / 32)

#define VF_ERR_NONFINITE 1
#define VF_ERR_EMPTY 2
#define VF_ERR_DRAFT 4          // a drafted token outside the vocabulary, or a probability that is none
#define VF_ERR_ROW 8            // a sequence names rows that the logits do not have

// What is known of a part of a row: its maximum (NaN where a logit is not finite) with the lowest place of it, and the
// sum of exp((l - max) / T) over its candidates.
struct PartStat {
    double sum;
    float max;
    int arg;
};

struct VerifyArgs {
    const float* logits;
    long long ld;
    int n_rows, vocab;
    const int* row0;
    const int* lens;
    const int* drafts;
    long long drafts_ld;
    const float* probs;
    long long probs_seq, probs_step;
    const float* accept;
    long long accept_ld;
    const float* draws;
    int n_seqs, width;           // width: drafted tokens a sequence has room for
    float temperature;           // 0: greedy
    double rate;                 // 32 log2(e) / T
    int top_k;
    float top_p, min_p;
    int* counts;
    int* tokens;
    int* err;
    PartStat* stats;             // [rows][parts]
    unsigned long long* floors;  // [rows]: the last candidate's key, 0 without filters
    int parts;
};

// exp((l - max) / T) in double to 2e-12 of itself: 2^(z / 32) with z = (l - max) 32 log2(e) / T cut into a whole number,
// whose upper bits are the exponent and whose lower five choose from a table, and a rest of at most a half, whose power is a
// polynomial of degree four ((ln 2 / 64)^5 / 120 = 1.2e-12). Eleven operations in double instead of the library
// function's eighteen among seventy instructions; 32 entries are two rows of the banks, so a warp's look-up takes two turns.
constexpr float LOWEST = -3.402823466e38f;
struct Exponential {
    double c, max;               // z = (l - max) c; the difference of two floats is exact enough at any temperature
    float least;                 // below this the result is no longer a normal number: zero (never below max - 700 T)
};
// A temperature below 2^-30 of the maximum, a 64th of a float's step there, leaves nothing but the maximum (e^-64 of it at most).
__device__ __forceinline__ bool only_largest(const VerifyArgs& a, float max) { return fabsf(max) * 9.313225746e-10f > a.temperature; }
__device__ __forceinline__ Exponential exponential_of(const VerifyArgs& a, float max) {
    Exponential e;
    e.c = a.rate;
    e.max = (double)max;
    e.least = only_largest(a, max) ? max : fmaxf(__fsub_ru(max, 700.f * a.temperature), LOWEST);
    return e;
}
__device__ __forceinline__ void fill_table(double* table) {       // by the first warp; a barrier follows
    if (threadIdx.x < 32) table[threadIdx.x] = exp2((double)threadIdx.x / 32.0);
}
// `l` at least e.least: what lies below stands for e^-700, which adds nothing to a sum of one or more.
__device__ __forceinline__ double power_of(float l, const Exponential& e, const double* table) {
    const double d = (double)l - e.max;
    const double shifted = fma(d, e.c, 6755399441055744.0);       // 1.5 * 2^52: the whole number in the low bits
    const double r = fma(d, e.c, -(shifted - 6755399441055744.0));
    const int k = __double2loint(shifted);
    constexpr double C1 = 0.021660849392498290, C2 = C1 * C1 / 2, C3 = C1 * C1 * C1 / 6, C4 = C1 * C1 * C1 * C1 / 24;
    const double p = fma(r, fma(r, fma(r, fma(r, C4, C3), C2), C1), 1.0);
    const double t = table[k & 31];
    return __hiloint2double(__double2hiint(t) + ((k << 15) & 0xfff00000), __double2loint(t)) * p;
}
// the same, and exactly zero below
__device__ __forceinline__ double weight_of(float l, const Exponential& e, const double* table) {
    const double w = power_of(fmaxf(l, e.least), e, table);
    return l < e.least ? 0.0 : w;
}

// a call instead of a copy, for kernels whose many loops would not fit the instruction cache with a copy for every element
__device__ __noinline__ double weight_call(float l, Exponential e, const double* table) { return weight_of(l, e, table); }

__device__ __forceinline__ bool finite(float v) { return fabsf(v) < CUDART_INF_F; }

// (1a) without filters. A warp takes a part at a time and keeps its 32 columns a lane in registers, so that the row is read
// once. The part's maximum is the reference of its exponentials; the parts are joined where they are read. No barriers;
// the blocks stay, so the table is made once.
__global__ void __launch_bounds__(VF_PART_THREADS, VF_PART_BLOCKS) verify_stats_kernel(VerifyArgs a) {
    __shared__ double table[32];
    fill_table(table);
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int warps = gridDim.x * (VF_PART_THREADS / 32), items = a.n_rows * a.parts;
    constexpr int U = VF_PART / 32;
    for (int item = blockIdx.x * (VF_PART_THREADS / 32) + (threadIdx.x >> 5); item < items; item += warps) {
        const int row = item / a.parts, begin = (item - row * a.parts) * VF_PART, n = min(VF_PART, a.vocab - begin);
        const float* r = a.logits + (long long)row * a.ld + begin;
        const bool vec = (((uintptr_t)r) & 15) == 0;
        float v[U];
        if (vec) {
#pragma unroll
            for (int g = 0; g < U / 4; ++g) {
                const int i = g * 128 + 4 * lane;
                if (i + 4 <= n) {
                    const float4 t = *reinterpret_cast<const float4*>(r + i);
                    v[4 * g] = t.x, v[4 * g + 1] = t.y, v[4 * g + 2] = t.z, v[4 * g + 3] = t.w;
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[4 * g + k] = i + k < n ? r[i + k] : LOWEST;
                }
            }
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = u * 32 + lane < n ? r[u * 32 + lane] : LOWEST;
        }
        float mx = LOWEST, check = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            mx = fmaxf(mx, v[u]);
            check = fmaf(v[u], 0.f, check);                       // not a number once a logit is not finite
        }
        PartStat st;
        st.max = warp_max(mx);
        st.sum = 0.0;
        st.arg = 0;
        if (a.temperature > 0.f) {
            const Exponential ex = exponential_of(a, st.max);
            double s[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
            for (int u = 0; u < U; ++u) s[u & 3] += power_of(fmaxf(v[u], ex.least), ex, table);
            double t = (s[0] + s[1]) + (s[2] + s[3]);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
            st.sum = t;
        } else {
            int at = 0x7fffffff;                                  // the lowest place of the maximum
#pragma unroll
            for (int u = U - 1; u >= 0; --u)
                if (v[u] == st.max) at = vec ? (u / 4) * 128 + 4 * lane + (u & 3) : u * 32 + lane;
            st.arg = begin + __reduce_min_sync(0xffffffffu, at);
        }
        if (__any_sync(0xffffffffu, check != 0.f)) st.max = CUDART_NAN_F;
        if (lane == 0) a.stats[item] = st;
    }
}

// (1b) with filters: a cluster per row finds the last candidate's key, and the sum over the candidates. The order and
// the stages are the sampler's: the k first, then p >= min_p * p_max, then the shortest prefix whose cumulative
// probability reaches top_p.
__global__ void __launch_bounds__(SAMPLE_THREADS, 1) verify_floor_kernel(VerifyArgs a) {
    extern __shared__ __align__(16) unsigned char raw[];
    FastSharedOf<double>& fs = *reinterpret_cast<FastSharedOf<double>*>(raw);
    __shared__ SelectShared sh;
    __shared__ TeamSlots ts;
    __shared__ float fred[33];
    __shared__ unsigned int counts_s[32];
    __shared__ double table[32];
    fill_table(table);
    if (threadIdx.x == 0) fs.n_list = 0u;
    cg::this_cluster().sync();                                    // every block has started before its memory is written
    pdl_wait();
    pdl_launch_dependents();
    Team tm;
    tm.n = (int)cg::this_cluster().num_blocks();
    tm.rank = (int)cg::this_cluster().block_rank();
    const int row_index = blockIdx.x / tm.n;
    const int vocab = a.vocab;
    {
        const int per = (((vocab + tm.n - 1) / tm.n) + 3) & ~3;
        tm.begin = min(vocab, tm.rank * per);
        tm.end = min(vocab, tm.begin + per);
    }
    TeamSlots* ts0 = tm.at0(&ts);
    FastSharedOf<double>* fs0 = tm.at0(&fs);
    const float* row = a.logits + (long long)row_index * a.ld;
    float mx = -CUDART_INF_F, mn = CUDART_INF_F;
    bool bad = false;
    for_each_in_slice<8>(row, tm, [&](float v, int) {
        if (!finite(v)) bad = true;
        mx = fmaxf(mx, v);
        mn = fminf(mn, v);
    });
    {
        const float bmx = block_max(mx, fred), bmn = -block_max(-mn, fred);
        const int any_bad = __syncthreads_or(bad ? 1 : 0);
        if (threadIdx.x == 0) ts0->f[0][tm.rank] = bmx, ts0->f[1][tm.rank] = bmn, ts0->u[1][tm.rank] = any_bad ? 1u : 0u;
    }
    tm.sync();
    mx = -CUDART_INF_F, mn = CUDART_INF_F;
    unsigned int team_bad = 0u;
    for (int r = 0; r < tm.n; ++r) {
        mx = fmaxf(mx, ts0->f[0][r]);
        mn = fminf(mn, ts0->f[1][r]);
        team_bad |= ts0->u[1][r];
    }
    const bool writer = tm.rank == 0 && threadIdx.x == 0;
    PartStat st;
    st.sum = 0.0;
    st.max = CUDART_NAN_F;
    st.arg = 0;
    if (team_bad != 0u) {
        if (writer) a.stats[row_index] = st, a.floors[row_index] = 0ull;
        tm.sync();
        return;
    }
    const Exponential ex = exponential_of(a, mx);
    // the place of a value in the order: never negative, monotone, and finite (masks of the type's lowest value are
    // all put at one far place, where their weight is zero)
    const float inv_t = fminf(1.0f / a.temperature, 1e30f), far = 1e30f;
    auto xof = [=](float v) { return fminf((mx - v) * inv_t, far); };
    const float x_max = xof(mn);
    const double* const powers = table;
    auto raw_weight = [=](float v, int) { return weight_call(v, ex, powers); };
    unsigned long long floor_key = 0ull, key;
    double cum;
    auto select_slow = [&](unsigned long long floor, double target, int strict, auto weight) {
        if (tm.rank == 0) {
            unsigned long long k;
            double c;
            select_by_mass(row, vocab, floor, target, strict, weight, &sh, &k, &c);
            if (threadIdx.x == 0) fs.key = k, fs.cum = c;
        }
        tm.sync();
        key = fs0->key;
        cum = fs0->cum;
        tm.sync();
    };
    float edge = CUDART_INF_F;                                    // nothing at or beyond this place is among the first top_k
    const bool first_k = a.top_k > 0 && a.top_k < vocab;
    // The first top_k by counting: the bin of 1/64 in which they end; where no more than the list holds lies up to there, the list takes
    // it all and the first k of it stay (one sequence of 4 drafts over 128,256 tokens, top_k 40: 29 us, for 51 by a selection before
    // the list).
    if (first_k && a.top_k <= FS_CAP) {
        for (int b = threadIdx.x; b < FS_BINS; b += SAMPLE_THREADS) fs.cnt[b] = 0u;
        tm.sync();                                                // block 0's bins are clear before anyone adds to them
        for_each_in_slice<8>(row, tm, [&](float v, int) {
            const float x = xof(v);
            if (x < (float)(FS_BINS / 64)) atomicAdd(&fs.cnt[(int)(x * 64.f)], 1u);
        });
        __syncthreads();
        if (tm.rank != 0) {
            for (int b = threadIdx.x; b < FS_BINS; b += SAMPLE_THREADS)
                if (fs.cnt[b] != 0u) atomicAdd(&fs0->cnt[b], fs.cnt[b]);
        }
        tm.sync();
        if (tm.rank == 0) {
            const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
            for (int w = warp; w < 32; w += SAMPLE_THREADS / 32) {            // 64 bins a warp's turn
                const unsigned int t = __reduce_add_sync(0xffffffffu, fs.cnt[w * 64 + lane] + fs.cnt[w * 64 + 32 + lane]);
                if (lane == 0) counts_s[w] = t;
            }
            __syncthreads();
            if (warp == 0) {
                auto scan = [&](unsigned int c) {
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const unsigned int t = __shfl_up_sync(0xffffffffu, c, o);
                        if (lane >= o) c += t;
                    }
                    return c;
                };
                const unsigned int k = (unsigned int)a.top_k, incl = scan(counts_s[lane]);
                const unsigned int reach = __ballot_sync(0xffffffffu, incl >= k);
                int bin = FS_BINS;
                unsigned int upto = 0u;
                if (reach) {
                    const int w = __ffs(reach) - 1;
                    const unsigned int before = __shfl_sync(0xffffffffu, incl - counts_s[lane], w);
                    const unsigned int c0 = fs.cnt[w * 64 + 2 * lane], c1 = fs.cnt[w * 64 + 2 * lane + 1], pair = before + scan(c0 + c1);
                    const int l = __ffs(__ballot_sync(0xffffffffu, pair >= k)) - 1;
                    const bool second = pair - c1 < k;            // in this lane's pair: the first of the two that reaches k
                    bin = __shfl_sync(0xffffffffu, w * 64 + 2 * lane + (second ? 1 : 0), l);
                    upto = __shfl_sync(0xffffffffu, second ? pair : pair - c1, l);
                }
                if (lane == 0) fs.bin = bin, fs.status = (int)upto;
            }
        }
        tm.sync();
        if (fs0->bin < FS_BINS && fs0->status <= FS_CAP) edge = (float)(fs0->bin + 1) / 64.f;
    }
    const bool counted = edge < CUDART_INF_F;
    if (first_k && !counted) {
        auto one = [](float, int) { return 1.0; };
        auto one_at = [](float) { return 1.0f; };
        tm.sync();                                                // (every block has read block 0's verdict)
        if (!select_fast(row, tm, 0ull, (double)a.top_k, 0, xof, x_max, one, one_at, &fs, &ts, &key, &cum))
            select_slow(0ull, (double)a.top_k, 0, one);
        floor_key = key;
    }
    // min_p: the weight of the maximum is one, so a candidate's own weight is compared
    const double least = (double)a.min_p;
    // (only places near enough are weighed: past -ln(min_p), with room for its rounding, nothing stays)
    const float near = least > 0.0 ? -logf(a.min_p) * 1.001f + 0.01f : CUDART_INF_F;
    // Few candidates, the usual case where there is a min_p or a top_k: their keys are collected in one pass, sorted by block 0, and
    // the rest of the way goes along that list.
    if (floor_key != 0ull || counted || least > 0.0) {
        if (first_k && !counted) {                                // the selection left its own list there
            if (writer) fs.n_list = 0u;
            tm.sync();
        }
        // Sixteen columns a thread are compared, and the few that are near enough looked at one by one.
        auto consider = [&](int i) {
            const float v = row[i];
            const unsigned long long ck = composite_key(v, i);
            if (ck < floor_key || (least > 0.0 && raw_weight(v, i) < least)) return;
            const unsigned int slot = atomicAdd(&fs0->n_list, 1u);
            if (slot < FS_CAP) fs0->list[slot] = ck;
        };
        auto close = [&](float v) {
            const float x = xof(v);
            return x <= near && x < edge;
        };
        const bool vec = (((uintptr_t)row) & 15) == 0;
        const int whole = vec ? tm.end & ~3 : tm.end;             // up to here in whole groups of four
        for (int g0 = tm.begin + (vec ? 4 : 1) * (int)threadIdx.x; g0 < whole; g0 += 16 * SAMPLE_THREADS) {
            unsigned int some = 0u;
            if (vec) {
                float4 t[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) t[u] = *reinterpret_cast<const float4*>(row + min(g0 + u * 4 * SAMPLE_THREADS, whole - 4));
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    some |= (close(t[u].x) ? 1u : 0u) << (4 * u);
                    some |= (close(t[u].y) ? 2u : 0u) << (4 * u);
                    some |= (close(t[u].z) ? 4u : 0u) << (4 * u);
                    some |= (close(t[u].w) ? 8u : 0u) << (4 * u);
                }
            } else {
#pragma unroll
                for (int u = 0; u < 16; ++u) some |= (close(row[min(g0 + u * SAMPLE_THREADS, whole - 1)]) ? 1u : 0u) << u;
            }
            while (some) {
                const int u = __ffs(some) - 1;
                some &= some - 1u;
                const int i = vec ? g0 + (u >> 2) * 4 * SAMPLE_THREADS + (u & 3) : g0 + u * SAMPLE_THREADS;
                if (i < whole) consider(i);
            }
        }
        if ((int)threadIdx.x < tm.end - whole && close(row[whole + threadIdx.x])) consider(whole + threadIdx.x);
        tm.sync();
        const unsigned int n = fs0->n_list;
        if (n <= FS_CAP) {                                        // the same in every block
            if (tm.rank == 0) {
                unsigned int m = 1u;
                while (m < n) m <<= 1;
                for (unsigned int i = n + threadIdx.x; i < m; i += blockDim.x) fs.list[i] = 0ull;
                __syncthreads();
                for (unsigned int k = 2; k <= m; k <<= 1) {
                    for (unsigned int j = k >> 1; j > 0; j >>= 1) {
                        for (unsigned int i = threadIdx.x; i < m; i += blockDim.x) {
                            const unsigned int l = i ^ j;
                            if (l > i) {
                                const unsigned long long x = fs.list[i], y = fs.list[l];
                                if ((i & k) == 0 ? x < y : x > y) { fs.list[i] = y; fs.list[l] = x; }
                            }
                        }
                        __syncthreads();
                    }
                }
                const unsigned int n_k = counted ? min(n, (unsigned int)a.top_k) : n;
                for (unsigned int i = threadIdx.x; i < n_k; i += blockDim.x) fs.lp[i] = raw_weight(value_of_key(fs.list[i]), 0);
                __syncthreads();
                if (threadIdx.x < 32) {                           // one warp adds up, a run of candidates a lane, in their order
                    const int lane = threadIdx.x;
                    const unsigned int run = ((n_k + 31) / 32) | 1u;          // (odd: no two lanes' runs meet a bank together)
                    const unsigned int from = min(n_k, lane * run), to = min(n_k, from + run);
                    double own = 0.0;
                    for (unsigned int i = from; i < to; ++i) own += fs.lp[i];
                    double incl = own;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const double t = __shfl_up_sync(0xffffffffu, incl, o);
                        if (lane >= o) incl += t;
                    }
                    const double sum = __shfl_sync(0xffffffffu, incl, 31);
                    unsigned int stay = n_k;                      // candidates that stay: up to the first that reaches top_p
                    double total = sum;
                    if (a.top_p < 1.f) {
                        const double target = (double)a.top_p * sum;
                        const unsigned int hit = __ballot_sync(0xffffffffu, to > from && incl >= target);
                        if (hit) {
                            const int who = __ffs(hit) - 1;
                            double c = incl - own;
                            unsigned int i = from;
                            if (lane == who)
                                for (; i < to; ++i) {
                                    c += fs.lp[i];
                                    if (c >= target || i + 1 == to) { ++i; break; }       // (the last where rounding leaves it short)
                                }
                            stay = __shfl_sync(0xffffffffu, i, who);
                            total = __shfl_sync(0xffffffffu, c, who);
                        }
                    }
                    if (lane == 0) {
                        st.sum = total;
                        st.max = mx;
                        a.stats[row_index] = st;
                        a.floors[row_index] = fs.list[stay - 1];
                    }
                }
            }
            tm.sync();                                            // block 0's memory stays until every block has read it
            return;
        }
    }
    double part = 0.0;
    unsigned long long kmin = ~0ull;
    for_each_in_slice(row, tm, [&](float v, int i) {
        if (xof(v) > near) return;
        const unsigned long long ck = composite_key(v, i);
        if (ck < floor_key) return;
        const double w = raw_weight(v, i);
        if (w >= least) { part += w; kmin = ck < kmin ? ck : kmin; }
    });
    part = block_sum_double(part, fs.dred);
    {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long ok = __shfl_xor_sync(0xffffffffu, kmin, o);
            kmin = ok < kmin ? ok : kmin;
        }
        __syncthreads();
        if (lane == 0) fs.list[warp] = kmin;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < nw; ++w) kmin = fs.list[w] < kmin ? fs.list[w] : kmin;
            ts0->d[3][tm.rank] = part;
            ts0->k[0][tm.rank] = kmin;
        }
    }
    tm.sync();
    double total = 0.0;
    unsigned long long k_all = ~0ull;
    for (int r = 0; r < tm.n; ++r) {
        total += ts0->d[3][r];
        k_all = ts0->k[0][r] < k_all ? ts0->k[0][r] : k_all;
    }
    if (a.min_p > 0.f && k_all != ~0ull) floor_key = k_all;
    if (a.top_p < 1.f) {
        auto a1 = [=](float x) { return __expf(-x); };
        const double target = (double)a.top_p * total;
        if (!select_fast(row, tm, floor_key, target, 0, xof, x_max, raw_weight, a1, &fs, &ts, &key, &cum))
            select_slow(floor_key, target, 0, raw_weight);
        floor_key = key;
        total = cum;
    }
    if (writer) {
        st.sum = total;
        st.max = mx;
        a.stats[row_index] = st;
        a.floors[row_index] = floor_key;
    }
    tm.sync();                       // block 0's shared memory stays until every block has read it
}

struct RowStat {
    double total;                    // the sum against the maximum
    float max;
    int arg;
    int bad;
};

// The parts of a row joined by a warp, the lanes in their order: the same in every lane. The first 128 are asked for by
// themselves, so that they come beside what else a decision reads.
#define VF_AHEAD 4
struct Parts {
    PartStat s[VF_AHEAD];
};
__device__ __forceinline__ Parts load_parts(const VerifyArgs& a, int row) {
    const PartStat* s = a.stats + (size_t)row * a.parts + (threadIdx.x & 31);
    Parts r;
#pragma unroll
    for (int u = 0; u < VF_AHEAD; ++u)
        if ((int)(threadIdx.x & 31) + 32 * u < a.parts) r.s[u] = s[32 * u];
        else r.s[u] = {0.0, LOWEST, 0x7fffffff};                  // (no part: what is at the type's lowest anyway adds nothing of its own)
    return r;
}
__device__ __forceinline__ RowStat join_parts(const VerifyArgs& a, int row, const Parts& first, const double* table) {
    const int lane = threadIdx.x & 31;
    const PartStat* s = a.stats + (size_t)row * a.parts;
    RowStat r;
    float mx = -CUDART_INF_F;
    int arg = 0x7fffffff;
    bool bad = false;
#pragma unroll
    for (int u = 0; u < VF_AHEAD; ++u) {
        if (!finite(first.s[u].max)) bad = true;
        if (first.s[u].max > mx) mx = first.s[u].max, arg = first.s[u].arg;
    }
    for (int p = lane + 32 * VF_AHEAD; p < a.parts; p += 32) {
        const float m = s[p].max;
        if (!finite(m)) bad = true;
        if (m > mx) mx = m, arg = s[p].arg;
    }
    r.max = warp_max(mx);
    r.arg = __reduce_min_sync(0xffffffffu, mx == r.max ? arg : 0x7fffffff);
    r.bad = __any_sync(0xffffffffu, bad) ? 1 : 0;
    r.total = 0.0;
    if (a.temperature > 0.f && !r.bad) {
        const Exponential ex = exponential_of(a, r.max);
        if (a.floors == nullptr && only_largest(a, r.max)) {      // the parts' sums counted what lies just below as well
            const float* l = a.logits + (long long)row * a.ld;
            for (int i = lane; i < a.vocab; i += 32) r.total += l[i] == r.max ? 1.0 : 0.0;
        } else {
#pragma unroll
            for (int u = 0; u < VF_AHEAD; ++u) r.total += first.s[u].sum * weight_of(first.s[u].max, ex, table);
            for (int p = lane + 32 * VF_AHEAD; p < a.parts; p += 32) r.total += s[p].sum * weight_of(s[p].max, ex, table);
            // LOWEST behind the row's end counts where the temperature is huge
            if (lane == 31 && a.floors == nullptr) r.total -= (a.parts * VF_PART - a.vocab) * weight_of(LOWEST, ex, table);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) r.total += __shfl_xor_sync(0xffffffffu, r.total, o);
    }
    return r;
}

// (2) a cluster per sequence.
#define VF_ROWS 32                   // rows whose joined parts a block remembers
#define VF_TEAM 16                   // blocks of a cluster at most
// PER_SM: blocks that share a multiprocessor; one alone has the registers to ask for the next tiles ahead (8 sequences 18.9 us for
// 23.4; 64 sequences of 7 drafts would take 127 us in several rounds, and take 96).
// GROUPS: a warp's stretch is cut into as many, whose sums stay in registers.
template <int PER_SM, int GROUPS>
__global__ void __launch_bounds__(VF_THREADS, PER_SM) verify_decide_kernel(VerifyArgs a) {
    __shared__ double table[32];
    __shared__ double warp_sums[2][VF_WARPS], block_sums[2][VF_TEAM];     // of two rounds
    __shared__ RowStat stats[VF_ROWS];
    __shared__ int first_bad, row_bad, err_bits;
    fill_table(table);
    if (threadIdx.x == 0) first_bad = 0x7fffffff, row_bad = 0, err_bits = 0;
    pdl_wait();
    const int team = (int)cg::this_cluster().num_blocks(), rank = (int)cg::this_cluster().block_rank();
    const int seq = blockIdx.x / team;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int len = max(0, min(a.lens[seq], a.width)), row0 = a.row0[seq];
    const int vocab = a.vocab;
    const bool greedy = !(a.temperature > 0.f), filtered = a.floors != nullptr;
    int* out = a.tokens + (size_t)seq * (a.width + 1);
    if (row0 < 0 || row0 > a.n_rows - 1 - len) {                  // the same in every block of the cluster
        if (rank == 0) {
            if (threadIdx.x == 0) atomicOr(a.err, VF_ERR_ROW), a.counts[seq] = 0;
            for (int j = threadIdx.x; j <= a.width; j += blockDim.x) out[j] = -1;
        }
        return;
    }
    __syncthreads();
    // the cluster's other blocks have started once all have arrived here: their memory is written only after the wait below
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    // every draft by a warp of its own: is it accepted?
    for (int j = warp; j <= len; j += VF_WARPS) {
        const Parts parts = load_parts(a, row0 + j);              // what the decision reads beside them does not wait for them
        int x = 0;
        float q = 1.f, l = 0.f, u = 0.f;
        bool known = false;
        if (j < len) {
            x = a.drafts[(long long)seq * a.drafts_ld + j];
            u = a.accept[(long long)seq * a.accept_ld + j];
            known = x >= 0 && x < vocab;
            if (known) {
                if (a.probs) q = a.probs[(long long)seq * a.probs_seq + (long long)j * a.probs_step + x];
                l = a.logits[(long long)(row0 + j) * a.ld + x];
            }
        }
        const RowStat r = join_parts(a, row0 + j, parts, table);
        if (lane == 0) {
            if (j < VF_ROWS) stats[j] = r;
            int bits = r.bad ? VF_ERR_NONFINITE : (!greedy && !(r.total > 0.0) ? VF_ERR_EMPTY : 0);
            if (bits) atomicOr(&row_bad, 1);
            if (j < len) {
                bool ok = false;
                if (!known) bits |= VF_ERR_DRAFT;
                else if (!r.bad) {
                    if (!(q >= 0.f) || !finite(q)) bits |= VF_ERR_DRAFT;
                    double p;
                    if (greedy) p = x == r.arg ? 1.0 : 0.0;
                    else {
                        const bool in = !filtered || composite_key(l, x) >= a.floors[row0 + j];
                        p = in ? weight_of(l, exponential_of(a, r.max), table) / r.total : 0.0;
                    }
                    ok = (double)u * (double)q < p;
                }
                if (!ok) atomicMin(&first_bad, j);
            }
            if (bits) atomicOr(&err_bits, bits);
        }
    }
    __syncthreads();
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    const int count = row_bad ? 0 : min(first_bad, len);
    const int row = row0 + count;
    const RowStat st = count < VF_ROWS ? stats[count] : join_parts(a, row, load_parts(a, row), table);
    if (rank == 0) {
        if (threadIdx.x == 0) {
            a.counts[seq] = count;
            if (err_bits) atomicOr(a.err, err_bits);
        }
        for (int j = threadIdx.x; j <= a.width; j += blockDim.x)
            if (j != count) out[j] = j < count ? a.drafts[(long long)seq * a.drafts_ld + j] : -1;
    }
    if (row_bad || greedy) {                                      // the same in every block
        if (rank == 0 && threadIdx.x == 0) out[count] = row_bad ? 0 : st.arg;
        return;
    }
    // the weight of the next token: the target's probability, less the drafter's where a draft was rejected
    const float* r = a.logits + (long long)row * a.ld;
    const bool rejected = count < len;
    const float* q = (rejected && a.probs) ? a.probs + (long long)seq * a.probs_seq + (long long)count * a.probs_step : nullptr;
    const int without = (rejected && !a.probs) ? a.drafts[(long long)seq * a.drafts_ld + count] : -1;
    const unsigned long long floor_key = filtered ? a.floors[row] : 0ull;
    const Exponential ex = exponential_of(a, st.max);
    const double inv_total = 1.0 / st.total;
    bool bad_q = false;
    bool plain = false;                                           // nothing is left of p - q: draw from p
    // stretches of GROUPS groups of whole tiles of 128 columns, a stretch a warp, in ascending order over the cluster's blocks
    const int warps = team * VF_WARPS;
    const int group = (vocab + warps * GROUPS * 128 - 1) / (warps * GROUPS * 128) * 128, per = group * GROUPS;
    const long long first = (long long)(rank * VF_WARPS + warp) * per;
    const int begin = (int)min((long long)vocab, first), end = (int)min((long long)vocab, first + per);
    const bool vec = (((uintptr_t)r) & 15) == 0 && (q == nullptr || (((uintptr_t)q) & 15) == 0);
    // four columns of a tile in a lane, ascending over the lanes
    auto load4 = [&](const float* from, int i, float (&v)[4]) {
        if (vec && i + 4 <= end) {
            const float4 t = *reinterpret_cast<const float4*>(from + i);
            v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = i + k < end ? from[i + k] : 0.f;
        }
    };
    auto weigh = [&](int i, const float (&l)[4], const float (&qi)[4], double (&w)[4]) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            double p = weight_of(l[k], ex, table) * inv_total;
            if (filtered && composite_key(l[k], i + k) < floor_key) p = 0.0;
            if (!plain) {
                if (q) {
                    bad_q = bad_q || !(qi[k] >= 0.f) || !finite(qi[k]);
                    p -= (double)qi[k];
                }
                if (i + k == without) p = 0.0;
            }
            w[k] = i + k < end && p > 0.0 ? p : 0.0;
        }
    };
    double total = 0.0, target, before = 0.0;
    double groups[GROUPS];                                     // this lane's share of every group's sum
    int owner = -1, round = 0;
    for (; round < 2; ++round) {
        double s = 0.0;
        constexpr bool AHEAD = PER_SM == 1;                       // two groups' tiles at a time; the next two on their way where registers allow
        float l0[4], l1[4], q0[4] = {0.f, 0.f, 0.f, 0.f}, q1[4] = {0.f, 0.f, 0.f, 0.f};
        auto load_two = [&](int i0, float (&l0)[4], float (&l1)[4], float (&q0)[4], float (&q1)[4]) {       // (behind the row: nothing)
            load4(r, i0, l0);
            load4(r, i0 + group, l1);
            if (q) load4(q, i0, q0), load4(q, i0 + group, q1);
        };
        if (AHEAD) load_two(begin + 4 * lane, l0, l1, q0, q1);
#pragma unroll
        for (int g = 0; g < GROUPS; g += 2) {
            double s0 = 0.0, s1 = 0.0;
            for (int i = 0; i < group; i += 128) {
                const int i0 = begin + g * group + i + 4 * lane;
                float nl0[4], nl1[4], nq0[4] = {0.f, 0.f, 0.f, 0.f}, nq1[4] = {0.f, 0.f, 0.f, 0.f};
                if (AHEAD) load_two(i + 128 < group ? i0 + 128 : begin + (g + 2) * group + 4 * lane, nl0, nl1, nq0, nq1);
                else load_two(i0, l0, l1, q0, q1);
                double w[4];
                weigh(i0, l0, q0, w);
                s0 += (w[0] + w[1]) + (w[2] + w[3]);
                weigh(i0 + group, l1, q1, w);
                s1 += (w[0] + w[1]) + (w[2] + w[3]);
                if (AHEAD) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) l0[k] = nl0[k], l1[k] = nl1[k], q0[k] = nq0[k], q1[k] = nq1[k];
                }
            }
            groups[g] = s0, groups[g + 1] = s1;
            s += s0 + s1;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) warp_sums[round][warp] = s;
        __syncthreads();
        if ((int)threadIdx.x < team) {                            // this block's sum to every block of the cluster
            double b = 0.0;
#pragma unroll
            for (int w = 0; w < VF_WARPS; ++w) b += warp_sums[round][w];
            cg::this_cluster().map_shared_rank(&block_sums[round][0], threadIdx.x)[rank] = b;
        }
        cg::this_cluster().sync();                                // the last access to another block's memory of this round
        total = 0.0;
        for (int b = 0; b < team; ++b) total += block_sums[round][b];
        if (total > 0.0 || round == 1) break;
        plain = true;
    }
    target = (double)a.draws[seq] * total;
    {
        double run = 0.0;
        for (int b = 0; b < team; ++b) {
            const double s = block_sums[round][b];
            if (s > 0.0) owner = b, before = run;                 // never reached: the last stretch with any weight
            run += s;
            if (run > target) break;
        }
    }
    if (owner == rank) {
        int mine = -1;
        double run = before;
        for (int w = 0; w < VF_WARPS; ++w) {
            const double s = warp_sums[round][w];
            if (s > 0.0) mine = w, before = run;
            run += s;
            if (run > target) break;
        }
        if (warp == mine) {
            // the group of the crossing from the sums in registers, then its columns
            int in = -1;
            run = before;
            // (the groups' sums over the lanes: every exchange halves what a lane holds, 32 / GROUPS lanes have one group's in the end)
#pragma unroll
            for (int o = 16, n = GROUPS / 2; n > 0; o >>= 1, n >>= 1) {
                const bool high = (lane & o) != 0;
#pragma unroll
                for (int g = 0; g < GROUPS / 2; ++g) {
                    if (g >= n) break;
                    const double away = high ? groups[g] : groups[g + n], here = high ? groups[g + n] : groups[g];
                    groups[g] = here + __shfl_xor_sync(0xffffffffu, away, o);
                }
            }
#pragma unroll
            for (int o = 16 / GROUPS; o > 0; o >>= 1) groups[0] += __shfl_xor_sync(0xffffffffu, groups[0], o);
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                const double s = __shfl_sync(0xffffffffu, groups[0], g * (32 / GROUPS));
                if (s > 0.0 && (in < 0 || !(run > target))) in = g, before = run;
                run += s;
            }
            run = before;
            int found = -1, last = -1;
            const int g_begin = begin + in * group, g_end = min(end, g_begin + group);
            for (int i0 = g_begin; i0 < g_end; i0 += 128) {
                const int i = i0 + 4 * lane;
                float l[4], qi[4] = {0.f, 0.f, 0.f, 0.f};
                double w[4];
                load4(r, i, l);
                if (q) load4(q, i, qi);
                weigh(i, l, qi, w);
                const double s = (w[0] + w[1]) + (w[2] + w[3]);
                double incl = s;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double t = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += t;
                }
                const unsigned int some = __ballot_sync(0xffffffffu, s > 0.0);
                const unsigned int hit = __ballot_sync(0xffffffffu, s > 0.0 && run + incl > target);
                if (some) {                                       // the lane of the crossing, or the last with any weight
                    const int who = hit ? __ffs(hit) - 1 : 31 - __clz(some);
                    double c = run + (incl - s);
                    int at = -1;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        c += w[k];
                        if (w[k] > 0.0) at = i + k;
                        if (hit && w[k] > 0.0 && c > target) break;
                    }
                    last = __shfl_sync(0xffffffffu, at, who);
                    if (hit) { found = last; break; }
                }
                run += __shfl_sync(0xffffffffu, incl, 31);
            }
            if (lane == 0) out[count] = found >= 0 ? found : last;
        }
    } else if (owner < 0 && rank == 0 && threadIdx.x == 0) {      // not a number in the sums
        out[count] = st.arg;
        atomicOr(a.err, VF_ERR_EMPTY);
    }
    if (bad_q) atomicOr(a.err, VF_ERR_DRAFT);
}

static int verify_parts(int vocab) { return (vocab + VF_PART - 1) / VF_PART; }

template <typename K>
static cudaError_t launch_cluster(K kernel, int blocks, int threads, size_t smem, int team, cudaStream_t stream, VerifyArgs a) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
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

// `scratch`: 16 bytes a row and part of 1,024 columns, then 8 bytes a row (16-byte aligned).
extern "C" int cml_verify_drafts(const float* logits, long long ld, int n_rows, int vocab, const int* row0, const int* lens,
                                 const int* drafts, long long drafts_ld, const float* probs, long long probs_seq,
                                 long long probs_step, const float* accept, long long accept_ld, const float* draws, int n_seqs,
                                 int width, float temperature, int top_k, float top_p, float min_p, int* counts, int* tokens,
                                 int* err, void* scratch, void* stream) {
    if (n_seqs <= 0) return 0;
    if (vocab <= 0 || vocab > (1 << 30) || n_rows < 0 || width < 0 || width > 65535 || !(temperature >= 0.f) ||
        !(temperature < __builtin_inff()))
        return CML_ERR_BAD_SIZE;
    if (((uintptr_t)scratch) & 15) return CML_ERR_BAD_ALIGN;
    const bool filters = temperature > 0.f && ((top_k > 0 && top_k < vocab) || top_p < 1.f || min_p > 0.f);
    VerifyArgs a = {};
    a.logits = logits; a.ld = ld; a.n_rows = n_rows; a.vocab = vocab; a.row0 = row0; a.lens = lens;
    a.drafts = drafts; a.drafts_ld = drafts_ld; a.probs = probs; a.probs_seq = probs_seq; a.probs_step = probs_step;
    a.accept = accept; a.accept_ld = accept_ld; a.draws = draws; a.n_seqs = n_seqs; a.width = width;
    a.temperature = temperature; a.rate = 46.166241308446828 / (double)temperature; a.top_k = top_k; a.top_p = top_p; a.min_p = min_p;
    a.counts = counts; a.tokens = tokens; a.err = err;
    a.stats = (PartStat*)scratch;
    a.parts = filters ? 1 : verify_parts(vocab);
    if ((long long)n_rows * (a.parts > 8 ? a.parts : 8) > 0x3fffffffLL || (long long)n_seqs * 8 > 0x7fffffffLL) return CML_ERR_BAD_SIZE;
    cudaStream_t s = (cudaStream_t)stream;
    int team = vocab >= 32768 ? 8 : (vocab >= 8192 ? 4 : 1);
    if (n_rows > 0) {
        cudaError_t e;
        if (filters) {
            // a block takes a multiprocessor to itself: as many share a row as all rows leave room for
            const int share = max(1, min(team, cml_sm_count() / n_rows));
            a.floors = (unsigned long long*)((char*)scratch + 16ll * n_rows * verify_parts(vocab));
            e = cml_allow_smem<verify_floor_kernel>(sizeof(FastSharedOf<double>));
            if (e != cudaSuccess) return (int)e;
            e = launch_cluster(verify_floor_kernel, n_rows * share, SAMPLE_THREADS, sizeof(FastSharedOf<double>), share, s, a);
        } else {
            const long long blocks = ((long long)n_rows * a.parts + VF_PART_THREADS / 32 - 1) / (VF_PART_THREADS / 32);
            const long long most = (long long)VF_PART_BLOCKS * cml_sm_count();
            e = launch_pdl(verify_stats_kernel, dim3((unsigned)(blocks < most ? blocks : most)), dim3(VF_PART_THREADS), 0, s, a);
        }
        if (e != cudaSuccess) return (int)e;
    }
    while (team > 1 && n_seqs * team > 2 * cml_sm_count()) team /= 2;          // one round of blocks, two a multiprocessor (64 sequences: 98 us for 104)
    // Where all clusters find room at the same time, a multiprocessor for every block (of clusters of eight 15 do: 15 sequences of
    // 128,256 tokens 24.6 us for 30.1, 16 would take 34.1 for 31.2).
    const bool alone = n_seqs * team <= (team < 8 ? cml_sm_count() : cml_sm_count() * 5 / 6);
    cudaError_t e;
    if (vocab >= 65536 && n_seqs <= 4) {
        // few sequences: sixteen blocks each (one of 128,256 tokens 9.4 us for 11.8)
        e = cml_allow_wide_clusters<verify_decide_kernel<1, 4>>();
        if (e == cudaSuccess) e = launch_cluster(verify_decide_kernel<1, 4>, n_seqs * VF_TEAM, VF_THREADS, 0, VF_TEAM, s, a);
    } else if (alone && vocab <= team * VF_WARPS * 512) {         // four groups are enough (50,257 tokens: 9.5 us for 12.2 with eight)
        e = launch_cluster(verify_decide_kernel<1, 4>, n_seqs * team, VF_THREADS, 0, team, s, a);
    } else if (alone) {
        e = launch_cluster(verify_decide_kernel<1, 8>, n_seqs * team, VF_THREADS, 0, team, s, a);
    } else {
        e = launch_cluster(verify_decide_kernel<2, 8>, n_seqs * team, VF_THREADS, 0, team, s, a);
    }
    if (e != cudaSuccess) return (int)e;
    return cml_launch_status();
}
