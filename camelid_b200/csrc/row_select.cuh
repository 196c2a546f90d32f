// Selections along a row of logits in the total order (logit descending, then index ascending), by a thread-block
// cluster per row: shared by the sampler and by the verification of drafted tokens. `W` is the type in which a
// candidate's weight is computed and listed; sums are double in both.
#pragma once
#include "common.cuh"
#include <cooperative_groups.h>
#include <math_constants.h>
namespace cg = cooperative_groups;

#define SAMPLE_THREADS 1024
#define SAMPLE_MAX_TEAM 8      // blocks that may share a row (a portable cluster)
#define SAMPLE_LIST_WALK 512    // a top_k up to this is finished along its sorted list by one thread
#define SAMPLE_ERR_NONFINITE 1
#define SAMPLE_ERR_EMPTY 2

__device__ __forceinline__ unsigned int orderable_bits(float v) {
    const unsigned int u = __float_as_uint(v);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);       // larger float -> larger unsigned
}
__device__ __forceinline__ unsigned long long composite_key(float v, int idx) {
    return ((unsigned long long)orderable_bits(v) << 32) | (unsigned long long)(0xFFFFFFFFu - (unsigned int)idx);
}

// ------------------------------------------------------------------------------------
// Selection in the total order (key descending). The weight of element i is given by the
// functor; elements with key < floor_key are not candidates. Finds the first candidate at
// which the inclusive cumulative weight reaches (`strict` 0: >=, 1: >) the target, and
// returns its key and that inclusive sum. If the total never reaches the target the last
// candidate (floor) is returned with the total.
struct SelectShared {
    double mass[256];
    unsigned int count[256];
    unsigned long long prefix;
    double before;
    int chosen;
    int found;
};

template <typename WeightFn>
__device__ void select_by_mass(const float* row, int vocab, unsigned long long floor_key, double target, int strict,
                               WeightFn weight, SelectShared* sh, unsigned long long* out_key, double* out_cum) {
    unsigned long long prefix = 0;      // digits chosen so far, in place
    double before = 0.0;                // mass of candidates ordered before the chosen prefix
    for (int shift = 56; shift >= 0; shift -= 8) {
        for (int b = threadIdx.x; b < 256; b += blockDim.x) sh->mass[b] = 0.0, sh->count[b] = 0u;
        __syncthreads();
        const unsigned long long hi_mask = shift == 56 ? 0ull : (~0ull << (shift + 8));
        for (int i = threadIdx.x; i < vocab; i += blockDim.x) {
            const float v = row[i];
            const unsigned long long key = composite_key(v, i);
            if (key < floor_key || (key & hi_mask) != prefix) continue;
            const int bin = (int)((key >> shift) & 0xFFull);
            atomicAdd(&sh->mass[bin], (double)weight(v, i));
            atomicAdd(&sh->count[bin], 1u);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            double acc = before;
            int chosen = -1, last = -1;
            for (int b = 255; b >= 0; --b) {
                if (sh->count[b] == 0u) continue;
                last = b;
                const double inc = acc + sh->mass[b];
                if (strict ? (inc > target) : (inc >= target)) { chosen = b; break; }
                acc = inc;
            }
            if (chosen < 0) {           // never reached: settle on the last candidate
                chosen = last;
                acc -= sh->mass[last];
            }
            sh->chosen = chosen;
            sh->before = acc;
        }
        __syncthreads();
        if (sh->chosen < 0) {           // no candidate at all
            *out_key = floor_key;
            *out_cum = before;
            return;
        }
        prefix |= ((unsigned long long)sh->chosen) << shift;
        before = sh->before;
        __syncthreads();
    }
    // prefix is now the full key of one element
    if (threadIdx.x == 0) sh->found = 0;
    __syncthreads();
    *out_key = prefix;
    const int idx = (int)(0xFFFFFFFFu - (unsigned int)(prefix & 0xFFFFFFFFull));
    double w = 0.0;
    if (idx >= 0 && idx < vocab) w = (double)weight(row[idx], idx);
    *out_cum = before + w;
}

// The blocks that share a row of logits: a thread-block cluster (of one block where the row is short). Every
// block scans its own slice of the row; what they find meets in the shared memory of block 0 (distributed shared
// memory), between cluster barriers.
struct Team {
    int n, rank;
    int begin, end;              // this block's slice of the row (begin a multiple of 4)
    __device__ void sync() { cg::this_cluster().sync(); }
    template <typename T> __device__ T* at0(T* p) { return cg::this_cluster().map_shared_rank(p, 0); }
};

// What a reduction over the team passes through block 0: one slot per block and place of use, written before a
// cluster barrier and read after it by whoever needs the result (every block, or block 0 alone).
struct TeamSlots {
    double d[4][SAMPLE_MAX_TEAM];
    float f[2][SAMPLE_MAX_TEAM];
    unsigned int u[2][SAMPLE_MAX_TEAM];
    unsigned long long k[1][SAMPLE_MAX_TEAM];
};

// Every element of this block's slice to `f(value, index)`, a thread's elements in ascending index order. Rows
// that start on a 16-byte boundary are read 16 bytes at a time, FLIGHT such loads in flight per thread (a scan with
// one 4-byte load at a time is bound by the loads' round trips).
template <int FLIGHT = 2, typename F>
__device__ __forceinline__ void for_each_in_slice(const float* __restrict__ row, const Team& tm, F f) {
    const int begin = tm.begin, end = tm.end;
    if ((((uintptr_t)row) & 15) == 0) {
        const int g_begin = begin >> 2, g_end = end >> 2;          // whole groups of four within the slice
        const float4* r4 = reinterpret_cast<const float4*>(row);
        for (int g0 = g_begin + threadIdx.x; g0 < g_end; g0 += FLIGHT * blockDim.x) {
            float4 v[FLIGHT];
#pragma unroll
            for (int u = 0; u < FLIGHT; ++u) v[u] = r4[min(g0 + u * (int)blockDim.x, g_end - 1)];
#pragma unroll
            for (int u = 0; u < FLIGHT; ++u) {
                const int g = g0 + u * (int)blockDim.x;
                if (g < g_end) { f(v[u].x, 4 * g); f(v[u].y, 4 * g + 1); f(v[u].z, 4 * g + 2); f(v[u].w, 4 * g + 3); }
            }
        }
        for (int i = max(begin, 4 * g_end) + threadIdx.x; i < end; i += blockDim.x) f(row[i], i);
    } else {
        for (int i = begin + threadIdx.x; i < end; i += blockDim.x) f(row[i], i);
    }
}

// Maximum over the block, in every thread. `scratch33`: 33 floats of shared memory.
__device__ __forceinline__ float block_max(float v, float* scratch33) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    v = warp_max(v);
    __syncthreads();
    if (lane == 0) scratch33[warp] = v;
    __syncthreads();
    return warp_max(lane < nw ? scratch33[lane] : -CUDART_INF_F);
}

// Sum over the block; the result is valid in thread 0.
__device__ __forceinline__ double block_sum_double(double v, double* scratch33) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) scratch33[warp] = v;
    __syncthreads();
    double t = 0.0;
    if (threadIdx.x == 0)
        for (int w = 0; w < nw; ++w) t += scratch33[w];
    return t;
}

// ------------------------------------------------------------------------------------
// The same selection in two passes over the row instead of eight, for the usual case. The order of the
// candidates is by value descending, so by x = max / T - value / T ascending. A first pass counts the
// candidates and adds their weights (in float: only to find the place) into 2,048 bins of x; the bin in which
// the cumulative weight reaches the target is found from those. A second pass adds, in double, the weights of
// all candidates ordered before that bin and collects the bin's own keys, which are then sorted and walked
// exactly as the selection above walks them. If the exact sums put the crossing into a neighbouring bin, that
// bin is taken and the second pass repeated. A bin with more keys than the list holds is divided into 2,048
// bins of its own (twice at most: then its keys are equal values, and the selection above, which orders equal
// values by index digit by digit, takes over).
#define FS_BINS 2048
#define FS_CAP 2048
template <typename W>
struct FastSharedOf {
    unsigned int cnt[FS_BINS];
    float mass[FS_BINS];
    unsigned long long list[FS_CAP];
    W lp[FS_CAP];
    double dred[33];
    unsigned int n_list;
    int bin;
    int status;              // 0: walk again with `bin`; 1: found; 2: divide the bin; 3: give up (fall back)
    unsigned long long key;
    double cum;
};

__device__ __forceinline__ float value_of_key(unsigned long long key) {
    const unsigned int u = (unsigned int)(key >> 32);
    return __uint_as_float((u & 0x80000000u) ? (u & 0x7FFFFFFFu) : ~u);
}

// Returns true and the choice if the fast way settled it, false if the caller has to run select_by_mass.
// `xof(v)` is the place of a value in the order (smaller first, monotone in v), `weight(v, i)` as above,
// `approx(x)` a cheap estimate of the weight of a value at place x, good enough to find the bin.
template <int FLIGHT = 2, typename W, typename XFn, typename WeightFn, typename ApproxFn>
__device__ bool select_fast(const float* row, Team& tm, unsigned long long floor_key, double target, int strict,
                            XFn xof, float x_max, WeightFn weight, ApproxFn approx, FastSharedOf<W>* fs, TeamSlots* ts,
                            unsigned long long* out_key, double* out_cum) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    FastSharedOf<W>* fs0 = tm.at0(fs);                        // block 0's: the merged bins, the list, the verdicts
    TeamSlots* ts0 = tm.at0(ts);
    float lo = 0.f, inv_w = 64.0f;                       // bins of 1/64 from 0; the last one takes all beyond
    bool open_end = true;
    for (int level = 0; level < 3; ++level) {
        // pass 1: counts and approximate weights of the candidates per bin of [lo, ...), block by block
        for (int b = threadIdx.x; b < FS_BINS; b += blockDim.x) fs->cnt[b] = 0u, fs->mass[b] = 0.f;
        tm.sync();                                       // block 0's bins are clear before anyone adds to them
        auto bin_at = [&](float x) {                     // -1: ordered before the range; FS_BINS: after it
            const float r = (x - lo) * inv_w;
            if (r < 0.f) return -1;
            if (r >= (float)FS_BINS) return open_end ? FS_BINS - 1 : FS_BINS;
            return (int)r;
        };
        auto bin_of = [&](float v) { return bin_at(xof(v)); };
        const bool has_floor = floor_key != 0ull;
        double head = 0.0;                               // weight ordered before the range
        for_each_in_slice<FLIGHT>(row, tm, [&](float v, int i) {
            if (has_floor && composite_key(v, i) < floor_key) return;
            const float x = xof(v);
            const int b = bin_at(x);
            if (b < 0) head += (double)weight(v, i);
            else if (b < FS_BINS) {
                atomicAdd(&fs->cnt[b], 1u);
                atomicAdd(&fs->mass[b], approx(x));
            }
        });
        head = block_sum_double(head, fs->dred);
        if (threadIdx.x == 0) ts0->d[0][tm.rank] = head;
        if (tm.rank != 0) {                              // this block's bins into block 0's
            for (int b = threadIdx.x; b < FS_BINS; b += blockDim.x) {
                const unsigned int c = fs->cnt[b];
                if (c != 0u) {
                    atomicAdd(&fs0->cnt[b], c);
                    atomicAdd(&fs0->mass[b], fs->mass[b]);
                }
            }
        }
        tm.sync();
        if (tm.rank == 0 && warp == 0) {
            // a lane sums 64 consecutive bins; the lane in which the cumulative weight reaches the target walks its own
            double acc0 = 0.0;
            for (int r = 0; r < tm.n; ++r) acc0 += ts->d[0][r];
            constexpr int PER = FS_BINS / 32;
            double mine = 0.0;
            int my_last = -1;
            for (int b = lane * PER; b < (lane + 1) * PER; ++b) {
                if (fs->cnt[b] == 0u) continue;
                my_last = b;
                mine += (double)fs->mass[b];
            }
            double incl = mine;                          // inclusive sum over lanes
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double t = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += t;
            }
            const double upto = acc0 + incl;             // weight up to the end of this lane's bins
            const bool reach = my_last >= 0 && (strict ? (upto > target) : (upto >= target));
            const unsigned int who = __ballot_sync(0xffffffffu, reach);
            int last = my_last;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
            if (who != 0u && lane == __ffs(who) - 1) {
                double acc = upto - mine;
                int chosen = -1;
                for (int b = lane * PER; b < (lane + 1) * PER; ++b) {
                    if (fs->cnt[b] == 0u) continue;
                    const double inc = acc + (double)fs->mass[b];
                    if (strict ? (inc > target) : (inc >= target)) { chosen = b; break; }
                    acc = inc;
                }
                if (chosen < 0) chosen = my_last;        // rounding between the two sums: the lane's last bin
                fs->bin = chosen;
                fs->status = 0;
            }
            if (who == 0u && lane == 0) {
                fs->bin = last;                          // never reached: the last bin with candidates
                fs->status = last < 0 ? 3 : 0;           // no candidate in the range at all: not ours
            }
            if (lane == 0) fs->n_list = 0u;
        }
        tm.sync();
        if (fs0->status == 3) { tm.sync(); return false; }
        // pass 2, repeated while the exact sums move the crossing to a neighbouring bin
        int st = 0;
        for (int tries = 0; tries < 6; ++tries) {
            const int bsel = fs0->bin;
            double before = 0.0;
            unsigned int after = 0u;
            for_each_in_slice<FLIGHT>(row, tm, [&](float v, int i) {
                if (has_floor && composite_key(v, i) < floor_key) return;
                const int b = bin_of(v);
                if (b < bsel) before += (double)weight(v, i);
                else if (b == bsel) {
                    const unsigned int slot = atomicAdd(&fs0->n_list, 1u);
                    if (slot < FS_CAP) fs0->list[slot] = composite_key(v, i);
                } else ++after;
            });
            before = block_sum_double(before, fs->dred);
            const double more_d = block_sum_double((double)after, fs->dred);
            if (threadIdx.x == 0) ts0->d[1][tm.rank] = before, ts0->u[0][tm.rank] = more_d > 0.0 ? 1u : 0u;
            tm.sync();
            if (tm.rank == 0) {
                const unsigned int n = fs->n_list;
                if (n > FS_CAP) {                        // too many for the list: divide this bin
                    if (threadIdx.x == 0) fs->status = 2;
                } else {
                    // sort the bin's keys, largest first (bitonic over the next power of two, padded with zeros)
                    unsigned int m = 1u;
                    while (m < n) m <<= 1;
                    for (unsigned int i = n + threadIdx.x; i < m; i += blockDim.x) fs->list[i] = 0ull;
                    __syncthreads();
                    for (unsigned int k = 2; k <= m; k <<= 1) {
                        for (unsigned int j = k >> 1; j > 0; j >>= 1) {
                            for (unsigned int i = threadIdx.x; i < m; i += blockDim.x) {
                                const unsigned int l = i ^ j;
                                if (l > i) {
                                    const unsigned long long a = fs->list[i], c = fs->list[l];
                                    const bool desc = (i & k) == 0;
                                    if (desc ? (a < c) : (a > c)) { fs->list[i] = c; fs->list[l] = a; }
                                }
                            }
                            __syncthreads();
                        }
                    }
                    for (unsigned int i = threadIdx.x; i < n; i += blockDim.x) {
                        const unsigned long long key = fs->list[i];
                        fs->lp[i] = weight(value_of_key(key), (int)(0xFFFFFFFFu - (unsigned int)(key & 0xFFFFFFFFull)));
                    }
                    __syncthreads();
                    if (threadIdx.x == 0) {
                        double cum = 0.0;
                        unsigned int more = 0u;
                        for (int r = 0; r < tm.n; ++r) cum += ts->d[1][r], more += ts->u[0][r];
                        int v = -1;
                        if (strict ? (cum > target) : (cum >= target)) {
                            // the crossing lies before this bin: the nearest bin with candidates before it, if any
                            int b = bsel - 1;
                            while (b >= 0 && fs->cnt[b] == 0u) --b;
                            if (b >= 0) { fs->bin = b; v = 0; }
                            else if (lo > 0.f) v = 3;        // before a divided bin's range: not ours to settle
                        }
                        if (v < 0) {
                            unsigned int i = 0;
                            for (; i < n; ++i) {
                                cum += (double)fs->lp[i];
                                if (strict ? (cum > target) : (cum >= target)) break;
                            }
                            if (i < n) { fs->key = fs->list[i]; fs->cum = cum; v = 1; }
                            else if (more > 0u) {
                                int b = bsel + 1;
                                while (b < FS_BINS && fs->cnt[b] == 0u) ++b;
                                if (b < FS_BINS) { fs->bin = b; v = 0; }
                                else v = 3;                  // candidates after the range: not ours to settle
                            } else if (n > 0u) { fs->key = fs->list[n - 1]; fs->cum = cum; v = 1; }   // never reached: the last candidate
                            else v = 3;
                        }
                        fs->status = v;
                        fs->n_list = 0u;
                    }
                }
            }
            tm.sync();
            st = fs0->status;
            if (st != 0) break;
        }
        if (st == 0) st = 3;                             // six tries and still moving: give up
        if (st == 1) {
            *out_key = fs0->key;
            *out_cum = fs0->cum;
            tm.sync();
            return true;
        }
        if (st != 2) { tm.sync(); return false; }
        // divide the chosen bin: its range of x in FS_BINS bins (the open last bin up to the largest x of the row)
        const int bsel = fs0->bin;
        const float blo = lo + (float)bsel / inv_w;
        const float bhi = (open_end && bsel == FS_BINS - 1) ? x_max : lo + (float)(bsel + 1) / inv_w;
        tm.sync();
        if (!(bhi > blo)) return false;
        lo = blo;
        inv_w = (float)FS_BINS / (bhi - blo);
        open_end = false;
        if (!isfinite(inv_w)) return false;
    }
    return false;
}
