// One step of beam search: selection over beams and vocabulary, and the reordering of the
// decoder's state by the chosen beams.
//
//   l[b, v] = (x[b, v] - m_b) - log sum_u exp(x[b, u] - m_b) + S_b,    m_b = max_u x[b, u]
// and the `width` largest l of an entry's beams, equal values by the lowest b V + v.  A
// finished beam has the one candidate (b, eos) at its own score.  Masked logits (-inf, or
// NaN) and what else scores -inf come last; +inf counts as the largest finite value.  Values
// are compared as they are rounded to 32 bits, so different logits can tie.  (x - m) - log s keeps rows apart whose logits are huge or at the type's lowest value.
#include <cooperative_groups.h>
#include <utility>

#include "token_common.cuh"


namespace slg {

namespace cg = cooperative_groups;

constexpr int BM_THREADS = 512;
constexpr int BM_WARPS = BM_THREADS / 32;
constexpr int BM_PER = 32;              // logits a lane holds at once
constexpr int BM_UNIT = 32 * BM_PER;    // logits of one unit of a warp's work
constexpr int BM_MAX = SLG_BEAM_MAX;
static_assert(BM_WARPS * BM_MAX <= BM_THREADS, "the join gives every winner a thread");
constexpr float BM_LARGEST = 3.402823466e+38f;

// NaN -> -inf, +inf -> the largest finite value (fmaxf returns its other argument for NaN)
__device__ __forceinline__ float clean(float v) { return fminf(fmaxf(v, -CUDART_INF_F), BM_LARGEST); }

__device__ __forceinline__ float max_nan(float a, float b) {     // NaN when either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

constexpr float BM_LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float exp2_fast(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float exp_fast(float v) { return exp2_fast(v * BM_LOG2E); }

// A lane's sum of exp(x - m) runs as s = sum 2^(x log2(e) - ref) with ref = m log2(e) rounded to
// 32 bits: a term is one multiply-add (one rounding, like x - m), one exponential and one
// addition.  ref's own rounding is a factor common to the terms, divided out at the end.  It
// grows with m: from |m| = 65,536 on (masks at a type's lowest value) terms are
// exp(x - m) as written.
__device__ __forceinline__ bool large(float m) { return fabsf(m) >= 65536.0f; }
__device__ __forceinline__ float rounding_of(float m) {     // log2 of the factor in s
    return large(m) ? 0.0f : fmaf(m, BM_LOG2E, -(m * BM_LOG2E));
}

// Candidate order as one integer: larger value first, then the lower index.  0 = none.
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);           // -0 -> +0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t o) {
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint64_t cand_key(float v, uint32_t index) {
    return ((uint64_t)ordered(v) << 32) | (uint32_t)~index;
}
__device__ __forceinline__ uint64_t warp_max(uint64_t k) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
    return ((uint64_t)hi << 32) | lo;
}

// A candidate's score, from the beam's maximum m, logarithm l of its sum and score S.  Every
// operation is monotone in x, so a beam's candidates in the order of their logits are in the
// order of their scores -- but different logits can have the same score.
__device__ __forceinline__ float beam_score(float x, float m, float l, float S) {
    const float v = m > -CUDART_INF_F ? (x - m) - l + S : -CUDART_INF_F;
    return v == v ? v : -CUDART_INF_F;
}
__device__ __forceinline__ float finished_score(bool is_eos, float S) { return is_eos && S == S ? S : -CUDART_INF_F; }

// The n largest keys of mem[0 .. count), keys being distinct; lane i returns the i-th
// (0: there is none).
__device__ __forceinline__ uint64_t warp_select(const uint64_t* mem, int count, int n, int lane) {
    uint64_t last = ~0ull, mine = 0;
    for (int i = 0; i < n; ++i) {
        uint64_t k = 0;
        for (int c = lane; c < count; c += 32) {
            const uint64_t v = mem[c];
            if (v < last && v > k) k = v;
        }
        last = warp_max(k);
        if (lane == i) mine = last;
        if (last == 0) break;
    }
    return mine;
}

// One cluster = one entry.  A beam's logits are cut into units of 1,024, its units into
// `parts` runs, and every warp of the cluster takes (beam, part) items.  Of an item a warp
// keeps, in one pass, each lane's running maximum and sum of exponentials, and the `width`
// largest logits (lane i: the i-th): a unit is only searched while one of its lanes' maxima
// beats the list's last, so later units cost little more than their loads.  It leaves (max,
// sum, list) in the first CTA's shared memory; that CTA joins maxima and sums per beam,
// turns lists into scores, and selects.  A list goes by logits, ties by token: a logit that it
// lacks can have the score of the last chosen candidate and a lower index, so warps also keep the
// largest logit that is in no list, and where its score reaches the last chosen one's the
// candidates of that score are looked for in order (choose_equal).  Keeping it costs 25.9 -> 27.1 us
// on 64 x 8 x 32,000 fp32 and 7.3 -> 7.9 on 1 x 4 x 2,000.  Which lane sums which logits depends on their place in
// the row alone: beams with the same logits get the same normaliser, and tie.
struct BeamSlots {
    uint64_t* key;          // [items][width] (ordered logit, ~token); then (ordered score, ~index)
    float* m;               // [items]
    float* s;               // [items]
    uint32_t* out;          // [items] largest ordered logit that the list lacks, 0: none
};

__host__ __device__ inline int beam_parts(int cs, int beams, int units) {
    const int p = cs * BM_WARPS / beams;
    return p < 1 ? 1 : p < units ? p : units;
}
// at most 38,784 bytes (8 CTAs, 32 beams, width 32) beside 8,752 of fixed size
constexpr int BM_LIST = 34;             // candidates and a 0 before a warp's list in its scratch
constexpr int BM_SCRATCH = BM_LIST + 32;
static inline size_t beam_smem(int items, int beams, int width) {
    return (size_t)(items * width + (items * width & 1)) * 8 + (size_t)BM_WARPS * width * 8 + (size_t)items * 12 + beams * 12;
}

// logits [at, at + E) of a row of V, masked past its end
template <typename T>
__device__ __forceinline__ void load_logits(const T* __restrict__ row, bool aligned, int64_t at, int64_t V, float* x,
                                            uint32_t& valid, int bit) {
    constexpr int E = Pack16<T>::E;
    if (aligned && at + E <= V) {
        unpack16<T>(__ldg(reinterpret_cast<const uint4*>(row + at)), x);
        valid |= ((1u << E) - 1u) << bit;
    } else {
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const bool on = at + j < V;
            x[j] = on ? to_f32(row[at + j]) : -CUDART_INF_F;
            valid |= (on ? 1u : 0u) << (bit + j);
        }
    }
}

// Places `found` and up of the result: the candidates whose score is `last`, lowest index first.
// One CTA reads the entry's logits again, 4,096 at a time, until the places are filled.  For ties
// at the end of the result alone, which are short of lists (random fp32 logits: below one call in
// a thousand) or found within the first tokens (scores all -inf, constant logits).
constexpr int BM_AGAIN = 8;
template <typename T>
__device__ __noinline__ void choose_equal(const T* __restrict__ logits, int64_t V, int64_t ldx, int beams, int64_t entry,
                                          const float* score, const uint8_t* done, const float* m, const float* l,
                                          int32_t eos, int width, float last, int found, int* sums,
                                          float* __restrict__ out_scores, int64_t* __restrict__ parents,
                                          int64_t* __restrict__ tokens, uint8_t* __restrict__ out_finished) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int b = 0; b < beams && found < width; ++b) {
        const float S = score[b];
        if ((done[b] ? finished_score(true, S) : beam_score(m[b], m[b], l[b], S)) < last) continue;     // its best
        const T* row = logits + (entry * beams + b) * ldx;
        for (int64_t t0 = 0; t0 < V && found < width; t0 += BM_THREADS * BM_AGAIN) {
            const int64_t t1 = t0 + threadIdx.x * BM_AGAIN;
            uint32_t hits = 0;
#pragma unroll
            for (int j = 0; j < BM_AGAIN; ++j) {
                const int64_t t = t1 + j;
                if (t >= V) continue;
                const float v = done[b] ? finished_score(t == eos, S) : beam_score(clean(to_f32(row[t])), m[b], l[b], S);
                hits |= v == last ? 1u << j : 0u;
            }
            if (!__syncthreads_or(hits != 0)) continue;
            int place = __popc(hits);                       // inclusive sum over the lanes, then the warps
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, place, o);
                if (lane >= o) place += v;
            }
            if (lane == 31) sums[warp] = place;
            __syncthreads();
            int all = 0, before = 0;
            for (int q = 0; q < BM_WARPS; ++q) {
                if (q == warp) before = all;
                all += sums[q];
            }
            place += found + before - __popc(hits);
            for (; hits && place < width; hits &= hits - 1, ++place) {
                const int64_t t = t1 + __ffs(hits) - 1, o = entry * width + place;
                out_scores[o] = last;
                parents[o] = b;
                tokens[o] = t;
                if (out_finished) out_finished[o] = done[b] || t == eos;
            }
            found += all;
            __syncthreads();                                // sums are written again
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(BM_THREADS, 2)
beam_step_kernel(const T* __restrict__ logits, int64_t V, int64_t ldx, int beams, int units, const float* __restrict__ scores,
                 const uint8_t* __restrict__ finished, int32_t eos, int width, float* __restrict__ out_scores,
                 int64_t* __restrict__ parents, int64_t* __restrict__ tokens, uint8_t* __restrict__ out_finished) {
    constexpr int E = Pack16<T>::E;
    extern __shared__ __align__(16) uint64_t smem[];
    __shared__ __align__(16) uint64_t scratches[BM_WARPS][BM_SCRATCH];
    __shared__ uint32_t floors[BM_WARPS];       // per beam of the CTA: `width` logits of it reach this
    cg::cluster_group cluster = cg::this_cluster();
    const int cs = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t entry = blockIdx.x / cs;
    const int parts = beam_parts(cs, beams, units), items = beams * parts;
    BeamSlots own;
    own.key = smem;
    uint64_t* best = own.key + items * width + (items * width & 1); // [warps][width]
    own.m = reinterpret_cast<float*>(best + BM_WARPS * width);
    own.s = own.m + items;
    own.out = reinterpret_cast<uint32_t*>(own.s + items);
    float* beam_m = own.s + 2 * items;                              // [beams] maximum, log of the sum
    float* beam_l = beam_m + beams;
    uint32_t* beam_out = reinterpret_cast<uint32_t*>(beam_l + beams);   // [beams] largest logit in no list

    __shared__ float own_score[BM_MAX];         // the entry's beams, read here for the join
    __shared__ uint8_t own_done[BM_MAX];

    uint64_t* scratch = scratches[warp];
    if (threadIdx.x < BM_WARPS) floors[threadIdx.x] = 0;
    if (threadIdx.x < beams) {
        own_score[threadIdx.x] = scores[entry * beams + threadIdx.x];
        own_done[threadIdx.x] = finished && finished[entry * beams + threadIdx.x];
    }
    __syncthreads();
    auto started = cluster.barrier_arrive();                        // the first CTA's memory is there
    bool waited = false;
    for (int item = rank * BM_WARPS + warp; item < items; item += cs * BM_WARPS) {
        const int b = item / parts, part = item - b * parts;
        const int64_t row_at = entry * beams + b;
        const bool done = own_done[b];
        // the warps of a beam share its floor (with one part per beam a warp has its own)
        volatile uint32_t* floor = &floors[parts > 1 ? b - rank * BM_WARPS / parts : warp];
        if (parts == 1) *floor = 0;
        uint64_t list = 0;                                          // lane i: the i-th best so far
        uint32_t out = 0;                                           // the lane's largest logit that was left out
        float m = -CUDART_INF_F, s = 0.0f;
        if (done) {
            // eos at the beam's own score, the other tokens masked: the first part lists them
            const int t = lane == 0 ? eos : lane - 1 + (lane - 1 >= eos);
            if (part == 0 && lane < width && t < V) list = cand_key(lane == 0 ? 0.0f : -CUDART_INF_F, (uint32_t)t);
        } else {
            const T* row = logits + row_at * ldx;
            const bool aligned = (reinterpret_cast<uintptr_t>(row) & 15u) == 0;
            const int q1 = (int)((int64_t)units * (part + 1) / parts);
            for (int q = (int)((int64_t)units * part / parts); q < q1; ++q) {
                const int64_t base = (int64_t)q * BM_UNIT + lane * E;
                float x[BM_PER];
                uint32_t valid = 0;
#pragma unroll
                for (int j = 0; j < BM_PER / E; ++j)
                    load_logits<T>(row, aligned, base + j * 32 * E, V, x + j * E, valid, j * E);
                float top = x[0];
#pragma unroll
                for (int i = 1; i < BM_PER; ++i) top = max_nan(top, x[i]);
                if (!(top < CUDART_INF_F)) {                // a NaN or +inf among them
#pragma unroll
                    for (int i = 0; i < BM_PER; ++i) x[i] = clean(x[i]);
                    top = x[0];
#pragma unroll
                    for (int i = 1; i < BM_PER; ++i) top = fmaxf(top, x[i]);
                }
                if (top > m) {
                    s *= exp2_fast(rounding_of(top) - rounding_of(m)) * exp_fast(m - top);     // s = 0 at the start
                    m = top;
                }
                if (!__any_sync(0xffffffffu, large(m))) {
                    const float ref = m * BM_LOG2E;
#pragma unroll
                    for (int i = 0; i < BM_PER; ++i) s += exp2_fast(fmaf(x[i], BM_LOG2E, -ref));
                } else {                                    // also while all logits are masked
                    const float ref = m > -CUDART_INF_F ? m : 0.0f, factor = exp2_fast(rounding_of(m));
                    float t = 0.0f;
#pragma unroll
                    for (int i = 0; i < BM_PER; ++i) t += exp_fast(x[i] - ref);
                    s = fmaf(t, factor, s);
                }
                // Logits that can be among the beam's best pass the last entry of the warp's own
                // list (an equal one is a later token), and reach that of the beam's other warps;
                // while a list is being filled, also the `width`-th largest of the lanes' maxima
                // (so many logits reach that).  With "reach" for the own list too, every unit of
                // a row that is masked but for fewer tokens than `width` was searched: 64 against
                // 37 us on 64 x 8 x 32,000 with 4 tokens allowed.
                uint64_t bar = __shfl_sync(0xffffffffu, list, width - 1);
                uint32_t reach = *floor;
                if (bar != 0) reach = max(reach, (uint32_t)(bar >> 32) + 1);
                if (!__any_sync(0xffffffffu, valid && ordered(top) >= reach)) {
                    out = max(out, ordered(top));
                    continue;
                }
                if (bar == 0) {
                    uint32_t t = valid ? ordered(top) : 0u, low = 0;
                    for (int n = 0; n < width; ++n) {
                        low = __reduce_max_sync(0xffffffffu, t);
                        if (lane == __ffs(__ballot_sync(0xffffffffu, t == low)) - 1) t = 0;
                    }
                    if (low > reach) {
                        reach = low;
                        if (lane == 0) atomicMax(const_cast<uint32_t*>(floor), low);
                    }
                }
                const float least = reach ? unordered(reach) : -CUDART_INF_F;
                uint32_t left = 0;
                float below = -CUDART_INF_F;
#pragma unroll
                for (int i = 0; i < BM_PER; ++i) {
                    if (x[i] >= least) left |= 1u << i;
                    else below = fmaxf(below, x[i]);
                }
                left &= valid;
                out = max(out, ordered(below));
                // the few that qualify are read again (from L1): short code, because a step of
                // few beams mostly waits for instructions
                while (__any_sync(0xffffffffu, left != 0)) {
                    uint64_t k = 0;
                    if (left) {
                        const int i = __ffs(left) - 1;
                        left &= left - 1;
                        const int64_t at = base + (i / E) * 32 * E + i % E;
                        k = cand_key(clean(to_f32(row[at])), (uint32_t)at);
                    }
                    const uint32_t in = __ballot_sync(0xffffffffu, k > bar);
                    if (k <= bar) out = max(out, (uint32_t)(k >> 32));
                    if (in == 0) continue;
                    // the place of every candidate and every list entry is the number of keys
                    // that beat it: all are counted side by side (inserted one by one, each
                    // waits for the one before)
                    const int count = __popc(in);
                    if (k > bar) scratch[__popc(in & ((1u << lane) - 1u))] = k;
                    if (lane == 0) scratch[count] = 0;
                    scratch[BM_LIST + lane] = list;
                    __syncwarp();
                    int place = 0, moved = lane;
                    for (int j = 0; j < count; j += 2) {
                        const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(scratch + j);
                        place += (w.x > k) + (w.y > k);
                        moved += (w.x > list) + (w.y > list);
                    }
                    for (int j = 0; j < width; j += 2) {
                        const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(scratch + BM_LIST + j);
                        place += (w.x > k) + (w.y > k);
                    }
                    __syncwarp();
                    if (moved < width) scratch[BM_LIST + moved] = list;
                    else out = max(out, (uint32_t)(list >> 32));
                    if (k > bar) {
                        if (place < width) scratch[BM_LIST + place] = k;
                        else out = max(out, (uint32_t)(k >> 32));
                    }
                    __syncwarp();
                    list = lane < width ? scratch[BM_LIST + lane] : 0;
                    bar = scratch[BM_LIST + width - 1];
                    __syncwarp();
                }
                if (lane == 0 && (uint32_t)(bar >> 32) > reach) atomicMax(const_cast<uint32_t*>(floor), (uint32_t)(bar >> 32));
            }
        }
        // lanes' maxima and sums -> the warp's
        float mw = m;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mw = fmaxf(mw, __shfl_xor_sync(0xffffffffu, mw, o));
        float sw = m > -CUDART_INF_F ? s * exp2_fast(-rounding_of(m)) * exp_fast(m - mw) : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sw += __shfl_xor_sync(0xffffffffu, sw, o);
        out = __reduce_max_sync(0xffffffffu, out);
        if (!waited) {
            cluster.barrier_wait(std::move(started));
            waited = true;
        }
        uint64_t* key0 = cluster.map_shared_rank(own.key, 0);
        if (lane < width) key0[(size_t)item * width + lane] = list;
        if (lane == 0) {
            *cluster.map_shared_rank(own.m + item, 0) = mw;
            *cluster.map_shared_rank(own.s + item, 0) = sw;
            *cluster.map_shared_rank(own.out + item, 0) = out;
        }
    }
    if (!waited) cluster.barrier_wait(std::move(started));
    cluster.sync();
    if (rank != 0) return;

    for (int b = warp; b < beams; b += BM_WARPS) {
        float m = -CUDART_INF_F;
        uint32_t out = 0;
        for (int i = b * parts + lane; i < (b + 1) * parts; i += 32) {
            m = fmaxf(m, own.m[i]);
            out = max(out, own.out[i]);
        }
        out = __reduce_max_sync(0xffffffffu, out);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        float s = 0.0f;
        for (int i = b * parts + lane; i < (b + 1) * parts; i += 32)
            if (own.m[i] > -CUDART_INF_F) s += own.s[i] * exp_fast(own.m[i] - m);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) { beam_m[b] = m; beam_l[b] = logf(s); beam_out[b] = out; }
    }
    __syncthreads();
    // logits -> scores, in place; the index of (beam, token) is beam V + token
    for (int i = threadIdx.x; i < items * width; i += BM_THREADS) {
        const int b = i / (width * parts);
        const uint64_t k = own.key[i];
        uint64_t r = 0;
        if (k != 0) {
            const float S = own_score[b], x = unordered((uint32_t)(k >> 32));
            const float v = own_done[b] ? finished_score(x == 0.0f, S) : beam_score(x, beam_m[b], beam_l[b], S);
            r = cand_key(v, (uint32_t)b * (uint32_t)V + ~(uint32_t)k);
        }
        own.key[i] = r;
    }
    __syncthreads();
    {   // each warp the best of its run of items; then every winner counts the winners ahead of it
        const int a = items * warp / BM_WARPS, e = items * (warp + 1) / BM_WARPS, count = (e - a) * width;
        const uint64_t* mem = own.key + (size_t)a * width;
        if (count <= 32) {
            const uint64_t k = lane < count ? mem[lane] : 0;
            int place = 0;
#pragma unroll 4
            for (int j = 0; j < count; ++j) place += mem[j] > k;
            if (lane < width) best[warp * width + lane] = 0;
            __syncwarp();
            if (k != 0 && place < width) best[warp * width + place] = k;
        } else {
            const uint64_t k = warp_select(mem, count, width, lane);
            if (lane < width) best[warp * width + lane] = k;
        }
    }
    __syncthreads();
    __shared__ float last_score;
    __shared__ int sums[BM_WARPS];
    const int total = BM_WARPS * width;                             // at most one per thread
    float mine = -CUDART_INF_F;
    if (threadIdx.x < total) {
        const uint64_t k = best[threadIdx.x];
        int place = 0;
#pragma unroll 4
        for (int j = 0; j < total; j += 2) {
            const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(best + j);
            place += (w.x > k) + (w.y > k);
        }
        if (k != 0 && place < width) {
            const uint32_t at = ~(uint32_t)k;
            const int b = (int)(at / (uint32_t)V);
            const int64_t t = at - (uint32_t)b * (uint32_t)V, o = entry * width + place;
            mine = unordered((uint32_t)(k >> 32));
            if (place == width - 1) last_score = mine;
            out_scores[o] = mine;
            parents[o] = b;
            tokens[o] = t;
            if (out_finished) out_finished[o] = own_done[b] || t == eos;
        }
    }
    __syncthreads();
    // A candidate in no list is no better than `width` of its beam's that are in one, so it can
    // only matter with the very score of the last chosen one.
    const float last = last_score;
    bool missed = last == -CUDART_INF_F;
    if (threadIdx.x < beams && !own_done[threadIdx.x] && beam_out[threadIdx.x])
        missed |= beam_score(unordered(beam_out[threadIdx.x]), beam_m[threadIdx.x], beam_l[threadIdx.x], own_score[threadIdx.x]) >= last;
    if (!__syncthreads_or(missed)) return;
    const int better = __syncthreads_count(mine > last);
    choose_equal<T>(logits, V, ldx, beams, entry, own_score, own_done, beam_m, beam_l, eos, width, last, better, sums,
                    out_scores, parents, tokens, out_finished);
}

template <typename T>
static cudaError_t beam_step_launch(const T* x, int64_t B, int beams, int64_t V, int64_t ldx, const float* scores,
                                    const uint8_t* finished, int32_t eos, int width, float* out_scores, int64_t* parents,
                                    int64_t* tokens, uint8_t* out_finished, cudaStream_t st) {
    const int units = (int)cdiv(V, BM_UNIT);
    // CTAs per entry: as many as have a unit for every warp, at most 8, and all resident at
    // once (two per SM): a second wave of clusters would start after the first one's joins
    int cs = 1;
    while (cs < 8 && (int64_t)cs * BM_WARPS < (int64_t)beams * units && B * cs * 2 <= 2 * sm_count()) cs *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(B * cs));
    cfg.blockDim = dim3(BM_THREADS);
    cfg.dynamicSmemBytes = beam_smem(beams * beam_parts(cs, beams, units), beams, width);
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = cs;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, beam_step_kernel<T>, x, V, ldx, beams, units, scores, finished, eos, width, out_scores,
                              parents, tokens, out_finished);
}

// ----------------------------------------------------------------- reorder
// Bytes of row r of `out` = row (r / width) * beams + parents[r] of `in`; W = bytes a thread moves.
template <typename W>
__global__ void reorder_rows_kernel(const W* __restrict__ in, int64_t words, const int64_t* __restrict__ parents,
                                    int beams, int width, W* __restrict__ out) {
    const int64_t r = blockIdx.x;
    const int64_t p = parents[r];
    const bool ok = p >= 0 && p < beams;
    const W* src = in + ((r / width) * beams + (ok ? p : 0)) * words;
    for (int64_t c = (int64_t)blockIdx.y * blockDim.x + threadIdx.x; c < words; c += (int64_t)gridDim.y * blockDim.x)
        out[r * words + c] = src[c];
}

// The sample that sample r of the output is
__device__ __forceinline__ int64_t beam_source(const int64_t* __restrict__ parents, uint32_t r, int beams, int width) {
    const int64_t p = parents[r];
    return (int64_t)(r / (uint32_t)width) * beams + (p >= 0 && p < beams ? p : 0);
}

// Column r of every feature row = column source(r); padding columns 0.  A thread keeps its
// column and walks rows, so the source is worked out once.
constexpr int RF_ROWS = 8;              // rows of a CTA per step
__global__ void __launch_bounds__(32 * RF_ROWS)
reorder_features_kernel(const float* __restrict__ in, int64_t F, int64_t ldi, int64_t n,
                        const int64_t* __restrict__ parents, int beams, int width, float* __restrict__ out,
                        int64_t ldo) {
    const int64_t r = (int64_t)blockIdx.x * 32 + threadIdx.x;
    if (r >= ldo) return;
    const bool on = r < n;
    const int64_t src = on ? beam_source(parents, (uint32_t)r, beams, width) : 0;
#pragma unroll 4
    for (int64_t f = (int64_t)blockIdx.y * RF_ROWS + threadIdx.y; f < F; f += (int64_t)gridDim.y * RF_ROWS)
        out[f * ldo + r] = on ? __ldg(&in[f * ldi + src]) : 0.0f;
}

// The same on bits.  A thread builds one 32-bit word of a row bit by bit; a CTA's threads
// walk (row, word) of 32 word columns, row by row, so stores are whole lines (a warp that
// built one word by ballot stored 4 bytes at a time: 10 us on 10,000 x 512).  The sources of the
// 1,024 samples are worked out once per CTA.  FOUR: a word's sources lie in four words, which are
// loaded first (sources_in_four below); otherwise every bit loads its word.
constexpr int RP_THREADS = 256;
constexpr int RP_WORDS = 32;
constexpr uint32_t RP_NONE = 0xffffffffu;

// A word's first sample is at most width - 1 into its entry, so its last one's entry begins at
// most (width + 30) / width entries after the first's, and that many times `beams` samples; the
// first source word begins at most 31 samples before its entry's first.
inline int64_t last_source_offset(int64_t beams, int64_t width) { return 31 + ((width + 30) / width) * beams + beams - 1; }
inline bool sources_in_four(int64_t beams, int64_t width) { return last_source_offset(beams, width) < 128; }

template <bool FOUR>
__global__ void __launch_bounds__(RP_THREADS)
reorder_packed_kernel(const uint32_t* __restrict__ in, int64_t F, int64_t ldi, int64_t n,
                      const int64_t* __restrict__ parents, int beams, int width, uint32_t* __restrict__ out,
                      int64_t ldo) {
    __shared__ int64_t word_of[RP_WORDS];       // first source word of an output word
    // bit's source: 32 (word - first) + bit; FOUR reads two at a time, and needs 7 bits
    using From = typename std::conditional<FOUR, uint16_t, uint32_t>::type;
    __shared__ __align__(4) From from[RP_WORDS][FOUR ? 34 : 33];
    const int64_t w0 = (int64_t)blockIdx.y * RP_WORDS;
    const int words = (int)min((int64_t)RP_WORDS, ldo - w0);
    for (int i = threadIdx.x; i < words * 32; i += RP_THREADS) {
        const int64_t r0 = (w0 + i / 32) * 32, r = r0 + i % 32;
        const int64_t first = ((int64_t)((uint32_t)r0 / (uint32_t)width) * beams) >> 5;
        from[i / 32][i % 32] =
            r < n ? (From)(beam_source(parents, (uint32_t)r, beams, width) - first * 32) : (From)RP_NONE;
        if (i % 32 == 0) word_of[i / 32] = first;
    }
    __syncthreads();
    const int64_t total = F * words;
    const int64_t t = (int64_t)blockIdx.x * RP_THREADS + threadIdx.x;
    if (t < total) {
        const int64_t f = total < (1ll << 32) ? (int64_t)((uint32_t)t / (uint32_t)words) : t / words;
        const int w = (int)(t - f * words);
        const int64_t first = word_of[w];
        const uint32_t* src = in + f * ldi + first;
        uint32_t bits = 0;
        if constexpr (FOUR) {
            uint32_t x[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) x[q] = first + q < ldi ? __ldg(src + q) : 0u;
#pragma unroll 8
            for (int j = 0; j < 32; j += 2) {
                const uint32_t two = *reinterpret_cast<const uint32_t*>(&from[w][j]);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t s = h ? two >> 16 : two & 0xffffu;
                    const uint32_t lo = s & 32u ? x[1] : x[0], hi = s & 32u ? x[3] : x[2];
                    const uint32_t bit = (s & 64u ? hi : lo) >> (s & 31u) & 1u;
                    bits |= (s == 0xffffu ? 0u : bit) << (j + h);
                }
            }
        } else {
#pragma unroll 8
            for (int j = 0; j < 32; ++j) {
                const uint32_t s = from[w][j];
                if (s != RP_NONE) bits |= (__ldg(src + (s >> 5)) >> (s & 31u) & 1u) << j;
            }
        }
        out[f * ldo + w0 + w] = bits;
    }
}

}  // namespace slg

using namespace slg;

extern "C" int slg_beam_step(const void* logits, int32_t dtype, int64_t B, int32_t beams, int64_t V, int64_t ldx,
                             const float* scores, const uint8_t* finished, int32_t eos, int32_t width,
                             float* out_scores, int64_t* parents, int64_t* tokens, uint8_t* out_finished,
                             void* stream) {
    const char* name = "slg_beam_step";
    if (B < 0 || beams <= 0 || V <= 0 || width <= 0) return set_error(SLG_ERR_ARG, "%s: bad sizes", name);
    if (beams > BM_MAX || width > BM_MAX)
        return set_error(SLG_ERR_UNSUPPORTED, "%s: at most %d beams", name, BM_MAX);
    if (V >= 1 << 27) return set_error(SLG_ERR_UNSUPPORTED, "%s: vocabulary must be below 2^27", name);
    if (width > beams * V) return set_error(SLG_ERR_ARG, "%s: width %d > beams * vocabulary", name, width);
    if (ldx < V) return set_error(SLG_ERR_ARG, "%s: ldx < vocabulary", name);
    if (finished && (eos < 0 || eos >= V)) return set_error(SLG_ERR_ARG, "%s: finished needs eos in the vocabulary", name);
    if (dtype != SLG_DT_F32 && dtype != SLG_DT_BF16 && dtype != SLG_DT_F16)
        return set_error(SLG_ERR_UNSUPPORTED, "%s: dtype %d not built", name, dtype);
    if (B >= 1 << 27) return set_error(SLG_ERR_ARG, "%s: batch too large", name);
    if (B == 0) return SLG_OK;
    if (!logits || !scores || !out_scores || !parents || !tokens)
        return set_error(SLG_ERR_ARG, "%s: null pointer", name);
    cudaError_t e = cudaSuccess;
    for_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        e = beam_step_launch<T>((const T*)logits, B, beams, V, ldx, scores, finished, eos, width, out_scores, parents,
                                tokens, out_finished, as_stream(stream));
    });
    if (e != cudaSuccess) {
        cudaGetLastError();             // reported here: the next call starts clean
        return set_error(SLG_ERR_CUDA, "%s: %s", name, cudaGetErrorString(e));
    }
    return check_launch(name);
}

static int check_reorder(const void* in, const int64_t* parents, const void* out, int64_t B, int32_t beams,
                         int32_t width, const char* name) {
    if (B < 0 || beams <= 0 || width <= 0) return set_error(SLG_ERR_ARG, "%s: bad sizes", name);
    if (!in || !parents || !out) return set_error(SLG_ERR_ARG, "%s: null pointer", name);
    if (in == out) return set_error(SLG_ERR_ARG, "%s: in-place reordering is not possible", name);
    if (B * width >= (1ll << 31)) return set_error(SLG_ERR_ARG, "%s: batch too large", name);
    return SLG_OK;
}

extern "C" int slg_beam_reorder_rows(const void* in, int64_t row_bytes, const int64_t* parents, int64_t B,
                                     int32_t beams, int32_t width, void* out, void* stream) {
    if (B == 0 || row_bytes == 0) return SLG_OK;
    int st = check_reorder(in, parents, out, B, beams, width, "slg_beam_reorder_rows");
    if (st) return st;
    if (row_bytes < 0) return set_error(SLG_ERR_ARG, "slg_beam_reorder_rows: bad sizes");
    cudaStream_t s = as_stream(stream);
    const unsigned n = (unsigned)(B * width);
    auto go = [&](auto w) {
        using W = decltype(w);
        const int64_t words = row_bytes / (int64_t)sizeof(W);
        const dim3 grid(n, (unsigned)std::min<int64_t>(cdiv(words, 256 * 4), 64));
        reorder_rows_kernel<W><<<grid, 256, 0, s>>>((const W*)in, words, parents, beams, width, (W*)out);
    };
    if (row_bytes % 16 == 0 && aligned16(in) && aligned16(out)) go(uint4());
    else if (row_bytes % 4 == 0 && aligned_to(in, 4) && aligned_to(out, 4)) go(uint32_t());
    else if (row_bytes % 2 == 0 && aligned_to(in, 2) && aligned_to(out, 2)) go(uint16_t());
    else go(uint8_t());
    return check_launch("slg_beam_reorder_rows");
}

extern "C" int slg_beam_reorder_features(const float* in, int64_t F, int64_t ldi, const int64_t* parents, int64_t B,
                                         int32_t beams, int32_t width, float* out, int64_t ldo, void* stream) {
    if (F == 0 || B == 0) return SLG_OK;
    int st = check_reorder(in, parents, out, B, beams, width, "slg_beam_reorder_features");
    if (st) return st;
    if (F < 0 || ldi < B * beams || ldo < B * width)
        return set_error(SLG_ERR_ARG, "slg_beam_reorder_features: bad sizes");
    const dim3 grid((unsigned)cdiv(ldo, 32), (unsigned)std::min<int64_t>(cdiv(F, RF_ROWS * 4), 65535));
    reorder_features_kernel<<<grid, dim3(32, RF_ROWS), 0, as_stream(stream)>>>(in, F, ldi, B * width, parents, beams, width, out, ldo);
    return check_launch("slg_beam_reorder_features");
}

extern "C" int slg_beam_reorder_packed(const uint64_t* in, int64_t F, int64_t ldi, const int64_t* parents, int64_t B,
                                       int32_t beams, int32_t width, uint64_t* out, int64_t ldo, void* stream) {
    if (F == 0 || B == 0) return SLG_OK;
    int st = check_reorder(in, parents, out, B, beams, width, "slg_beam_reorder_packed");
    if (st) return st;
    if (F < 0 || ldi * 64 < B * beams || ldo * 64 < B * width)
        return set_error(SLG_ERR_ARG, "slg_beam_reorder_packed: bad sizes");
    const int64_t per_row = std::min<int64_t>(2 * ldo, RP_WORDS), tiles = cdiv(2 * ldo, RP_WORDS);
    if (tiles > 65535) return set_error(SLG_ERR_ARG, "slg_beam_reorder_packed: batch too large");
    if (last_source_offset(beams, width) >= (int64_t)RP_NONE)
        return set_error(SLG_ERR_UNSUPPORTED, "slg_beam_reorder_packed: %d beams per entry", beams);
    const dim3 grid((unsigned)cdiv(F * per_row, RP_THREADS), (unsigned)tiles);
    auto go = [&](auto kernel) {
        kernel<<<grid, RP_THREADS, 0, as_stream(stream)>>>(reinterpret_cast<const uint32_t*>(in), F, 2 * ldi, B * width,
                                                           parents, beams, width, reinterpret_cast<uint32_t*>(out), 2 * ldo);
    };
    if (sources_in_four(beams, width)) go(reorder_packed_kernel<true>);
    else go(reorder_packed_kernel<false>);
    return check_launch("slg_beam_reorder_packed");
}
