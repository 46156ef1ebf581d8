// Token embedding: scaled lookup, and its gradient by sorted tokens.
//
//   y[i, :]  = s W[t_i, :]                              (forward)
//   dW[v, :] = s sum_{i : t_i = v} g[i, :]              (backward)
//
// The gradient is a segmented sum over the tokens in sorted order.  A stable radix sort
// orders (token, position) pairs, so every row's terms are added in a fixed order and the
// result is the same from run to run; sums are held in 32 bits and rounded once.
#include "token_common.cuh"

namespace slg {

constexpr int EM_THREADS = 256;
constexpr int EM_UNROLL = 4;        // 16-byte vectors per thread of the lookup

// ------------------------------------------------------------------ lookup
// One thread = EM_UNROLL 16-byte vectors of the output; VEC: rows are whole vectors.
template <typename T, typename I, bool VEC>
__global__ void __launch_bounds__(EM_THREADS)
embed_fwd_kernel(const I* __restrict__ ids, int64_t N, const T* __restrict__ w, int64_t V, int64_t D,
                 float scale, T* __restrict__ y) {
    constexpr int E = Pack16<T>::E;
    const int64_t total = N * D;
    const int64_t base = ((int64_t)blockIdx.x * EM_THREADS * EM_UNROLL + threadIdx.x) * E;
#pragma unroll
    for (int u = 0; u < EM_UNROLL; ++u) {
        const int64_t e0 = base + (int64_t)u * EM_THREADS * E;
        if (e0 >= total) continue;
        int64_t i = e0 / D, c = e0 - i * D;
        int64_t t = (int64_t)ids[i];
        float v[E];
        if constexpr (VEC) {
            if (t >= 0 && t < V) unpack16<T>(__ldg(reinterpret_cast<const uint4*>(w + t * D + c)), v);
            else
#pragma unroll
                for (int j = 0; j < E; ++j) v[j] = CUDART_NAN_F;
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j) {
                v[j] = e0 + j >= total ? 0.0f : t >= 0 && t < V ? to_f32(w[t * D + c]) : CUDART_NAN_F;
                if (++c == D && e0 + j + 1 < total) { c = 0; t = (int64_t)ids[++i]; }
            }
        }
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] *= scale;
        if (e0 + E <= total) *reinterpret_cast<uint4*>(y + e0) = pack16<T>(v);
        else
#pragma unroll
            for (int j = 0; j < E; ++j)
                if (e0 + j < total) y[e0 + j] = from_f32<T>(v[j]);
    }
}

// -------------------------------------------------------------------- sort
// Stable LSD radix sort of (token, position), 8 bits a pass.  Tokens that get no gradient
// (padding, out of range) carry the key V and sort past every row.
constexpr int RS_THREADS = 256;
constexpr int RS_WARPS = RS_THREADS / 32;
constexpr int RS_PER = 16;                          // keys per thread of a tile
constexpr int RS_TILE = RS_THREADS * RS_PER;
constexpr int RS_BINS = 256;
constexpr int RS_MAX_TILES = 256;

__host__ __device__ inline int64_t rs_span(int64_t N) {   // keys per CTA: whole tiles, at most RS_MAX_TILES CTAs
    return RS_TILE * cdiv(cdiv(N, RS_TILE), RS_MAX_TILES);
}

template <typename I>
struct KeysOfIds {
    const I* ids; int64_t V; int64_t pad;
    __device__ __forceinline__ uint32_t key(int64_t i) const {
        const int64_t t = (int64_t)ids[i];
        return t >= 0 && t < V && t != pad ? (uint32_t)t : (uint32_t)V;
    }
    __device__ __forceinline__ uint32_t pos(int64_t i) const { return (uint32_t)i; }
};
struct KeysOfPairs {
    const uint32_t* k; const uint32_t* p;
    __device__ __forceinline__ uint32_t key(int64_t i) const { return k[i]; }
    __device__ __forceinline__ uint32_t pos(int64_t i) const { return p[i]; }
};

// hist[cta][digit]
template <typename S>
__global__ void __launch_bounds__(RS_THREADS)
radix_count_kernel(S src, int64_t N, int64_t span, int shift, uint32_t* __restrict__ hist) {
    __shared__ uint32_t h[RS_BINS];
    h[threadIdx.x] = 0;
    __syncthreads();
    const int64_t a = (int64_t)blockIdx.x * span, b = a + span < N ? a + span : N;
    for (int64_t i = a + threadIdx.x; i < b; i += RS_THREADS) atomicAdd(&h[(src.key(i) >> shift) & 255u], 1u);
    __syncthreads();
    hist[(int64_t)blockIdx.x * RS_BINS + threadIdx.x] = h[threadIdx.x];
}

// Thread d owns digit d.  Its first slot is the number of keys with a smaller digit plus
// those with digit d in earlier CTAs; inside a tile a warp owns consecutive keys, ranks
// them 32 at a time by matching digits, and warps follow one another: the order is stable.
template <typename S>
__global__ void __launch_bounds__(RS_THREADS)
radix_scatter_kernel(S src, int64_t N, int64_t span, int shift, const uint32_t* __restrict__ hist,
                     uint32_t* __restrict__ ko, uint32_t* __restrict__ po) {
    __shared__ uint32_t base[RS_BINS];
    __shared__ uint32_t cnt[RS_WARPS][RS_BINS];
    __shared__ uint32_t wsum[RS_WARPS];
    const int d = threadIdx.x, warp = d >> 5, lane = d & 31;
    uint32_t before = 0, all = 0;
#pragma unroll 8
    for (int t = 0; t < (int)gridDim.x; ++t) {
        const uint32_t c = hist[(int64_t)t * RS_BINS + d];
        before += t < (int)blockIdx.x ? c : 0u;
        all += c;
    }
    uint32_t inc = all;                                    // inclusive scan over digits
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
    }
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    for (int q = 0; q < warp; ++q) inc += wsum[q];
    base[d] = inc - all + before;

    const int64_t a = (int64_t)blockIdx.x * span, b = a + span < N ? a + span : N;
    for (int64_t t0 = a; t0 < b; t0 += RS_TILE) {
#pragma unroll
        for (int q = 0; q < RS_WARPS; ++q) cnt[q][d] = 0;
        __syncthreads();
        uint32_t key[RS_PER], rank[RS_PER];
        const int64_t w0 = t0 + warp * (32 * RS_PER) + lane;
#pragma unroll
        for (int j = 0; j < RS_PER; ++j) key[j] = w0 + 32 * j < b ? src.key(w0 + 32 * j) : 0u;
#pragma unroll
        for (int j = 0; j < RS_PER; ++j) {
            const bool on = w0 + 32 * j < b;
            const uint32_t dg = on ? (key[j] >> shift) & 255u : 256u;
            const uint32_t peers = __match_any_sync(0xffffffffu, dg);
            rank[j] = __popc(peers & ((1u << lane) - 1u));
            if (on) rank[j] += cnt[warp][dg];
            __syncwarp();
            if (on && (peers >> lane) == 1u) cnt[warp][dg] += __popc(peers);    // the last of them
            __syncwarp();
        }
        __syncthreads();
        uint32_t run = base[d];                            // warps of the tile follow one another
#pragma unroll
        for (int q = 0; q < RS_WARPS; ++q) {
            const uint32_t c = cnt[q][d];
            cnt[q][d] = run;
            run += c;
        }
        base[d] = run;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < RS_PER; ++j)
            if (w0 + 32 * j < b) {
                const uint32_t o = cnt[warp][(key[j] >> shift) & 255u] + rank[j];
                ko[o] = key[j];
                po[o] = src.pos(w0 + 32 * j);
            }
        __syncthreads();
    }
}

// ------------------------------------------------------------ segmented sum
// The sorted tokens and the row ends 0 .. V-1 are merged into one list of V + N items (a
// row's end comes after its tokens), and the list is cut into equal chunks: an entry costs
// a read of D values, a row end a write of D values, so every chunk costs the same
// whatever the tokens' distribution.  A row whose items lie in one chunk is written there.  A row
// that is cut leaves its sums in `tail` (row goes on in the next chunk) and `head` (row
// ends here, begun earlier); embed_join_kernel adds those in chunk order.
struct Cut { int64_t r, i; };

// Row ends and entries among the first d items, by a 33-way search of a full warp.  Row
// end r is among them iff at most d - r - 1 entries have a token <= r.
__device__ __forceinline__ Cut merge_cut(const uint32_t* __restrict__ key, int64_t N, int64_t V, int64_t d, int lane) {
    int64_t lo = d > N ? d - N : 0, hi = d < V ? d : V;        // answer in [lo, hi]
    while (lo < hi) {
        const int64_t step = (hi - lo + 32) / 33;              // probes lo + step*(lane+1) - 1
        const int64_t r = lo + step * (lane + 1) - 1;
        bool in = false;
        if (r < hi) {
            const int64_t m = d - r - 1;
            in = m >= N || (int64_t)key[m] > r;
        }
        const int n = __popc(__ballot_sync(0xffffffffu, in));   // the first n probes hold
        const int64_t nlo = lo + step * n;
        hi = n == 32 ? hi : (nlo + step - 1 < hi ? nlo + step - 1 : hi);
        lo = nlo;
    }
    return {lo, d - lo};
}

// A lane's E values of columns [c0, c0 + 32 E) of a row: one vector, or (VEC false: rows
// start on no 16-byte boundary) every 32nd value.
template <typename T, bool VEC> struct Cols {
    static constexpr int E = Pack16<T>::E;
    uint4 u;
    __device__ __forceinline__ void load(const T* __restrict__ row, int64_t c0, int64_t D, int lane) {
        const int64_t c = c0 + lane * E;
        u = c < D ? __ldg(reinterpret_cast<const uint4*>(row + c)) : make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void add_to(float (&acc)[E]) const {
        float x[E];
        unpack16<T>(u, x);
#pragma unroll
        for (int j = 0; j < E; ++j) acc[j] += x[j];
    }
};
template <typename T> struct Cols<T, false> {
    static constexpr int E = Pack16<T>::E;
    T x[E];
    __device__ __forceinline__ void load(const T* __restrict__ row, int64_t c0, int64_t D, int lane) {
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const int64_t c = c0 + lane + 32 * j;
            x[j] = c < D ? row[c] : from_f32<T>(0.0f);
        }
    }
    __device__ __forceinline__ void add_to(float (&acc)[E]) const {
#pragma unroll
        for (int j = 0; j < E; ++j) acc[j] += to_f32(x[j]);
    }
};

template <typename T, bool VEC>
__device__ __forceinline__ void store_row(T* __restrict__ row, int64_t c0, int64_t D, int lane, float scale,
                                          const float (&acc)[Pack16<T>::E]) {
    constexpr int E = Pack16<T>::E;
    if constexpr (VEC) {
        const int64_t c = c0 + lane * E;
        float v[E];
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = acc[j] * scale;
        if (c < D) *reinterpret_cast<uint4*>(row + c) = pack16<T>(v);
    } else {
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const int64_t c = c0 + lane + 32 * j;
            if (c < D) row[c] = from_f32<T>(acc[j] * scale);
        }
    }
}

// carry rows hold a lane's E sums side by side: [slice][lane][E] floats
template <int E>
__device__ __forceinline__ void store_carry(float* __restrict__ p, int lane, const float (&acc)[E]) {
#pragma unroll
    for (int j = 0; j < E; j += 4)
        *reinterpret_cast<float4*>(p + lane * E + j) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
}
template <int E>
__device__ __forceinline__ void add_carry(const float* __restrict__ p, int lane, float (&acc)[E]) {
#pragma unroll
    for (int j = 0; j < E; j += 4) {
        const float4 v = *reinterpret_cast<const float4*>(p + lane * E + j);
        acc[j] += v.x; acc[j + 1] += v.y; acc[j + 2] += v.z; acc[j + 3] += v.w;
    }
}

constexpr int SG_WARPS = 4;
constexpr int SG_UNROLL = 8;

// head_row[chunk] = row that ends in this chunk but began earlier, else -1
template <typename T, bool VEC>
__global__ void __launch_bounds__(SG_WARPS * 32)
embed_sum_kernel(const uint32_t* __restrict__ key, const uint32_t* __restrict__ pos, int64_t N, int64_t V,
                 int64_t D, int64_t chunk, const T* __restrict__ g, float scale, T* __restrict__ gw,
                 float* __restrict__ carry, int64_t slices, int32_t* __restrict__ head_row) {
    constexpr int E = Pack16<T>::E;
    constexpr int SLICE = 32 * E;
    __shared__ Cut cut[2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t total = V + N;
    const int64_t c = blockIdx.x;
    if (warp < 2) {
        const int64_t d = (c + warp) * chunk;
        const Cut x = merge_cut(key, N, V, d < total ? d : total, lane);
        if (lane == 0) cut[warp] = x;
    }
    __syncthreads();
    const int64_t r0 = cut[0].r, i0 = cut[0].i, r1 = cut[1].r;
    int64_t i1 = cut[1].i;
    const bool begun = r0 < V && i0 > 0 && (int64_t)key[i0 - 1] == r0;      // r0 has entries in earlier chunks
    if (threadIdx.x == 0 && blockIdx.y == 0) head_row[c] = begun && r1 > r0 ? (int32_t)r0 : -1;
    if (r1 == V) {                      // what follows the last row's end has no gradient
        while (i1 > i0 && (int64_t)key[i1 - 1] >= V) --i1;
    }
    for (int64_t s = (int64_t)blockIdx.y * SG_WARPS + warp; s < slices; s += (int64_t)gridDim.y * SG_WARPS) {
        const int64_t c0 = s * SLICE;
        float* head = carry + ((2 * c) * slices + s) * SLICE;
        float* tail = carry + ((2 * c + 1) * slices + s) * SLICE;
        float acc[E];
#pragma unroll
        for (int j = 0; j < E; ++j) acc[j] = 0.0f;
        int64_t r = r0;
        auto end_rows = [&](int64_t upto) {                 // rows r .. upto-1 end here
            for (; r < upto; ++r) {
                if (r == r0 && begun) store_carry<E>(head, lane, acc);
                else store_row<T, VEC>(gw + r * D, c0, D, lane, scale, acc);
#pragma unroll
                for (int j = 0; j < E; ++j) acc[j] = 0.0f;
            }
        };
        for (int64_t i = i0; i < i1; i += SG_UNROLL) {
            Cols<T, VEC> v[SG_UNROLL];
            uint32_t k[SG_UNROLL];
#pragma unroll
            for (int u = 0; u < SG_UNROLL; ++u) {
                k[u] = i + u < i1 ? key[i + u] : 0u;
                if (i + u < i1) v[u].load(g + (int64_t)pos[i + u] * D, c0, D, lane);
            }
#pragma unroll
            for (int u = 0; u < SG_UNROLL; ++u) {
                if (i + u >= i1) break;
                end_rows((int64_t)k[u]);
                v[u].add_to(acc);
            }
        }
        end_rows(r1);
        if (r1 < V) store_carry<E>(tail, lane, acc);        // all zeros when r1 has no entry here
    }
}

// One warp = one cut row x one slice: tails from the row's first chunk on, then the head.
template <typename T, bool VEC>
__global__ void __launch_bounds__(SG_WARPS * 32)
embed_join_kernel(const uint32_t* __restrict__ key, int64_t N, int64_t V, int64_t D, int64_t chunk,
                  int64_t nchunk, float scale, T* __restrict__ gw, const float* __restrict__ carry,
                  int64_t slices, const int32_t* __restrict__ head_row) {
    constexpr int E = Pack16<T>::E;
    constexpr int SLICE = 32 * E;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t c = blockIdx.x;
    const int64_t r = head_row[c];
    if (r < 0) return;
    // the row's first entry: the number of entries with a smaller token (33-way search)
    int64_t lo = 0, hi = N;
    while (lo < hi) {
        const int64_t step = (hi - lo + 32) / 33;
        const int64_t m = lo + step * (lane + 1) - 1;
        const int n = __popc(__ballot_sync(0xffffffffu, m < hi && (int64_t)key[m] < r));
        const int64_t nlo = lo + step * n;
        hi = n == 32 ? hi : (nlo + step - 1 < hi ? nlo + step - 1 : hi);
        lo = nlo;
    }
    const int64_t first = (lo + r) / chunk;                 // r row ends come before it
    for (int64_t s = (int64_t)blockIdx.y * SG_WARPS + warp; s < slices; s += (int64_t)gridDim.y * SG_WARPS) {
        float acc[E];
#pragma unroll
        for (int j = 0; j < E; ++j) acc[j] = 0.0f;
#pragma unroll 8
        for (int64_t q = first; q < c; ++q) add_carry<E>(carry + ((2 * q + 1) * slices + s) * SLICE, lane, acc);
        add_carry<E>(carry + ((2 * c) * slices + s) * SLICE, lane, acc);
        store_row<T, VEC>(gw + r * D, s * SLICE, D, lane, scale, acc);
    }
}

// ------------------------------------------------------------------- plans
struct EmbedPlan {
    int64_t keys_at, hist_at, head_at, carry_at, bytes;
    int64_t chunk, nchunk, slices, tiles;
    int passes;
};

static int bits_of(uint64_t v) { int n = 0; while (v) { ++n; v >>= 1; } return n; }

static EmbedPlan embed_plan(int64_t N, int64_t V, int64_t D, int es) {
    EmbedPlan p;
    auto up = [](int64_t v) { return cdiv(v, 256) * 256; };
    p.tiles = N > 0 ? cdiv(N, rs_span(N)) : 0;
    p.passes = (int)cdiv(bits_of((uint64_t)V), 8);          // keys 0 .. V
    p.slices = cdiv(D * es, 512);                           // 32 lanes x 16 bytes
    p.chunk = 64;
    p.nchunk = cdiv(V + N, p.chunk);
    p.keys_at = 0;
    p.hist_at = p.keys_at + up(4 * 4 * N);
    p.head_at = p.hist_at + up(p.tiles * RS_BINS * 4);
    p.carry_at = p.head_at + up(p.nchunk * 4);
    p.bytes = p.carry_at + p.nchunk * 2 * p.slices * (512 / es) * 4;
    return p;
}

static int check_embed(int64_t N, int64_t V, int64_t D, int ids64, int dtype, const char* name) {
    if (N < 0 || V <= 0 || D <= 0) return set_error(SLG_ERR_ARG, "%s: bad sizes", name);
    if (N >= (1ll << 31) || V >= (1ll << 31) - 1)
        return set_error(SLG_ERR_UNSUPPORTED, "%s: tokens and vocabulary must be below 2^31", name);
    if (ids64 != 0 && ids64 != 1) return set_error(SLG_ERR_ARG, "%s: ids64 must be 0 or 1", name);
    if (dtype != SLG_DT_F32 && dtype != SLG_DT_BF16 && dtype != SLG_DT_F16)
        return set_error(SLG_ERR_UNSUPPORTED, "%s: dtype %d not built", name, dtype);
    return SLG_OK;
}

template <typename T, typename I>
static void embed_fwd_launch(const I* ids, int64_t N, const T* w, int64_t V, int64_t D, float scale, T* y,
                             cudaStream_t st) {
    const int64_t vecs = cdiv(N * D, Pack16<T>::E);
    const unsigned grid = (unsigned)cdiv(vecs, EM_THREADS * EM_UNROLL);
    if (D % Pack16<T>::E == 0 && aligned16(w))
        embed_fwd_kernel<T, I, true><<<grid, EM_THREADS, 0, st>>>(ids, N, w, V, D, scale, y);
    else
        embed_fwd_kernel<T, I, false><<<grid, EM_THREADS, 0, st>>>(ids, N, w, V, D, scale, y);
}

template <typename I>
static const uint32_t* embed_sort(const I* ids, int64_t N, int64_t V, int64_t pad, const EmbedPlan& p, char* ws,
                                  cudaStream_t st) {
    uint32_t* buf[2] = {reinterpret_cast<uint32_t*>(ws + p.keys_at),
                        reinterpret_cast<uint32_t*>(ws + p.keys_at) + 2 * N};
    uint32_t* hist = reinterpret_cast<uint32_t*>(ws + p.hist_at);
    const int64_t span = rs_span(N);
    const KeysOfIds<I> in{ids, V, pad};
    uint32_t* src = nullptr;
    for (int q = 0; q < p.passes; ++q) {
        uint32_t* dst = buf[q & 1];
        const unsigned grid = (unsigned)p.tiles;
        if (q == 0) {
            radix_count_kernel<<<grid, RS_THREADS, 0, st>>>(in, N, span, 0, hist);
            radix_scatter_kernel<<<grid, RS_THREADS, 0, st>>>(in, N, span, 0, hist, dst, dst + N);
        } else {
            const KeysOfPairs pairs{src, src + N};
            radix_count_kernel<<<grid, RS_THREADS, 0, st>>>(pairs, N, span, 8 * q, hist);
            radix_scatter_kernel<<<grid, RS_THREADS, 0, st>>>(pairs, N, span, 8 * q, hist, dst, dst + N);
        }
        src = dst;
    }
    return src;
}

template <typename T>
static void embed_bwd_launch(const uint32_t* key, int64_t N, int64_t V, int64_t D, const T* g, float scale, T* gw,
                             const EmbedPlan& p, char* ws, cudaStream_t st) {
    float* carry = reinterpret_cast<float*>(ws + p.carry_at);
    int32_t* head = reinterpret_cast<int32_t*>(ws + p.head_at);
    const uint32_t* pos = key + N;
    const dim3 grid((unsigned)p.nchunk, (unsigned)std::min<int64_t>(cdiv(p.slices, SG_WARPS), 65535));
    auto go = [&](auto vec) {
        constexpr bool VEC = decltype(vec)::value;
        embed_sum_kernel<T, VEC><<<grid, SG_WARPS * 32, 0, st>>>(key, pos, N, V, D, p.chunk, g, scale, gw, carry,
                                                                 p.slices, head);
        if (N > 0)
            embed_join_kernel<T, VEC><<<grid, SG_WARPS * 32, 0, st>>>(key, N, V, D, p.chunk, p.nchunk, scale, gw,
                                                                      carry, p.slices, head);
    };
    if (D % Pack16<T>::E == 0 && aligned16(g) && aligned16(gw)) go(std::true_type{});
    else go(std::false_type{});
}

}  // namespace slg

using namespace slg;

extern "C" int slg_embed_fwd(const void* ids, int32_t ids64, int64_t N, const void* weight, int32_t dtype, int64_t V,
                             int64_t D, float scale, void* out, void* stream) {
    int st = check_embed(N, V, D, ids64, dtype, "slg_embed_fwd");
    if (st) return st;
    if (N == 0) return SLG_OK;
    if (!ids || !weight || !out) return set_error(SLG_ERR_ARG, "slg_embed_fwd: null pointer");
    if (!aligned16(out)) return set_error(SLG_ERR_ALIGN, "slg_embed_fwd: out not 16-byte aligned");
    if (cdiv(N * D, 4) > (1ll << 31) * 1000) return set_error(SLG_ERR_ARG, "slg_embed_fwd: too many values");
    cudaStream_t s = as_stream(stream);
    for_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        if (ids64) embed_fwd_launch<T, int64_t>((const int64_t*)ids, N, (const T*)weight, V, D, scale, (T*)out, s);
        else embed_fwd_launch<T, int32_t>((const int32_t*)ids, N, (const T*)weight, V, D, scale, (T*)out, s);
    });
    return check_launch("slg_embed_fwd");
}

extern "C" int64_t slg_embed_bwd_workspace_bytes(int64_t N, int64_t V, int64_t D, int32_t dtype) {
    if (N < 0 || V <= 0 || D <= 0) return 0;
    return embed_plan(N, V, D, dtype == SLG_DT_F32 ? 4 : 2).bytes;
}

extern "C" int slg_embed_bwd(const void* ids, int32_t ids64, int64_t N, const void* g, int32_t dtype, int64_t V,
                             int64_t D, float scale, int64_t padding_idx, void* gw, void* workspace,
                             int64_t workspace_bytes, void* stream) {
    int st = check_embed(N, V, D, ids64, dtype, "slg_embed_bwd");
    if (st) return st;
    if ((N > 0 && (!ids || !g)) || !gw || !workspace) return set_error(SLG_ERR_ARG, "slg_embed_bwd: null pointer");
    if (!aligned16(workspace)) return set_error(SLG_ERR_ALIGN, "slg_embed_bwd: workspace not 16-byte aligned");
    const EmbedPlan p = embed_plan(N, V, D, dtype == SLG_DT_F32 ? 4 : 2);
    if (workspace_bytes < p.bytes)
        return set_error(SLG_ERR_WORKSPACE, "slg_embed_bwd: workspace %lld < %lld bytes", (long long)workspace_bytes,
                         (long long)p.bytes);
    cudaStream_t s = as_stream(stream);
    char* ws = static_cast<char*>(workspace);
    const uint32_t* key = reinterpret_cast<const uint32_t*>(ws);
    if (N > 0)
        key = ids64 ? embed_sort((const int64_t*)ids, N, V, padding_idx, p, ws, s)
                    : embed_sort((const int32_t*)ids, N, V, padding_idx, p, ws, s);
    for_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        embed_bwd_launch<T>(key, N, V, D, (const T*)g, scale, (T*)gw, p, ws, s);
    });
    return check_launch("slg_embed_bwd");
}
