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
// One thread = EM_UNROLL 16-byte vectors of the output.  VEC: rows are whole vectors (`per` of
// them); otherwise a vector may cross rows and its values are read one by one.  Below 2^32
// vectors (S = uint32_t) the row of a vector is one 32-bit division: with the 64-bit one the
// divisions took longer than the copy (262,144 bf16 rows of 1,024: 123 us against 109).
template <typename T, typename I, typename S, bool VEC>
__global__ void __launch_bounds__(EM_THREADS)
embed_fwd_kernel(const I* __restrict__ ids, int64_t N, const T* __restrict__ w, int64_t V, int64_t D,
                 S per, float scale, T* __restrict__ y) {
    constexpr int E = Pack16<T>::E;
    const S first = (S)blockIdx.x * (EM_THREADS * EM_UNROLL) + threadIdx.x;
    if constexpr (VEC) {
        const S total = (S)N * per;
        uint4 u[EM_UNROLL];
        bool ok[EM_UNROLL];
#pragma unroll
        for (int q = 0; q < EM_UNROLL; ++q) {
            const S k = first + q * EM_THREADS;
            ok[q] = false;
            u[q] = make_uint4(0, 0, 0, 0);
            if (k < total) {
                const S i = k / per, c = k - i * per;
                const int64_t t = (int64_t)ids[i];
                ok[q] = t >= 0 && t < V;
                if (ok[q]) u[q] = __ldg(reinterpret_cast<const uint4*>(w + t * D) + c);
            }
        }
#pragma unroll
        for (int q = 0; q < EM_UNROLL; ++q) {
            const S k = first + q * EM_THREADS;
            if (k >= total) continue;
            float v[E];
            unpack16<T>(u[q], v);
#pragma unroll
            for (int j = 0; j < E; ++j) v[j] = ok[q] ? v[j] * scale : CUDART_NAN_F;
            __stcs(reinterpret_cast<uint4*>(y) + k, pack16<T>(v));
        }
    } else {
        const int64_t total = N * D;
#pragma unroll
        for (int q = 0; q < EM_UNROLL; ++q) {
            const int64_t e0 = (int64_t)(first + q * EM_THREADS) * E;
            if (e0 >= total) continue;
            int64_t i = total < (1ll << 32) ? (int64_t)((uint32_t)e0 / (uint32_t)D) : e0 / D, c = e0 - i * D;
            int64_t t = (int64_t)ids[i];
            float v[E];
#pragma unroll
            for (int j = 0; j < E; ++j) {
                v[j] = e0 + j >= total ? 0.0f : t >= 0 && t < V ? to_f32(w[t * D + c]) * scale : CUDART_NAN_F;
                if (++c == D && e0 + j + 1 < total) { c = 0; t = (int64_t)ids[++i]; }
            }
            if (e0 + E <= total) *reinterpret_cast<uint4*>(y + e0) = pack16<T>(v);
            else
#pragma unroll
                for (int j = 0; j < E; ++j)
                    if (e0 + j < total) y[e0 + j] = from_f32<T>(v[j]);
        }
    }
}

// Rows of at least 32 vectors: a warp copies a row, so there is nothing to divide and the id
// is read once (262,144 bf16 rows of 1,024: 83 instructions a vector above, 109 us).
template <typename T, typename I>
__global__ void __launch_bounds__(EM_THREADS)
embed_fwd_rows_kernel(const I* __restrict__ ids, int64_t N, const T* __restrict__ w, int64_t V, int per, float scale,
                      T* __restrict__ y) {
    constexpr int E = Pack16<T>::E;
    const int lane = threadIdx.x & 31;
    const int64_t i = (int64_t)blockIdx.x * (EM_THREADS / 32) + (threadIdx.x >> 5);
    if (i >= N) return;
    const int64_t t = (int64_t)ids[i];
    const bool ok = t >= 0 && t < V;
    const uint4* src = reinterpret_cast<const uint4*>(w) + (ok ? t : 0) * per;
    uint4* dst = reinterpret_cast<uint4*>(y) + i * per;
    for (int c0 = 0; c0 < per; c0 += 32 * EM_UNROLL) {
        uint4 u[EM_UNROLL];
#pragma unroll
        for (int q = 0; q < EM_UNROLL; ++q) {
            const int c = c0 + q * 32 + lane;
            u[q] = ok && c < per ? __ldg(src + c) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int q = 0; q < EM_UNROLL; ++q) {
            const int c = c0 + q * 32 + lane;
            float v[E];
            unpack16<T>(u[q], v);
#pragma unroll
            for (int j = 0; j < E; ++j) v[j] = ok ? v[j] * scale : CUDART_NAN_F;
            if (c < per) __stcs(dst + c, pack16<T>(v));
        }
    }
}

// -------------------------------------------------------------------- sort
// Tokens that get no gradient (padding, out of range) carry the key V and sort past every
// row.  Up to RK_MAX tokens every token counts the tokens before it in sorted order (N^2
// comparisons, one launch); above, a stable LSD radix sort of (token, position) with digits
// of at most 9 bits, so two passes (four launches) sort vocabularies below 2^18.
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

constexpr int RK_MAX = 8192;            // 13 us there; the radix sort's four launches take 21 up to 16,384
constexpr int RK_THREADS = 256;
constexpr int RK_WARPS = RK_THREADS / 32;

// A CTA ranks 32 tokens (one per lane), each warp against its eighth of the batch: tokens
// at earlier positions count when they are <= its own, later ones when they are <.
template <typename I>
__global__ void __launch_bounds__(RK_THREADS)
rank_sort_kernel(KeysOfIds<I> src, int N, uint32_t* __restrict__ ko, uint32_t* __restrict__ po, int32_t* __restrict__ zero) {
    __shared__ alignas(16) uint32_t key[RK_MAX];
    __shared__ int part[RK_WARPS][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n4 = (N + 3) & ~3;
    if (blockIdx.x == 0 && threadIdx.x < 2) zero[threadIdx.x] = 0;
    for (int i = threadIdx.x; i < n4; i += RK_THREADS) key[i] = i < N ? src.key(i) : 0xffffffffu;
    __syncthreads();
    const int i0 = blockIdx.x * 32, i = i0 + lane;
    const uint32_t mine = i < N ? key[i] : 0u;
    const int a = n4 / 4 * warp / RK_WARPS, b = n4 / 4 * (warp + 1) / RK_WARPS;    // groups of 4 keys
    const uint4* k4 = reinterpret_cast<const uint4*>(key);
    int rank = 0;
    const int lo = min(max(i0 / 4, a), b), hi = min(max(i0 / 4 + 8, a), b);        // the CTA's own tokens
#pragma unroll 4
    for (int g = a; g < lo; ++g) {
        const uint4 k = k4[g];
        rank += (k.x <= mine) + (k.y <= mine) + (k.z <= mine) + (k.w <= mine);
    }
    for (int g = lo; g < hi; ++g)
        for (int j = 4 * g; j < 4 * g + 4; ++j) rank += key[j] < mine || (key[j] == mine && j < i);
#pragma unroll 4
    for (int g = hi; g < b; ++g) {
        const uint4 k = k4[g];
        rank += (k.x < mine) + (k.y < mine) + (k.z < mine) + (k.w < mine);
    }
    part[warp][lane] = rank;
    __syncthreads();
    if (warp == 0 && i < N) {
        int at = 0;
#pragma unroll
        for (int w = 0; w < RK_WARPS; ++w) at += part[w][lane];
        ko[at] = mine;
        po[at] = (uint32_t)i;
    }
}

constexpr int RS_THREADS = 512;
constexpr int RS_WARPS = RS_THREADS / 32;
constexpr int RS_PER = 4;                           // keys per thread of a tile
constexpr int RS_TILE = RS_THREADS * RS_PER;
constexpr int RS_BITS = 9;
constexpr int RS_BINS = 1 << RS_BITS;               // one per thread
constexpr int RS_MAX_TILES = 128;

__host__ __device__ inline int64_t rs_span(int64_t N) {   // keys per CTA: whole tiles, at most RS_MAX_TILES CTAs
    return RS_TILE * cdiv(cdiv(N, RS_TILE), RS_MAX_TILES);
}

// hist[cta][digit]
template <typename S>
__global__ void __launch_bounds__(RS_THREADS)
radix_count_kernel(S src, int64_t N, int64_t span, int shift, uint32_t mask, uint32_t* __restrict__ hist,
                   int32_t* __restrict__ zero) {
    __shared__ uint32_t h[RS_BINS];
    if (blockIdx.x == 0 && threadIdx.x < 2) zero[threadIdx.x] = 0;
    h[threadIdx.x] = 0;
    __syncthreads();
    const int64_t a = (int64_t)blockIdx.x * span, b = a + span < N ? a + span : N;
#pragma unroll 4
    for (int64_t i = a + threadIdx.x; i < b; i += RS_THREADS) atomicAdd(&h[(src.key(i) >> shift) & mask], 1u);
    __syncthreads();
    hist[(int64_t)blockIdx.x * RS_BINS + threadIdx.x] = h[threadIdx.x];
}

// Thread d owns digit d.  Its first slot is the number of keys with a smaller digit plus
// those with digit d in earlier CTAs; inside a tile a warp owns consecutive keys, ranks
// them 32 at a time among the lanes with the same digit (one ballot per bit: match_any is
// several times slower on 32 different digits), and warps follow one another: the order is stable.
template <typename S>
__global__ void __launch_bounds__(RS_THREADS)
radix_scatter_kernel(S src, int64_t N, int64_t span, int shift, int bits, const uint32_t* __restrict__ hist,
                     uint32_t* __restrict__ ko, uint32_t* __restrict__ po) {
    __shared__ uint32_t base[RS_BINS];
    __shared__ uint32_t cnt[RS_WARPS][RS_BINS];
    __shared__ uint32_t wsum[RS_WARPS];
    const int d = threadIdx.x, warp = d >> 5, lane = d & 31;
    const uint32_t mask = (1u << bits) - 1u;
    const int64_t a = (int64_t)blockIdx.x * span, b = a + span < N ? a + span : N;
    uint32_t key[RS_PER], pos[RS_PER];
    auto load = [&](int64_t w0) {
#pragma unroll
        for (int j = 0; j < RS_PER; ++j) {
            const bool on = w0 + 32 * j < b;
            key[j] = on ? src.key(w0 + 32 * j) : 0u;
            pos[j] = on ? src.pos(w0 + 32 * j) : 0u;
        }
    };
    load(a + warp * (32 * RS_PER) + lane);
    uint32_t before = 0, all = 0;
    for (int t0 = 0; t0 < (int)gridDim.x; t0 += 32) {      // 32 loads at a time: this is latency
        uint32_t c[32];
#pragma unroll
        for (int q = 0; q < 32; ++q) c[q] = t0 + q < (int)gridDim.x ? __ldg(&hist[(int64_t)(t0 + q) * RS_BINS + d]) : 0u;
#pragma unroll
        for (int q = 0; q < 32; ++q) {
            before += t0 + q < (int)blockIdx.x ? c[q] : 0u;
            all += c[q];
        }
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

    for (int64_t t0 = a; t0 < b; t0 += RS_TILE) {
        const int64_t w0 = t0 + warp * (32 * RS_PER) + lane;
        if (t0 > a) load(w0);
#pragma unroll
        for (int q = 0; q < RS_WARPS; ++q) cnt[q][d] = 0;
        __syncthreads();
        uint32_t rank[RS_PER], peers[RS_PER];
#pragma unroll
        for (int j = 0; j < RS_PER; ++j) {
            uint32_t p = __ballot_sync(0xffffffffu, w0 + 32 * j < b);
            for (int q = 0; q < bits; ++q) {
                const bool one = key[j] >> (shift + q) & 1u;
                const uint32_t v = __ballot_sync(0xffffffffu, one);
                p &= one ? v : ~v;
            }
            peers[j] = p;
        }
#pragma unroll
        for (int j = 0; j < RS_PER; ++j) {
            const bool on = w0 + 32 * j < b;
            const uint32_t dg = (key[j] >> shift) & mask;
            rank[j] = __popc(peers[j] & ((1u << lane) - 1u)) + (on ? cnt[warp][dg] : 0u);
            __syncwarp();
            if (on && (peers[j] >> lane) == 1u) cnt[warp][dg] += __popc(peers[j]);    // the last of them
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
                const uint32_t o = cnt[warp][(key[j] >> shift) & mask] + rank[j];
                ko[o] = key[j];
                po[o] = pos[j];
            }
        __syncthreads();
    }
}

// ------------------------------------------------------------ segmented sum
// The sorted tokens and the row ends 0 .. V-1 are merged into one list of V + N items (a
// row's end comes after its tokens), and the list is cut into equal chunks: an entry costs
// a read of D values, a row end a write of D values, so every chunk costs the same
// whatever the tokens' distribution.  A row whose items lie in one chunk is written there.  A row
// that is cut leaves its sums in carry rows: `tail` (the row goes on in the next chunk) and
// `head` (it ends here, begun earlier); embed_join_kernel adds those in chunk order.
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

// carry rows are fp32 and padded to whole slices, so no column check
template <int E, bool VEC>
__device__ __forceinline__ void store_carry(float* __restrict__ p, int lane, const float (&acc)[E]) {
    if constexpr (VEC) {
#pragma unroll
        for (int j = 0; j < E; j += 4)
            *reinterpret_cast<float4*>(p + lane * E + j) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
    } else {
#pragma unroll
        for (int j = 0; j < E; ++j) p[lane + 32 * j] = acc[j];
    }
}

constexpr int SG_WARPS = 4;
constexpr int SG_UNROLL = 8;
constexpr int SG_CHUNK = 128;       // largest chunk
constexpr int JN_WARPS = 8;
constexpr int JN_SHORT = 8;

// head_row[chunk] = row that ends in this chunk but began earlier; cuts: the lists of such
// chunks, in any order -- every one is joined by itself -- those of long rows from the end
// backwards, with their lengths in cut_count; start[row] = chunk with the row's first entry.
template <typename T, bool VEC>
__global__ void __launch_bounds__(SG_WARPS * 32)
embed_sum_kernel(const uint32_t* __restrict__ key, const uint32_t* __restrict__ pos, int64_t N, int64_t V,
                 int64_t D, int64_t chunk, const T* __restrict__ g, float scale, T* __restrict__ gw,
                 float* __restrict__ carry, int64_t slices, int32_t* __restrict__ head_row, int32_t* __restrict__ start,
                 int32_t* __restrict__ cuts, int32_t* __restrict__ cut_count) {
    constexpr int E = Pack16<T>::E;
    constexpr int SLICE = 32 * E;
    __shared__ Cut cut[2];
    __shared__ uint32_t skey[SG_CHUNK], spos[SG_CHUNK];
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
    int n = (int)(cut[1].i - i0);                       // the chunk's entries: at most SG_CHUNK
    for (int i = threadIdx.x; i < n; i += SG_WARPS * 32) {
        skey[i] = key[i0 + i];
        spos[i] = pos[i0 + i];
    }
    const bool begun = r0 < V && i0 > 0 && (int64_t)key[i0 - 1] == r0;      // r0 has entries in earlier chunks
    __syncthreads();
    const bool open = r1 < V && n > 0 && (int64_t)skey[n - 1] == r1;        // r1 goes on in the next one
    if (threadIdx.x == 0 && blockIdx.y == 0) {
        if (begun && r1 > r0) {
            head_row[c] = (int32_t)r0;
            // long: the row also fills the JN_SHORT chunks before this one
            const int64_t back = i0 - 1 - (JN_SHORT * chunk);
            const bool lengthy = back >= 0 && (int64_t)key[back] == r0;
            const int32_t at = atomicAdd(&cut_count[lengthy], 1);
            cuts[lengthy ? gridDim.x - 1 - at : at] = (int32_t)c;
        }
        if (open && !(begun && r1 == r0)) start[r1] = (int32_t)c;
    }
    if (r1 == V) {                      // what follows the last row's end has no gradient
        while (n > 0 && (int64_t)skey[n - 1] >= V) --n;
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
                if (r == r0 && begun) store_carry<E, VEC>(head, lane, acc);
                else store_row<T, VEC>(gw + r * D, c0, D, lane, scale, acc);
#pragma unroll
                for (int j = 0; j < E; ++j) acc[j] = 0.0f;
            }
        };
        for (int i = 0; i < n; i += SG_UNROLL) {
            Cols<T, VEC> v[SG_UNROLL];
#pragma unroll
            for (int u = 0; u < SG_UNROLL; ++u)
                if (i + u < n) v[u].load(g + (int64_t)spos[i + u] * D, c0, D, lane);
#pragma unroll
            for (int u = 0; u < SG_UNROLL; ++u) {
                if (i + u >= n) break;
                end_rows((int64_t)skey[i + u]);
                v[u].add_to(acc);
            }
        }
        end_rows(r1);
        if (open) store_carry<E, VEC>(tail, lane, acc);
    }
}

// Joins the cut rows, 128 columns at a time.  Short rows: a warp adds the row's tails, then
// its head.  Long ones (a frequent token's row is cut into hundreds of chunks): a CTA's
// warps take equal runs of the tails, joined in shared memory.
template <typename T, bool VEC>
__global__ void __launch_bounds__(JN_WARPS * 32)
embed_join_kernel(int64_t D, float scale, T* __restrict__ gw, const float* __restrict__ carry, int64_t ldc,
                  const int32_t* __restrict__ head_row, const int32_t* __restrict__ start,
                  const int32_t* __restrict__ cuts, const int32_t* __restrict__ cut_count, int64_t nchunk) {
    __shared__ float4 part[JN_WARPS][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t shorts = cut_count[0], longs = cut_count[1];
    int64_t c = 0, r = 0, first = 0;
    const int64_t groups = ldc / 128;
    auto sum = [&](int64_t g, int64_t a, int64_t b) {           // tails of chunks first+a .. first+b-1
        const float4* p = reinterpret_cast<const float4*>(carry + (2 * (first + a) + 1) * ldc + g * 128) + lane;
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int64_t q = a; q < b; q += 8, p += 8 * (ldc / 2)) {
            float4 v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = q + u < b ? __ldg(p + (int64_t)u * (ldc / 2)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int u = 0; u < 8; ++u) { s.x += v[u].x; s.y += v[u].y; s.z += v[u].z; s.w += v[u].w; }
        }
        return s;
    };
    auto finish = [&](int64_t g, float4 s) {
        const float4 h = *(reinterpret_cast<const float4*>(carry + 2 * c * ldc + g * 128) + lane);
        const float v[4] = {(s.x + h.x) * scale, (s.y + h.y) * scale, (s.z + h.z) * scale, (s.w + h.w) * scale};
        const int64_t col = g * 128 + lane * 4;
        T* o = gw + r * D + col;
        if (VEC && col + 4 <= D) {
            if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
            else *reinterpret_cast<uint2*>(o) = make_uint2(pack2<T>(v), pack2<T>(v + 2));
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (col + j < D) o[j] = from_f32<T>(v[j]);
        }
    };
    auto pick = [&](int64_t at) {
        c = cuts[at];
        r = head_row[c];
        first = start[r];
    };
    for (int64_t i = blockIdx.x; i < longs * groups; i += gridDim.x) {
        const int64_t e = i / groups, g = i - e * groups;
        pick(nchunk - 1 - e);
        const int64_t n = c - first;
        part[warp][lane] = sum(g, n * warp / JN_WARPS, n * (warp + 1) / JN_WARPS);
        __syncthreads();
        if (warp == 0) {
            float4 s = part[0][lane];
#pragma unroll
            for (int w = 1; w < JN_WARPS; ++w) {
                const float4 v = part[w][lane];
                s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
            }
            finish(g, s);
        }
        __syncthreads();
    }
    for (int64_t i = (int64_t)blockIdx.x * JN_WARPS + warp; i < shorts * groups; i += (int64_t)gridDim.x * JN_WARPS) {
        const int64_t e = i / groups, g = i - e * groups;
        pick(e);
        finish(g, sum(g, 0, c - first));
    }
}

// ------------------------------------------------------------------- plans
struct EmbedPlan {
    int64_t hist_at, head_at, cuts_at, start_at, carry_at, bytes;
    int64_t chunk, nchunk, slices, tiles;
    int passes, bits;
};

static int bits_of(uint64_t v) { int n = 0; while (v) { ++n; v >>= 1; } return n; }

static EmbedPlan embed_plan(int64_t N, int64_t V, int64_t D, int es) {
    EmbedPlan p;
    auto up = [](int64_t v) { return cdiv(v, 256) * 256; };
    p.tiles = N > RK_MAX ? cdiv(N, rs_span(N)) : 0;
    const int bits = bits_of((uint64_t)V);                  // keys 0 .. V
    p.passes = (bits + RS_BITS - 1) / RS_BITS;
    p.bits = (bits + p.passes - 1) / p.passes;
    p.slices = cdiv(D * es, 512);                           // 32 lanes x 16 bytes
    // about 16 chunks per SM, between 16 items (a chunk costs two searches) and 128
    p.chunk = 16;
    while (p.chunk < SG_CHUNK && (V + N) / p.chunk > 148 * 16) p.chunk *= 2;
    p.nchunk = cdiv(V + N, p.chunk);
    p.hist_at = up(4 * 4 * N);                              // two (token, position) buffers
    p.head_at = p.hist_at + up(p.tiles * RS_BINS * 4);
    p.cuts_at = p.head_at + up(p.nchunk * 4);               // lists of cut rows, then their two lengths
    p.start_at = p.cuts_at + up(p.nchunk * 4 + 8);
    p.carry_at = p.start_at + up(V * 4);
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
    constexpr int E = Pack16<T>::E;
    const int64_t vecs = cdiv(N * D, E);
    const unsigned grid = (unsigned)cdiv(vecs, EM_THREADS * EM_UNROLL);
    if (D % E || !aligned16(w))
        embed_fwd_kernel<T, I, int64_t, false><<<grid, EM_THREADS, 0, st>>>(ids, N, w, V, D, 0, scale, y);
    else if (D / E >= 32 && D / E < (1ll << 31))
        embed_fwd_rows_kernel<T, I><<<(unsigned)cdiv(N, EM_THREADS / 32), EM_THREADS, 0, st>>>(ids, N, w, V, (int)(D / E),
                                                                                               scale, y);
    else if (vecs + EM_THREADS * EM_UNROLL < (1ll << 32))
        embed_fwd_kernel<T, I, uint32_t, true><<<grid, EM_THREADS, 0, st>>>(ids, N, w, V, D, (uint32_t)(D / E), scale, y);
    else
        embed_fwd_kernel<T, I, int64_t, true><<<grid, EM_THREADS, 0, st>>>(ids, N, w, V, D, D / E, scale, y);
}

// sorted tokens, followed by their positions (at + N)
template <typename I>
static const uint32_t* embed_sort(const I* ids, int64_t N, int64_t V, int64_t pad, const EmbedPlan& p, char* ws,
                                  cudaStream_t st) {
    int32_t* zero = reinterpret_cast<int32_t*>(ws + p.cuts_at) + p.nchunk;
    uint32_t* buf[2] = {reinterpret_cast<uint32_t*>(ws), reinterpret_cast<uint32_t*>(ws) + 2 * N};
    const KeysOfIds<I> in{ids, V, pad};
    if (N <= RK_MAX) {
        rank_sort_kernel<I><<<(unsigned)cdiv(N, 32), RK_THREADS, 0, st>>>(in, (int)N, buf[0], buf[0] + N, zero);
        return buf[0];
    }
    uint32_t* hist = reinterpret_cast<uint32_t*>(ws + p.hist_at);
    const int64_t span = rs_span(N);
    const unsigned grid = (unsigned)p.tiles;
    const uint32_t mask = (1u << p.bits) - 1u;
    uint32_t* src = nullptr;
    for (int q = 0; q < p.passes; ++q) {
        uint32_t* dst = buf[q & 1];
        if (q == 0) {
            radix_count_kernel<<<grid, RS_THREADS, 0, st>>>(in, N, span, 0, mask, hist, zero);
            radix_scatter_kernel<<<grid, RS_THREADS, 0, st>>>(in, N, span, 0, p.bits, hist, dst, dst + N);
        } else {
            const KeysOfPairs pairs{src, src + N};
            radix_count_kernel<<<grid, RS_THREADS, 0, st>>>(pairs, N, span, p.bits * q, mask, hist, zero);
            radix_scatter_kernel<<<grid, RS_THREADS, 0, st>>>(pairs, N, span, p.bits * q, p.bits, hist, dst, dst + N);
        }
        src = dst;
    }
    return src;
}

template <typename T>
static void embed_bwd_launch(const uint32_t* key, int64_t N, int64_t V, int64_t D, const T* g, float scale, T* gw,
                             const EmbedPlan& p, char* ws, cudaStream_t st) {
    constexpr int E = Pack16<T>::E;
    float* carry = reinterpret_cast<float*>(ws + p.carry_at);
    int32_t* head = reinterpret_cast<int32_t*>(ws + p.head_at);
    int32_t* start = reinterpret_cast<int32_t*>(ws + p.start_at);
    int32_t* cuts = reinterpret_cast<int32_t*>(ws + p.cuts_at);
    int32_t* count = cuts + p.nchunk;
    const dim3 grid((unsigned)p.nchunk, (unsigned)std::min<int64_t>(cdiv(p.slices, SG_WARPS), 65535));
    const int64_t ldc = p.slices * 32 * E;
    const unsigned jgrid = (unsigned)std::min<int64_t>(cdiv(p.nchunk * (ldc / 128), JN_WARPS), 4 * sm_count());
    auto go = [&](auto vec) {
        constexpr bool VEC = decltype(vec)::value;
        embed_sum_kernel<T, VEC><<<grid, SG_WARPS * 32, 0, st>>>(key, key + N, N, V, D, p.chunk, g, scale, gw, carry,
                                                                 p.slices, head, start, cuts, count);
        if (N > 0)
            embed_join_kernel<T, VEC><<<jgrid, JN_WARPS * 32, 0, st>>>(D, scale, gw, carry, ldc, head, start, cuts, count, p.nchunk);
    };
    if (D % E == 0 && aligned16(g) && aligned16(gw)) go(std::true_type{});
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
