// One step of beam search: selection over beams and vocabulary, and the reordering of the
// decoder's state by the chosen beams.
//
//   l[b, v] = (x[b, v] - m_b) - log sum_u exp(x[b, u] - m_b) + S_b,    m_b = max_u x[b, u]
// and the `width` largest l of an entry's beams, equal values by the lowest b V + v.  A
// finished beam has the one candidate (b, eos) at its own score.  Masked logits (-inf, or
// NaN) are never chosen while another candidate is left; +inf counts as the largest finite
// value.  (x - m) - log s keeps rows apart whose logits are huge or at the type's lowest value.
#include "token_common.cuh"

namespace slg {

constexpr int BM_THREADS = 256;
constexpr int BM_WARPS = BM_THREADS / 32;
constexpr int BM_MAX = SLG_BEAM_MAX;
constexpr float BM_LARGEST = 3.402823466e+38f;

// candidate order: larger value first, then the lower index
__device__ __forceinline__ bool ahead(float v, int64_t i, float w, int64_t j) { return v > w || (v == w && i < j); }

__device__ __forceinline__ float clean(float v) { return v != v ? -CUDART_INF_F : fminf(v, BM_LARGEST); }

struct Cand { float v; int32_t i; };
constexpr int32_t NO_INDEX = 0x7fffffff;

__device__ __forceinline__ Cand warp_best(Cand c) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float v = __shfl_xor_sync(0xffffffffu, c.v, o);
        const int32_t i = __shfl_xor_sync(0xffffffffu, c.i, o);
        if (ahead(v, i, c.v, c.i)) { c.v = v; c.i = i; }
    }
    return c;
}

// One CTA = one beam: its `width` best tokens, in order.
template <typename T>
__global__ void __launch_bounds__(BM_THREADS)
beam_row_kernel(const T* __restrict__ x, int64_t V, int64_t ldx, const float* __restrict__ scores,
                const uint8_t* __restrict__ finished, int32_t eos, int width, float* __restrict__ val,
                int32_t* __restrict__ tok) {
    __shared__ float red[BM_WARPS];
    __shared__ Cand best[BM_WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row = blockIdx.x;
    const T* p = x + row * ldx;
    const float S = scores[row];
    const bool done = finished && finished[row];
    float m = -CUDART_INF_F, logs = 0.0f;
    if (!done) {
        for (int64_t v = threadIdx.x; v < V; v += BM_THREADS) m = fmaxf(m, clean(to_f32(p[v])));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (lane == 0) red[warp] = m;
        __syncthreads();
        for (int q = 0; q < BM_WARPS; ++q) m = fmaxf(m, red[q]);
        __syncthreads();
        float s = 0.0f;
        if (m > -CUDART_INF_F)
            for (int64_t v = threadIdx.x; v < V; v += BM_THREADS) s += expf(clean(to_f32(p[v])) - m);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) red[warp] = s;
        __syncthreads();
        s = 0.0f;
        for (int q = 0; q < BM_WARPS; ++q) s += red[q];
        logs = logf(s);
    }
    auto value = [&](int64_t v) {
        float l = -CUDART_INF_F;
        if (done) l = v == eos ? S : l;
        else if (m > -CUDART_INF_F) l = (clean(to_f32(p[v])) - m) - logs + S;
        return l != l ? -CUDART_INF_F : l;
    };
    Cand last = {CUDART_INF_F, -1};
    for (int n = 0; n < width; ++n) {
        Cand c = {-CUDART_INF_F, NO_INDEX};
        for (int64_t v = threadIdx.x; v < V; v += BM_THREADS) {
            const float l = value(v);
            if (ahead(last.v, last.i, l, v) && ahead(l, v, c.v, c.i)) c = {l, (int32_t)v};
        }
        c = warp_best(c);
        __syncthreads();
        if (lane == 0) best[warp] = c;
        __syncthreads();
        for (int q = 0; q < BM_WARPS; ++q)
            if (ahead(best[q].v, best[q].i, c.v, c.i)) c = best[q];
        last = c;
        if (threadIdx.x == 0) { val[row * width + n] = c.v; tok[row * width + n] = c.i; }
    }
}

// One warp = one entry: the best of its beams' lists, which are in order.
__global__ void beam_join_kernel(const float* __restrict__ val, const int32_t* __restrict__ tok, int64_t B, int beams,
                                 int64_t V, int width, const uint8_t* __restrict__ finished, int32_t eos,
                                 float* __restrict__ scores, int64_t* __restrict__ parents,
                                 int64_t* __restrict__ tokens, uint8_t* __restrict__ done) {
    const int lane = threadIdx.x & 31;
    const int64_t b = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (b >= B) return;
    int at = 0;                                             // lane = beam: its next candidate
    for (int n = 0; n < width; ++n) {
        float v = -CUDART_INF_F;
        int64_t i = INT64_MAX;
        if (lane < beams && at < width) {
            const int64_t q = ((int64_t)b * beams + lane) * width + at;
            v = val[q];
            if (tok[q] != NO_INDEX) i = lane * V + tok[q];
        }
        float bv = v;
        int64_t bi = i;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
            const int64_t oi = __shfl_xor_sync(0xffffffffu, bi, o);
            if (ahead(ov, oi, bv, bi)) { bv = ov; bi = oi; }
        }
        if (bi == i && i != INT64_MAX) {
            ++at;
            const int64_t t = i - lane * V;
            scores[b * width + n] = v;
            parents[b * width + n] = lane;
            tokens[b * width + n] = t;
            if (done) done[b * width + n] = (finished && finished[b * beams + lane]) || t == eos;
        }
    }
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

// Column r of every feature row = column (r / width) * beams + parents[r]; padding columns 0.
__global__ void reorder_features_kernel(const float* __restrict__ in, int64_t F, int64_t ldi, int64_t n,
                                        const int64_t* __restrict__ parents, int beams, int width,
                                        float* __restrict__ out, int64_t ldo) {
    const int64_t r = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (r >= ldo) return;
    int64_t src = -1;
    if (r < n) {
        const int64_t p = parents[r];
        src = (r / width) * beams + (p >= 0 && p < beams ? p : 0);
    }
    for (int64_t f = blockIdx.y; f < F; f += gridDim.y) out[f * ldo + r] = src >= 0 ? in[f * ldi + src] : 0.0f;
}

// The same on bits: bit r of every packed row; a warp builds 32 samples of a row by ballot.
__global__ void reorder_packed_kernel(const uint32_t* __restrict__ in, int64_t F, int64_t ldi, int64_t n,
                                      const int64_t* __restrict__ parents, int beams, int width,
                                      uint32_t* __restrict__ out, int64_t ldo) {
    const int lane = threadIdx.x & 31;
    const int64_t w = blockIdx.x;                           // 32-bit word of the output rows
    const int64_t r = w * 32 + lane;
    int64_t src = -1;
    if (r < n) {
        const int64_t p = parents[r];
        src = (r / width) * beams + (p >= 0 && p < beams ? p : 0);
    }
    const int warps = blockDim.x >> 5;
    for (int64_t f = (int64_t)blockIdx.y * warps + (threadIdx.x >> 5); f < F; f += (int64_t)gridDim.y * warps) {
        const bool bit = src >= 0 && ((in[f * ldi + (src >> 5)] >> (src & 31)) & 1u);
        const uint32_t word = __ballot_sync(0xffffffffu, bit);
        if (lane == 0) out[f * ldo + w] = word;
    }
}

}  // namespace slg

using namespace slg;

extern "C" int64_t slg_beam_step_workspace_bytes(int64_t B, int32_t beams, int64_t V, int32_t width) {
    (void)V;
    if (B <= 0 || beams <= 0 || width <= 0) return 0;
    return B * beams * width * 8;
}

extern "C" int slg_beam_step(const void* logits, int32_t dtype, int64_t B, int32_t beams, int64_t V, int64_t ldx,
                             const float* scores, const uint8_t* finished, int32_t eos, int32_t width,
                             float* out_scores, int64_t* parents, int64_t* tokens, uint8_t* out_finished,
                             void* workspace, int64_t workspace_bytes, void* stream) {
    const char* name = "slg_beam_step";
    if (B < 0 || beams <= 0 || V <= 0 || width <= 0) return set_error(SLG_ERR_ARG, "%s: bad sizes", name);
    if (beams > BM_MAX || width > BM_MAX)
        return set_error(SLG_ERR_UNSUPPORTED, "%s: at most %d beams", name, BM_MAX);
    if (V >= (1ll << 31) - 1) return set_error(SLG_ERR_UNSUPPORTED, "%s: vocabulary must be below 2^31 - 1", name);
    if (width > beams * V) return set_error(SLG_ERR_ARG, "%s: width %d > beams * vocabulary", name, width);
    if (ldx < V) return set_error(SLG_ERR_ARG, "%s: ldx < vocabulary", name);
    if (finished && (eos < 0 || eos >= V)) return set_error(SLG_ERR_ARG, "%s: finished needs eos in the vocabulary", name);
    if (dtype != SLG_DT_F32 && dtype != SLG_DT_BF16 && dtype != SLG_DT_F16)
        return set_error(SLG_ERR_UNSUPPORTED, "%s: dtype %d not built", name, dtype);
    if (B * beams >= (1ll << 31)) return set_error(SLG_ERR_ARG, "%s: batch too large", name);
    if (B == 0) return SLG_OK;
    if (!logits || !scores || !out_scores || !parents || !tokens || !workspace)
        return set_error(SLG_ERR_ARG, "%s: null pointer", name);
    const int64_t need = slg_beam_step_workspace_bytes(B, beams, V, width);
    if (workspace_bytes < need)
        return set_error(SLG_ERR_WORKSPACE, "%s: workspace %lld < %lld bytes", name, (long long)workspace_bytes,
                         (long long)need);
    cudaStream_t s = as_stream(stream);
    float* val = static_cast<float*>(workspace);
    int32_t* tok = reinterpret_cast<int32_t*>(val + B * beams * width);
    for_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        beam_row_kernel<T><<<(unsigned)(B * beams), BM_THREADS, 0, s>>>((const T*)logits, V, ldx, scores, finished,
                                                                       eos, width, val, tok);
    });
    beam_join_kernel<<<(unsigned)cdiv(B, 4), 128, 0, s>>>(val, tok, B, beams, V, width, finished, eos, out_scores,
                                                          parents, tokens, out_finished);
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
    const dim3 grid((unsigned)cdiv(ldo, 128), (unsigned)std::min<int64_t>(F, 8192));
    reorder_features_kernel<<<grid, 128, 0, as_stream(stream)>>>(in, F, ldi, B * width, parents, beams, width, out, ldo);
    return check_launch("slg_beam_reorder_features");
}

extern "C" int slg_beam_reorder_packed(const uint64_t* in, int64_t F, int64_t ldi, const int64_t* parents, int64_t B,
                                       int32_t beams, int32_t width, uint64_t* out, int64_t ldo, void* stream) {
    if (F == 0 || B == 0) return SLG_OK;
    int st = check_reorder(in, parents, out, B, beams, width, "slg_beam_reorder_packed");
    if (st) return st;
    if (F < 0 || ldi * 64 < B * beams || ldo * 64 < B * width)
        return set_error(SLG_ERR_ARG, "slg_beam_reorder_packed: bad sizes");
    const dim3 grid((unsigned)(2 * ldo), (unsigned)std::min<int64_t>(cdiv(F, 8), 4096));
    reorder_packed_kernel<<<grid, 256, 0, as_stream(stream)>>>(reinterpret_cast<const uint32_t*>(in), F, 2 * ldi,
                                                               B * width, parents, beams, width,
                                                               reinterpret_cast<uint32_t*>(out), 2 * ldo);
    return check_launch("slg_beam_reorder_packed");
}
