// Activation checkpoints in 8 bits.
//
// A row of activations is cut into blocks of 128 columns.  A block keeps lo = min and
// step = (max - lo) / 255 in fp32 and one byte per value:
//   code = rint((x - lo) * (255 / (max - lo))),   x^ = code * step + lo,   |x - x^| <= step / 2.
// Every operation is one IEEE rounding (no contraction), so the codes are reproducible by
// any implementation of these lines.  A block whose step is below 2^-100 is constant
// (step = 0); a block that holds a value that is not finite reads back as NaN, so it is
// as visible in the gradients as it would be without checkpoints.
#include "token_common.cuh"

namespace slg {

constexpr int CK_BLOCK = SLG_CKPT_BLOCK;        // columns per (lo, step)
constexpr int CK_WARPS = 8;
constexpr float CK_TINY = 7.888609052210118e-31f;    // 2^-100

static_assert(CK_BLOCK == 128, "a warp covers a block, 4 values per lane");

template <typename T>
__device__ __forceinline__ void load4(const T* __restrict__ p, int64_t c, int64_t cols, bool vec, float (&v)[4]) {
    if (vec && c + 4 <= cols) {
        if constexpr (sizeof(T) == 4) {
            const float4 q = __ldg(reinterpret_cast<const float4*>(p + c));
            v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
        } else {
            const uint2 q = __ldg(reinterpret_cast<const uint2*>(p + c));
            unpack2<T>(q.x, v);
            unpack2<T>(q.y, v + 2);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = c + j < cols ? to_f32(p[c + j]) : 0.0f;
    }
}

__device__ __forceinline__ float warp_min_f32(float v) {
    float r;
    asm("redux.sync.min.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float warp_max_nan_f32(float v) {        // NaN when any lane has one
    float r;
    asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float max_nan_f32(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// A warp handles CK_UNIT consecutive blocks (all loads first): with one block per warp the
// kernels ran at 41% and 72% of the copy rate on 10,000 x 65,536 fp32.
constexpr int CK_UNIT = 4;

// row and block of block number q (32-bit division where it suffices)
__device__ __forceinline__ void block_of(int64_t q, int64_t nblk, int64_t& row, int64_t& blk) {
    row = q < (1ll << 32) && nblk < (1ll << 32) ? (int64_t)((uint32_t)q / (uint32_t)nblk) : q / nblk;
    blk = q - row * nblk;
}

// Codes and bounds of CK_UNIT blocks held by a warp, 4 values per lane; count(u) of the
// lane's values of block u exist, write(u, word) keeps its code word.  Returns block `lane`'s
// bounds in lanes below CK_UNIT.
template <typename N, typename W>
__device__ __forceinline__ float2 encode_blocks(const float (&v)[CK_UNIT][4], int lane, N&& count, W&& write) {
    float lo[CK_UNIT], my_lo = 0.0f, my_range = 0.0f;
#pragma unroll
    for (int u = 0; u < CK_UNIT; ++u) {
        float l = CUDART_INF_F, h = -CUDART_INF_F;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < count(u)) {
                l = fminf(l, v[u][j]);
                h = max_nan_f32(h, v[u][j]);
            }
        lo[u] = warp_min_f32(l);
        const float range = __fsub_rn(warp_max_nan_f32(h), lo[u]);      // NaN or infinite: something is not finite
        if (lane == u) { my_lo = lo[u]; my_range = range; }
    }
    // lane u works out block u's step and its inverse: one division per warp
    const bool bad = !isfinite(my_range);
    const float step = __fmul_rn(my_range, 1.0f / 255.0f);
    const bool flat = bad || step < CK_TINY;
    const float my_inv = flat ? 0.0f : __fdiv_rn(255.0f, my_range);
#pragma unroll
    for (int u = 0; u < CK_UNIT; ++u) {
        const float inv = __shfl_sync(0xffffffffu, my_inv, u);
        // Adding 1.5 2^23 rounds to the nearest even integer, as rint does, and leaves it in the
        // low byte (0 <= code <= 255 as lo <= x <= hi); conversion instructions run at an
        // eighth of the rate.
        uint32_t bits[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            bits[j] = __float_as_uint(__fadd_rn(__fmul_rn(__fsub_rn(v[u][j], lo[u]), inv), 12582912.0f));
        const uint32_t word =
            __byte_perm(__byte_perm(bits[0], bits[1], 0x0040), __byte_perm(bits[2], bits[3], 0x0040), 0x5410);
        write(u, inv == 0.0f ? 0u : word);                  // 0: a constant block, or one that is not finite
    }
    return bad ? make_float2(CUDART_NAN_F, CUDART_NAN_F) : make_float2(my_lo, flat ? 0.0f : step);
}

template <typename T>
__global__ void __launch_bounds__(CK_WARPS * 32)
ckpt_store_kernel(const T* __restrict__ x, int64_t rows, int64_t cols, int64_t ldx, int vec,
                  uint32_t* __restrict__ codes, int64_t ldw, float2* __restrict__ bounds, int64_t nblk) {
    const int lane = threadIdx.x & 31;
    const int64_t q0 = ((int64_t)blockIdx.x * CK_WARPS + (threadIdx.x >> 5)) * CK_UNIT;
    const int64_t total = rows * nblk;
    if (q0 >= total) return;
    int64_t row, blk;
    block_of(q0, nblk, row, blk);
    float v[CK_UNIT][4];
    float2 mine;
    if (vec && (blk + CK_UNIT) * CK_BLOCK <= cols) {
        // whole blocks of one row: no bounds checks (with them integer instructions are the
        // bound, 80% of their pipe: 770 us on 10,000 x 65,536)
        const T* p = x + row * ldx + blk * CK_BLOCK + lane * 4;
        uint32_t* w = codes + row * ldw + blk * (CK_BLOCK / 4) + lane;
#pragma unroll
        for (int u = 0; u < CK_UNIT; ++u) load4(p, u * CK_BLOCK, (int64_t)(u + 1) * CK_BLOCK, true, v[u]);
        mine = encode_blocks(v, lane, [](int) { return 4; }, [&](int u, uint32_t word) { w[u * (CK_BLOCK / 4)] = word; });
    } else {
        int64_t at[CK_UNIT];
        int n[CK_UNIT];
#pragma unroll
        for (int u = 0; u < CK_UNIT; ++u) {
            const int64_t c = blk * CK_BLOCK + lane * 4;
            const bool on = q0 + u < total && c < cols;
            n[u] = on ? (int)(cols - c < 4 ? cols - c : 4) : 0;
            at[u] = row * ldw + (c >> 2);
            if (on) load4(x + row * ldx, c, cols, vec, v[u]);
            if (++blk == nblk) { blk = 0; ++row; }
        }
        mine = encode_blocks(v, lane, [&](int u) { return n[u]; }, [&](int u, uint32_t word) {
            if (n[u]) codes[at[u]] = n[u] < 4 ? word & ((1u << (8 * n[u])) - 1u) : word;
        });
    }
    if (lane < CK_UNIT && q0 + lane < total) bounds[q0 + lane] = mine;
}

template <typename T>
__global__ void __launch_bounds__(CK_WARPS * 32)
ckpt_load_kernel(const uint32_t* __restrict__ codes, int64_t ldw, const float2* __restrict__ bounds, int64_t rows,
                 int64_t cols, int64_t nblk, T* __restrict__ x, int64_t ldx, int vec) {
    const int lane = threadIdx.x & 31;
    const int64_t q0 = ((int64_t)blockIdx.x * CK_WARPS + (threadIdx.x >> 5)) * CK_UNIT;
    const int64_t total = rows * nblk;
    if (q0 >= total) return;
    int64_t row, blk;
    block_of(q0, nblk, row, blk);
    uint32_t word[CK_UNIT];
    float2 b[CK_UNIT];
    T* p[CK_UNIT];
    int n[CK_UNIT];
#pragma unroll
    for (int u = 0; u < CK_UNIT; ++u) {
        const int64_t c = blk * CK_BLOCK + lane * 4;
        const bool on = q0 + u < total && c < cols;
        n[u] = on ? (int)(cols - c < 4 ? cols - c : 4) : 0;
        p[u] = x + row * ldx + c;
        word[u] = on ? __ldg(&codes[row * ldw + (c >> 2)]) : 0u;
        b[u] = on ? __ldg(&bounds[q0 + u]) : make_float2(0.f, 0.f);
        if (++blk == nblk) { blk = 0; ++row; }
    }
#pragma unroll
    for (int u = 0; u < CK_UNIT; ++u) {
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            v[j] = __fadd_rn(__fmul_rn((float)((word[u] >> (8 * j)) & 255u), b[u].y), b[u].x);
        if (vec && n[u] == 4) {
            if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(p[u]) = make_float4(v[0], v[1], v[2], v[3]);
            else *reinterpret_cast<uint2*>(p[u]) = make_uint2(pack2<T>(v), pack2<T>(v + 2));
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < n[u]) p[u][j] = from_f32<T>(v[j]);
        }
    }
}

// Rows [B, F] -> feature-major [F, ldb] (columns >= B zero) and its checkpoint in one pass: a
// CTA holds 32 features x 128 samples, one block of each feature, so the codes cost no
// second read of the activations.  Lane l has samples l, l + 32, ...: reads and writes of
// the tile are free of bank conflicts, and codes are stored byte by byte in whole lines.
constexpr int TC_F = 32;
template <bool WHOLE>       // the tile lies inside [B, F]: no bounds checks
__device__ __forceinline__ void to_fm_ckpt_tile(const float* __restrict__ x, int64_t B, int64_t F, float* __restrict__ out,
                                                int64_t ldb, uint8_t* __restrict__ codes, int64_t ldc,
                                                float2* __restrict__ bounds, int64_t nblk,
                                                float (&t)[TC_F][CK_BLOCK + 1]) {
    constexpr int ROWS = TC_F / 8;              // features per warp
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t f0 = (int64_t)blockIdx.x * TC_F, blk = blockIdx.y, b0 = blk * CK_BLOCK;
    {
        float v[16];
        const float* p = x + (b0 + warp) * F + f0 + lane;
#pragma unroll
        for (int i = 0; i < 16; ++i, p += 8 * F)
            v[i] = WHOLE || (b0 + warp + 8 * i < B && f0 + lane < F) ? __ldg(p) : 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) t[lane][warp + 8 * i] = v[i];
    }
    __syncthreads();
    const int left = (int)(B - b0 < CK_BLOCK ? B - b0 : CK_BLOCK);          // samples of the tile
    const int width = (int)(ldb - b0 < CK_BLOCK ? ldb - b0 : CK_BLOCK);     // its columns
    const int64_t f = f0 + warp * ROWS;
    float lo[ROWS], my_lo = 0.0f, my_range = 0.0f;
    float* o = out + f * ldb + b0 + lane;
#pragma unroll
    for (int u = 0; u < ROWS; ++u, o += ldb) {
        float l = CUDART_INF_F, h = -CUDART_INF_F;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float v = t[warp * ROWS + u][lane + 32 * j];
            if (WHOLE || lane + 32 * j < left) {
                l = fminf(l, v);
                h = max_nan_f32(h, v);
            }
            if (WHOLE || (f + u < F && lane + 32 * j < width)) o[32 * j] = v;
        }
        lo[u] = warp_min_f32(l);
        const float range = __fsub_rn(warp_max_nan_f32(h), lo[u]);
        if (lane == u) { my_lo = lo[u]; my_range = range; }
    }
    const bool bad = !isfinite(my_range);
    const float step = __fmul_rn(my_range, 1.0f / 255.0f);
    const bool flat = bad || step < CK_TINY;
    const float my_inv = flat ? 0.0f : __fdiv_rn(255.0f, my_range);
    if (lane < ROWS && f + lane < F)
        bounds[(f + lane) * nblk + blk] =
            bad ? make_float2(CUDART_NAN_F, CUDART_NAN_F) : make_float2(my_lo, flat ? 0.0f : step);
    uint8_t* c = codes + f * ldc + b0 + lane;
#pragma unroll
    for (int u = 0; u < ROWS; ++u, c += ldc) {
        const float inv = __shfl_sync(0xffffffffu, my_inv, u);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t code = __float_as_uint(
                __fadd_rn(__fmul_rn(__fsub_rn(t[warp * ROWS + u][lane + 32 * j], lo[u]), inv), 12582912.0f));
            if (WHOLE) c[32 * j] = (uint8_t)(inv != 0.0f ? code : 0u);
            else if (f + u < F && lane + 32 * j < width)
                c[32 * j] = (uint8_t)(lane + 32 * j < left && inv != 0.0f ? code : 0u);
        }
    }
}

__global__ void __launch_bounds__(256, 5)
to_fm_ckpt_kernel(const float* __restrict__ x, int64_t B, int64_t F, float* __restrict__ out, int64_t ldb,
                  uint8_t* __restrict__ codes, int64_t ldc, float2* __restrict__ bounds, int64_t nblk) {
    __shared__ float t[TC_F][CK_BLOCK + 1];
    if (((int64_t)blockIdx.x + 1) * TC_F <= F && ((int64_t)blockIdx.y + 1) * CK_BLOCK <= B)
        to_fm_ckpt_tile<true>(x, B, F, out, ldb, codes, ldc, bounds, nblk, t);
    else to_fm_ckpt_tile<false>(x, B, F, out, ldb, codes, ldc, bounds, nblk, t);
}

static int check_ckpt(const void* codes, int64_t ldc, const void* bounds, int64_t rows, int64_t cols, int64_t ldx,
                      int dtype, const char* name) {
    if (rows < 0 || cols < 0) return set_error(SLG_ERR_ARG, "%s: bad sizes", name);
    if (ldx < cols) return set_error(SLG_ERR_ARG, "%s: ldx < cols", name);
    if (ldc < cols) return set_error(SLG_ERR_ARG, "%s: ldc < cols", name);
    if (ldc % 4) return set_error(SLG_ERR_ALIGN, "%s: ldc must be a multiple of 4", name);
    if (dtype != SLG_DT_F32 && dtype != SLG_DT_BF16 && dtype != SLG_DT_F16)
        return set_error(SLG_ERR_UNSUPPORTED, "%s: dtype %d not built", name, dtype);
    if (rows * cols > 0 && (!codes || !bounds)) return set_error(SLG_ERR_ARG, "%s: null pointer", name);
    if (!aligned_to(codes, 4) || !aligned_to(bounds, 8))
        return set_error(SLG_ERR_ALIGN, "%s: codes / bounds misaligned", name);
    if (cdiv(rows * cdiv(cols, CK_BLOCK), CK_WARPS) >= (1ll << 31))
        return set_error(SLG_ERR_ARG, "%s: too many blocks", name);
    return SLG_OK;
}

}  // namespace slg

using namespace slg;

extern "C" int slg_ckpt_store(const void* x, int32_t dtype, int64_t rows, int64_t cols, int64_t ldx, uint8_t* codes,
                              int64_t ldc, float* bounds, void* stream) {
    int st = check_ckpt(codes, ldc, bounds, rows, cols, ldx, dtype, "slg_ckpt_store");
    if (st) return st;
    if (rows * cols == 0) return SLG_OK;
    if (!x) return set_error(SLG_ERR_ARG, "slg_ckpt_store: null pointer");
    const int64_t nblk = cdiv(cols, CK_BLOCK);
    cudaStream_t s = as_stream(stream);
    for_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const int vec = ldx % 4 == 0 && aligned_to(x, 4 * sizeof(T));
        ckpt_store_kernel<T><<<(unsigned)cdiv(rows * nblk, CK_WARPS * CK_UNIT), CK_WARPS * 32, 0, s>>>(
            (const T*)x, rows, cols, ldx, vec, reinterpret_cast<uint32_t*>(codes), ldc / 4,
            reinterpret_cast<float2*>(bounds), nblk);
    });
    return check_launch("slg_ckpt_store");
}

extern "C" int slg_ckpt_load(const uint8_t* codes, int64_t ldc, const float* bounds, int64_t rows, int64_t cols,
                             void* x, int32_t dtype, int64_t ldx, void* stream) {
    int st = check_ckpt(codes, ldc, bounds, rows, cols, ldx, dtype, "slg_ckpt_load");
    if (st) return st;
    if (rows * cols == 0) return SLG_OK;
    if (!x) return set_error(SLG_ERR_ARG, "slg_ckpt_load: null pointer");
    const int64_t nblk = cdiv(cols, CK_BLOCK);
    cudaStream_t s = as_stream(stream);
    for_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const int vec = ldx % 4 == 0 && aligned_to(x, 4 * sizeof(T));
        ckpt_load_kernel<T><<<(unsigned)cdiv(rows * nblk, CK_WARPS * CK_UNIT), CK_WARPS * 32, 0, s>>>(
            reinterpret_cast<const uint32_t*>(codes), ldc / 4, reinterpret_cast<const float2*>(bounds), rows, cols,
            nblk, (T*)x, ldx, vec);
    });
    return check_launch("slg_ckpt_load");
}

extern "C" int slg_to_feature_major_ckpt(const float* x, int64_t B, int64_t F, float* out, int64_t ldb, uint8_t* codes,
                                         int64_t ldc, float* bounds, void* stream) {
    const char* name = "slg_to_feature_major_ckpt";
    if (B <= 0 || F < 0 || ldb < B || ldc < ldb) return set_error(SLG_ERR_ARG, "%s: bad sizes", name);
    const int64_t nblk = cdiv(B, CK_BLOCK);
    // one tile row per block: padding columns may not begin another block
    if (cdiv(ldb, CK_BLOCK) != nblk) return set_error(SLG_ERR_ARG, "%s: ldb reaches past the last block", name);
    if (nblk > 65535) return set_error(SLG_ERR_ARG, "%s: batch too large", name);
    if (F == 0) return SLG_OK;
    if (!x || !out || !codes || !bounds) return set_error(SLG_ERR_ARG, "%s: null pointer", name);
    if (!aligned_to(bounds, 8)) return set_error(SLG_ERR_ALIGN, "%s: bounds misaligned", name);
    const dim3 grid((unsigned)cdiv(F, TC_F), (unsigned)nblk);
    to_fm_ckpt_kernel<<<grid, 256, 0, as_stream(stream)>>>(x, B, F, out, ldb, codes, ldc,
                                                           reinterpret_cast<float2*>(bounds), nblk);
    return check_launch(name);
}
