// Backward of a soft FC layer whose input was kept as an 8-bit checkpoint
// (checkpoint8.cu): fc_soft_bwd_kernel with the gathers reading codes.
//
// A warp owns a node and walks 1,024 samples, 128 at a time -- one block of each candidate
// row, so (lo, step) are warp-uniform.  With q the codes, x = step q + lo:
//   a_j   = sum_k w_jk x_jk = sum_k (w_jk step_jk) q_jk + sum_k w_jk lo_jk
//   dL/dw_jk = sum_b ga_j x_jk = step_jk sum_b ga_j q_jk + lo_jk sum_b ga_j
// so the codes are used as they are and the bounds enter once per block.  A gather moves 1
// byte instead of 4, and the node's 16 code words (4 samples each) stay in registers between
// the two uses.  Partials and their finish kernel are the fp32 kernel's.
//
// gx is a sum over the nodes that read a row.  Each slot's terms of a block (8 x 512 bytes)
// are laid out in shared memory and added to the rows by bulk reductions: one instruction
// per candidate, where vector atomics from registers take 16 passes of the load/store unit's
// data pipe each and made it the bound (81% busy).  10,000 nodes x 10,000 inputs x 4,096
// samples, Top-8 Walsh: 486 us (352 without gx, 606 with vector atomics); the fp32 kernel
// takes 622 (391 without gx).  What is left is instruction issue (about 800 per warp and
// block) and, for gx, 2.6 GB of additions in L2, whose units alone would take 230 us.
#include "fc_soft_impl.cuh"

namespace slg {

// Two fp32 values in one 64-bit register: the packed instructions do two samples an issue
// slot, and issue slots bound the scalar form of this kernel (72% busy, L2 at 53%).
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float a, float b) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(f32x2 p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// bytes j and j + 1 of a code word as floats: 2^23 + q has q in its low mantissa bits
__device__ __forceinline__ f32x2 codes_f32(uint32_t word, int j) {
    const f32x2 raw = pair(__uint_as_float(__byte_perm(word, 0x4b000000u, 0x7540u + j)),
                           __uint_as_float(__byte_perm(word, 0x4b000000u, 0x7541u + j)));
    return add2(raw, pair(-8388608.0f, -8388608.0f));
}
// twice bytes j and j + 1, from 2^24 + 2 q: another expression than codes_f32's, so that the
// second use of a word decodes it again instead of keeping 64 decoded values in registers
__device__ __forceinline__ f32x2 codes2_f32(uint32_t word, int j) {
    const f32x2 raw = pair(__uint_as_float(__byte_perm(word, 0x4b800000u, 0x7640u + j)),
                           __uint_as_float(__byte_perm(word, 0x4b800000u, 0x7641u + j)));
    return add2(raw, pair(-16777216.0f, -16777216.0f));
}

constexpr int CB_ITER = 8;              // blocks of 128 samples per warp
constexpr int CB_WARPS = 8;

// Per candidate (slot j's k-th at j KT + k) and block of the chunk.  Places past K have
// weight and bounds 0 and read row 0.
template <int NODE, int KT>
struct CkptSmem {
    float4 out[KT][32];                 // a slot's terms of gx for a block
    float2 back[CB_ITER][2 * KT];       // step / 2, lo
    float mix[CB_ITER][2 * KT];         // w step
    float c[CB_ITER][2];                // sum_k w lo
    const uint32_t* codes[2 * KT];
    FcSmem<NODE, 2> node;
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

template <int NODE, int KT>
__global__ void __launch_bounds__(CB_WARPS * 32, 3)
fc_soft_bwd_ckpt_kernel(const uint32_t* __restrict__ codes, uint32_t ldw, const float2* __restrict__ bounds,
                        int64_t nblk, int64_t nv, const int32_t* __restrict__ cand, const float* __restrict__ conn,
                        int K, int conn_ste, const float* __restrict__ params, int np_stride, int gate_hard,
                        float inv_tau, int64_t out_dim, int64_t wire_r, const float4* __restrict__ gy,
                        float4* __restrict__ gx, float* __restrict__ ws, int npart) {
    constexpr int NPG = NodeSize<NODE, 2>::NPG;
    constexpr int EK = 2 * KT;
    extern __shared__ __align__(16) char raw[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t o = (int64_t)blockIdx.x * CB_WARPS + warp;
    if (o >= out_dim) return;
    const int64_t chunk = blockIdx.y;
    const int64_t v0 = chunk * (32 * CB_ITER);
    float* wrow = ws + (chunk * out_dim + o) * npart;
    if (o < wire_r) {
        if (gx)
            for (int it = 0; it < CB_ITER; ++it) {
                const int64_t v = v0 + it * 32 + lane;
                if (v < nv) atomicAdd(&gx[o * nv + v], gy[o * nv + v]);
            }
        for (int e = lane; e < npart; e += 32) wrow[e] = 0.0f;
        return;
    }
    CkptSmem<NODE, KT>& S = reinterpret_cast<CkptSmem<NODE, KT>*>(raw)[warp];
    stage_node<NODE, 2>(S.node, o, cand, conn, K, conn_ste, params, np_stride, gate_hard, inv_tau, lane);
    for (int e = lane; e < EK * CB_ITER; e += 32) {
        const int it = e % CB_ITER, p = e / CB_ITER, j = p / KT, k = p % KT;
        float mix = 0.0f;
        float2 back = make_float2(0.f, 0.f);
        const int64_t blk = chunk * CB_ITER + it;
        const int64_t row = k < K ? S.node.cand[j * K + k] : 0;
        if (k < K && blk < nblk) {
            const float2 b = __ldg(&bounds[row * nblk + blk]);
            const float w = S.node.w[j * K + k];
            mix = w * b.y;
            back = make_float2(0.5f * b.y, b.x);
        }
        S.mix[it][p] = mix;
        S.back[it][p] = back;
        if (it == 0) S.codes[p] = codes + row * ldw;
    }
    // lane e sends candidate e's terms to its row of gx
    float4* target = nullptr;
    if (gx && lane < EK && lane % KT < K) {
        const int at = (lane / KT) * K + lane % KT;
        if (S.node.w[at] != 0.0f) target = gx + (int64_t)S.node.cand[at] * nv;
    }
    __syncwarp();
    if (lane < 2 * CB_ITER) {
        const int it = lane >> 1, j = lane & 1;
        float c = 0.0f;
        for (int k = 0; k < K; ++k) c += S.node.w[j * K + k] * S.back[it][j * KT + k].y;
        S.c[it][j] = c;
    }
    float acc_node[NPG], acc_w[EK];
#pragma unroll
    for (int q = 0; q < NPG; ++q) acc_node[q] = 0.0f;
#pragma unroll
    for (int e = 0; e < EK; ++e) acc_w[e] = 0.0f;

#pragma unroll 1
    for (int it = 0; it < CB_ITER; ++it) {
        const int64_t v = v0 + it * 32 + lane;
        if (v0 + it * 32 >= nv) break;
        __syncwarp();       // wiring and weights are read from shared memory each time, not kept
        const bool on = v < nv;
        uint32_t q[EK];
#pragma unroll
        for (int e = 0; e < EK; ++e) q[e] = on ? __ldg(S.codes[e] + v) : 0u;
        const float4 g = on ? gy[o * nv + v] : make_float4(0.f, 0.f, 0.f, 0.f);
        float a[4][2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float c = S.c[it][j];
            f32x2 a01 = pair(c, c), a23 = a01;
#pragma unroll
            for (int k = 0; k < KT; ++k) {
                const float w = S.mix[it][j * KT + k];
                const f32x2 ww = pair(w, w);
                a01 = fma2(ww, codes_f32(q[j * KT + k], 0), a01);
                a23 = fma2(ww, codes_f32(q[j * KT + k], 2), a23);
            }
            unpair(a01, a[0][j], a[1][j]);
            unpair(a23, a[2][j], a[3][j]);
        }
        const float gs[4] = {g.x, g.y, g.z, g.w};
        float ga[4][2];
#pragma unroll
        for (int s = 0; s < 4; ++s) node_bwd<NODE, 2>(S.node.np, a[s], gs[s], ga[s], acc_node);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            // the copies of the slot before have read S.out
            if (gx) {
                asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                __syncwarp();
            }
            const f32x2 g01 = pair(ga[0][j], ga[1][j]), g23 = pair(ga[2][j], ga[3][j]);
            const float sum = (ga[0][j] + ga[1][j]) + (ga[2][j] + ga[3][j]);
#pragma unroll
            for (int k = 0; k < KT; ++k) {
                const int e = j * KT + k;
                const float2 b = S.back[it][e];
                const float half_step = b.x, lo = b.y;
                const float w = k < K ? S.node.w[j * K + k] : 0.0f;
                const f32x2 ww = pair(w, w);
                if (KT > 1 || conn) {       // a single given weight has a gradient too
                    const f32x2 t = fma2(g01, codes2_f32(q[e], 0), mul2(g23, codes2_f32(q[e], 2)));
                    float t0, t1;
                    unpair(t, t0, t1);
                    acc_w[e] = fmaf(half_step, t0 + t1, fmaf(lo, sum, acc_w[e]));
                }
                *reinterpret_cast<ulonglong2*>(&S.out[k][lane]) = make_ulonglong2(mul2(g01, ww), mul2(g23, ww));
            }
            if (gx) {
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                const int64_t left = nv - (v0 + it * 32);
                const uint32_t bytes = left < 32 ? (uint32_t)left * 16u : 512u;
                if (target && lane / KT == j)
                    asm volatile("cp.reduce.async.bulk.global.shared::cta.bulk_group.add.f32 [%0], [%1], %2;" ::"l"(
                                     target + v0 + it * 32),
                                 "r"(smem_addr(&S.out[lane % KT][0])), "r"(bytes)
                                 : "memory");
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
        }
    }
    if (gx) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int k = 0; k < KT; ++k)
            if (k < K) {
                const float s = warp_sum(acc_w[j * KT + k]);
                if (lane == 0) wrow[j * K + k] = s;
            }
#pragma unroll
    for (int q = 0; q < NPG; ++q) {
        const float s = warp_sum(acc_node[q]);
        if (lane == 0) wrow[2 * K + q] = s;
    }
}

template <int NODE, int KT>
static void launch_ckpt(const FcArgs& A, const uint32_t* codes, int64_t ldw, const float2* bounds, const float* gy,
                        float* gx, float* ws, float* gconn, float* gparams, cudaStream_t st) {
    const int64_t nv = A.ldb / 4, nchunk = cdiv(nv, 32 * CB_ITER);
    constexpr int smem = CB_WARPS * (int)sizeof(CkptSmem<NODE, KT>);
    static_assert(sizeof(CkptSmem<NODE, KT>) % 16 == 0 && 3 * (smem + 1024) <= 227 * 1024 + 512, "three CTAs per SM");
    if (smem > 48 * 1024)
        cudaFuncSetAttribute(fc_soft_bwd_ckpt_kernel<NODE, KT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    const int npart = 2 * A.K + NodeSize<NODE, 2>::NPG;
    dim3 grid((unsigned)cdiv(A.out_dim, CB_WARPS), (unsigned)nchunk);
    fc_soft_bwd_ckpt_kernel<NODE, KT><<<grid, CB_WARPS * 32, smem, st>>>(
        codes, (uint32_t)ldw, bounds, cdiv(A.ldb, SLG_CKPT_BLOCK), nv, A.cand, A.conn, A.K, A.conn_ste, A.params,
        np_stride_of(NODE, 2), A.gate_hard, A.inv_tau, A.out_dim, A.wire_r, reinterpret_cast<const float4*>(gy),
        reinterpret_cast<float4*>(gx), ws, npart);
    fc_soft_finish_kernel<NODE, 2><<<(unsigned)cdiv(A.out_dim, 128), 128, 0, st>>>(
        ws, nchunk, A.out_dim, npart, A.K, A.conn, A.conn_ste, A.params, np_stride_of(NODE, 2), A.wire_r, gconn, gparams);
}

}  // namespace slg

using namespace slg;

extern "C" int32_t slg_fc_soft_bwd_ckpt_built(int32_t K, int32_t node, int32_t arity) {
    return arity == 2 && K >= 1 && K <= 8 && (node == N_GATE16 || node == N_WALSH || node == N_MULTI || node == N_HYBRID);
}

extern "C" int slg_fc_soft_bwd_ckpt(const uint8_t* codes, int64_t ldc, const float* bounds, int64_t in_dim, int64_t ldb,
                                    const int32_t* cand, const float* conn, int32_t K, int32_t conn_ste, int32_t node,
                                    int32_t arity, const float* params, int32_t gate_hard, float inv_tau,
                                    int64_t out_dim, int64_t wire_r, const float* gy, float* gx, float* gconn,
                                    float* gparams, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* name = "slg_fc_soft_bwd_ckpt";
    if (in_dim <= 0 || out_dim < 0 || ldb <= 0 || K <= 0 || wire_r < 0) return set_error(SLG_ERR_ARG, "%s: bad sizes", name);
    if (!slg_fc_soft_bwd_ckpt_built(K, node, arity))
        return set_error(SLG_ERR_UNSUPPORTED, "%s: node %d arity %d K=%d not built", name, node, arity, K);
    if (ldb % 4 || ldc % 4) return set_error(SLG_ERR_ALIGN, "%s: ldb and ldc must be multiples of 4", name);
    if (ldc < ldb) return set_error(SLG_ERR_ARG, "%s: ldc < ldb", name);
    if (ldc / 4 >= (1ll << 32)) return set_error(SLG_ERR_ARG, "%s: rows too long", name);
    if (conn_ste < 0 || conn_ste > 2) return set_error(SLG_ERR_ARG, "%s: conn_ste %d not in 0..2", name, conn_ste);
    if (wire_r > 0 && (wire_r > in_dim || wire_r > out_dim)) return set_error(SLG_ERR_ARG, "%s: wire_r exceeds a width", name);
    if (cdiv(ldb / 4, 32 * FS_ITER) > 65535) return set_error(SLG_ERR_ARG, "%s: batch too large", name);
    if (!codes || !bounds || !cand || !params || !gy || !gparams || !workspace)
        return set_error(SLG_ERR_ARG, "%s: null pointer", name);
    if (conn && !gconn) return set_error(SLG_ERR_ARG, "%s: gconn required with conn", name);
    if (!aligned16(gy) || (gx && !aligned16(gx)) || (reinterpret_cast<uintptr_t>(codes) & 3u) ||
        (reinterpret_cast<uintptr_t>(bounds) & 7u))
        return set_error(SLG_ERR_ALIGN, "%s: gy/gx/codes/bounds misaligned", name);
    const int64_t need = slg_fc_soft_workspace_bytes(ldb, K, node, arity, out_dim);
    if (workspace_bytes < need)
        return set_error(SLG_ERR_WORKSPACE, "%s: workspace %lld < %lld bytes", name, (long long)workspace_bytes,
                         (long long)need);
    const FcArgs A{nullptr, in_dim, ldb, cand, conn, K, conn_ste, params, gate_hard, inv_tau, out_dim, wire_r};
    const uint32_t* c = reinterpret_cast<const uint32_t*>(codes);
    const float2* b = reinterpret_cast<const float2*>(bounds);
    float* ws = static_cast<float*>(workspace);
    cudaStream_t s = as_stream(stream);
    if (gx) {
        const cudaError_t err = cudaMemsetAsync(gx, 0, (size_t)in_dim * (size_t)ldb * 4, s);
        if (err != cudaSuccess) return set_error(SLG_ERR_CUDA, "%s: %s", name, cudaGetErrorString(err));
    }
    if (out_dim == 0) return SLG_OK;
    auto go = [&](auto node_tag) {
        constexpr int NODE = decltype(node_tag)::value;
        if (K == 1) launch_ckpt<NODE, 1>(A, c, ldc / 4, b, gy, gx, ws, gconn, gparams, s);
        else if (K <= 4) launch_ckpt<NODE, 4>(A, c, ldc / 4, b, gy, gx, ws, gconn, gparams, s);
        else launch_ckpt<NODE, 8>(A, c, ldc / 4, b, gy, gx, ws, gconn, gparams, s);
    };
    switch (node) {
        case N_GATE16: go(std::integral_constant<int, N_GATE16>()); break;
        case N_WALSH: go(std::integral_constant<int, N_WALSH>()); break;
        case N_MULTI: go(std::integral_constant<int, N_MULTI>()); break;
        default: go(std::integral_constant<int, N_HYBRID>()); break;
    }
    return check_launch(name);
}
