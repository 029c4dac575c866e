// K8: the products of proj_skinny.cuh / proj_tcgen05.cuh with 4-bit weights:
//     C[m x N] = (residual +) A[m x K] . W^T,   W[n][k] = (q[n][k] - z[n][k/g]) * scale[n][k/g],
// q in 0..15 two to a byte (even k in the low half), scale bf16, z a byte (8 where no zeros are given),
// g = 32, 64 or 128 inputs to a group.
//
// Up to 16 rows (a decode step): proj_w4_kernel.  Bound by streaming the packed weights, N K / 2 bytes,
// once; everything else has to stay below that.  A warp takes 16 columns as the M side of m16n8k16 and
// the rows as one or two N blocks of 8, like the bf16 kernel's transposed form, and
//   * streams its weights through a private ring of 16-byte asynchronous copies (each is used once, no
//     sharing, no CTA barrier in the loop), requested before the wait for the stream's previous kernel;
//   * reads one 32-bit word = 8 consecutive inputs of a column per lane: the four lanes of a quad hold the
//     32 inputs of one 32-block, so no product mixes two groups and the scale is applied to the fp32
//     sums, not to the weights - q - z (exact in bf16) is what the tensor core multiplies;
//   * turns a word into four bf16 pairs with a shift, a logic operation (0x4300 | q is 128 + q in bf16)
//     and a subtraction of 128 + z each; the pairs are inputs (i, i+4) of the word, and the rows'
//     fragments are paired the same way with byte permutes;
//   * reuses a row fragment for CB column blocks, so that the rows' traffic (2 bytes x m per input and
//     pass) stays at or below the weights'.
// The CTA's 8 warps split K; their sums are added in warp order, so the result does not depend on timing.
//
// More rows: w4_unpack_kernel writes the weights once as bf16 (this rounds (q - z) * scale to 8 bits, half
// a bf16 step per weight; unlike above the tensor-memory accumulator runs over all groups, so the scale
// has to be in the operand) and proj_tcgen05_kernel multiplies.
#pragma once
#include "common.cuh"

namespace ellm {

constexpr int kW4Warps = 8;
constexpr int kW4Threads = kW4Warps * 32;
constexpr int kW4MaxRows = 16;
constexpr int kW4StageBytes = 4096;   // per warp: CB * 16 columns x 512 / CB inputs
constexpr int kW4Stages = 5;
constexpr int kW4RingBytes = kW4Warps * kW4Stages * kW4StageBytes;

struct W4Params {
    const __nv_bfloat16* a;
    long long lda;
    const uint8_t* w;              // [n_cols][k / 2]
    const __nv_bfloat16* scales;   // [n_cols][k / g]
    const uint8_t* zeros;          // [n_cols][k / g] or nullptr (8)
    const __nv_bfloat16* residual;
    long long ldr;
    __nv_bfloat16* c;
    long long ldc;
    int m_rows, batch, max_batch;  // rows with (row % max_batch) >= batch are skipped
    int n_cols, k;                 // k a multiple of 128
};

__host__ __device__ inline int w4_smem_bytes(int cb, int nb) { return kW4RingBytes + kW4Warps * cb * 16 * nb * 8 * 4; }

// inputs (i, i + 4), i = 0..3, of a word of 8, minus the zero point: q - z as exact bf16 pairs
__device__ __forceinline__ void w4_pairs(uint32_t word, uint32_t z128, uint32_t (&r)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t q = ((word >> (4 * i)) & 0x000f000fu) | 0x43004300u;
        const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&q), *reinterpret_cast<const __nv_bfloat162*>(&z128));
        r[i] = *reinterpret_cast<const uint32_t*>(&d);
    }
}

// 128 + z twice; z up to 127 exact
__device__ __forceinline__ uint32_t w4_z128(uint32_t z) { return 0x43004300u + z * 0x00010001u; }

template <int CB, int NB, int GW>   // column blocks per pass, blocks of 8 rows, 32-blocks per group (group = 32 * GW)
__global__ void __launch_bounds__(kW4Threads, 1) proj_w4_kernel(const W4Params p) {
    extern __shared__ __align__(128) unsigned char smem[];
    constexpr int kUnit = 512 / CB;             // inputs per stage
    constexpr int kBlocks = kUnit / 128;        // 128-blocks per stage
    constexpr int kRow = kUnit / 2;             // bytes of a column in a stage
    constexpr int kChunks = kRow / 16;          // 16-byte pieces of it
    constexpr int kGroups = 4 / GW;             // groups per 128-block
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t ring = smem_u32(smem) + warp * kW4Stages * kW4StageBytes;
    float* part = reinterpret_cast<float*>(smem + kW4RingBytes);   // [warp][CB * 16 columns][NB * 8 rows]

    // this CTA's column blocks, and how many units of K each warp takes of every pass
    long long blk0, blk1;
    if (!assign_range((p.n_cols + 15) / 16, gridDim.x, blockIdx.x, &blk0, &blk1)) return;
    const int nblk = static_cast<int>(blk1 - blk0), passes = (nblk + CB - 1) / CB;
    const int units = (p.k + kUnit - 1) / kUnit;
    long long u0 = 0, u1 = 0;
    assign_range(units, kW4Warps, warp, &u0, &u1);
    const int mine = static_cast<int>(u1 - u0), total = mine * passes;
    const long long row_bytes = p.k / 2;

    // 16-byte piece c of column r sits at c ^ swz(r): the 8 columns a load touches fall in 8 different bank groups
    auto swz = [](int r) { return kChunks >= 8 ? (r & 7) : ((r >> 1) & 3); };
    auto issue = [&](int step) {
        const int pass = step / mine, unit = static_cast<int>(u0) + step % mine;
        const int n_first = static_cast<int>(blk0 + pass * CB) * 16, n_last = min(p.n_cols, static_cast<int>(blk1) * 16);
        const uint32_t dst = ring + (step % kW4Stages) * kW4StageBytes;
#pragma unroll
        for (int i = 0; i < kW4StageBytes / 512; ++i) {
            const int piece = i * 32 + lane, r = piece / kChunks, c = piece % kChunks;
            const int n = n_first + r;
            const long long byte = static_cast<long long>(unit) * kRow + c * 16;
            const bool ok = n < n_last && byte < row_bytes;
            cp_async_16(dst + r * kRow + ((c ^ swz(r)) << 4), p.w + (ok ? n * row_bytes + byte : 0), ok ? 16 : 0);
        }
    };
#pragma unroll
    for (int s = 0; s < kW4Stages - 1; ++s) {
        if (s < total) issue(s);
        cp_async_commit();
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    const __nv_bfloat16* xrow[NB];
    bool live[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const int m = nb * 8 + g;
        live[nb] = m < p.m_rows && (m % p.max_batch) < p.batch;
        xrow[nb] = p.a + (live[nb] ? m * p.lda : 0);
    }
    const int groups_row = p.k / (32 * GW);

    int step = 0;
    for (int pass = 0; pass < passes; ++pass) {
        float acc[CB][NB][4];
#pragma unroll
        for (int cb = 0; cb < CB; ++cb)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) acc[cb][nb][0] = acc[cb][nb][1] = acc[cb][nb][2] = acc[cb][nb][3] = 0.0f;
        const int n_first = static_cast<int>(blk0 + pass * CB) * 16;
        const int cbs = min(CB, nblk - pass * CB);
        for (int u = 0; u < mine; ++u, ++step) {
            if (step + kW4Stages - 1 < total) issue(step + kW4Stages - 1);
            cp_async_commit();
            cp_async_wait<kW4Stages - 1>();
            __syncwarp();
            const uint32_t st = ring + (step % kW4Stages) * kW4StageBytes;
            const int k0 = (static_cast<int>(u0) + u) * kUnit;
#pragma unroll 1
            for (int kb = 0; kb < kBlocks; ++kb) {
                const int k = k0 + kb * 128;
                if (k >= p.k) break;
                // rows: inputs [k + 32 w + 8 t, +8) of row g, paired (i, i + 4) like the weights
                uint32_t x[NB][4][4];
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        uint4 v = make_uint4(0u, 0u, 0u, 0u);
                        if (live[nb]) v = *reinterpret_cast<const uint4*>(xrow[nb] + k + w * 32 + t * 8);
                        x[nb][w][0] = __byte_perm(v.x, v.z, 0x5410);
                        x[nb][w][1] = __byte_perm(v.x, v.z, 0x7632);
                        x[nb][w][2] = __byte_perm(v.y, v.w, 0x5410);
                        x[nb][w][3] = __byte_perm(v.y, v.w, 0x7632);
                    }
#pragma unroll
                for (int cb = 0; cb < CB; ++cb) {
                    if (cb >= cbs) break;
                    // scales and zero points of this lane's two columns, all groups of the 128-block
                    float sc[2][kGroups];
                    uint32_t zz[2][kGroups];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int n = n_first + cb * 16 + h * 8 + g;
                        const long long at = static_cast<long long>(min(n, p.n_cols - 1)) * groups_row + k / (32 * GW);
#pragma unroll
                        for (int gr = 0; gr < kGroups; ++gr) {
                            sc[h][gr] = __bfloat162float(p.scales[at + gr]);
                            zz[h][gr] = w4_z128(p.zeros ? p.zeros[at + gr] : 8u);
                        }
                    }
                    const int r0 = cb * 16 + g, r1 = r0 + 8;
#pragma unroll
                    for (int gr = 0; gr < kGroups; ++gr) {
                        float d[NB][4];
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) d[nb][0] = d[nb][1] = d[nb][2] = d[nb][3] = 0.0f;
#pragma unroll
                        for (int wi = 0; wi < GW; ++wi) {
                            const int w = gr * GW + wi, c = kb * 4 + w;
                            uint32_t lo, hi, pl[4], ph[4];
                            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(lo) : "r"(st + r0 * kRow + ((c ^ swz(r0)) << 4) + t * 4));
                            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(hi) : "r"(st + r1 * kRow + ((c ^ swz(r1)) << 4) + t * 4));
                            w4_pairs(lo, zz[0][gr], pl);
                            w4_pairs(hi, zz[1][gr], ph);
                            const uint32_t a0[4] = {pl[0], ph[0], pl[1], ph[1]}, a1[4] = {pl[2], ph[2], pl[3], ph[3]};
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb) {
                                mma_bf16_16816(d[nb], a0, x[nb][w][0], x[nb][w][1]);
                                mma_bf16_16816(d[nb], a1, x[nb][w][2], x[nb][w][3]);
                            }
                        }
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            acc[cb][nb][0] += d[nb][0] * sc[0][gr];
                            acc[cb][nb][1] += d[nb][1] * sc[0][gr];
                            acc[cb][nb][2] += d[nb][2] * sc[1][gr];
                            acc[cb][nb][3] += d[nb][3] * sc[1][gr];
                        }
                    }
                }
            }
            __syncwarp();   // all lanes are done with the stage before it is refilled
        }
        // ---- the warps' sums of this pass, added in warp order ----
        // a lane holds columns g and g + 8 of rows 2t and 2t + 1 of every block
        float* mypart = part + warp * CB * 16 * NB * 8;
#pragma unroll
        for (int cb = 0; cb < CB; ++cb)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                float* row = mypart + (nb * 8 + 2 * t) * (CB * 16) + cb * 16 + g;
                row[0] = acc[cb][nb][0];
                row[CB * 16] = acc[cb][nb][1];
                row[8] = acc[cb][nb][2];
                row[CB * 16 + 8] = acc[cb][nb][3];
            }
        __syncthreads();
        for (int idx = threadIdx.x; idx < p.m_rows * CB * 16; idx += kW4Threads) {
            const int m = idx / (CB * 16), j = idx % (CB * 16), n = n_first + j;
            if (j >= cbs * 16 || n >= p.n_cols || (m % p.max_batch) >= p.batch) continue;
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kW4Warps; ++w) sum += part[(w * NB * 8 + m) * (CB * 16) + j];
            if (p.residual) sum += __bfloat162float(p.residual[m * p.ldr + n]);
            p.c[m * p.ldc + n] = __float2bfloat16_rn(sum);
        }
        if (pass + 1 < passes) __syncthreads();
    }
    cp_async_wait<0>();
}

// Packed weights -> bf16 [n][k]; a thread unpacks 8 inputs.  HBM-bound: 0.5 byte read, 2 written per weight.
__global__ void __launch_bounds__(256) w4_unpack_kernel(const uint32_t* w, const __nv_bfloat16* scales, const uint8_t* zeros, uint4* out,
                                                        long long words, int words_row, int words_group) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int groups_row = words_row / words_group;
    for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < words; i += static_cast<long long>(gridDim.x) * blockDim.x) {
        const long long n = i / words_row;
        const long long at = n * groups_row + static_cast<int>(i - n * words_row) / words_group;
        const float s = __bfloat162float(scales[at]);
        const float zs = static_cast<float>(zeros ? zeros[at] : 8);
        const uint32_t word = w[i];
        uint32_t r[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            r[j] = pack_bf16((static_cast<float>((word >> (8 * j)) & 15u) - zs) * s, (static_cast<float>((word >> (8 * j + 4)) & 15u) - zs) * s);
        out[i] = make_uint4(r[0], r[1], r[2], r[3]);
    }
}

}  // namespace ellm
