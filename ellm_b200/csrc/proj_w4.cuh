// K8: the products of proj_skinny.cuh / proj_tcgen05.cuh with 4-bit weights:
//     C[m x N] = (residual +) A[m x K] . W^T,   W[n][k] = (q[n][k] - z[n][k/g]) * scale[n][k/g],
// q in 0..15 two to a byte (even k in the low half), scale bf16, z a byte (8 where no zeros are given),
// g = 32, 64 or 128 inputs to a group.
//
// Up to 16 rows (a decode step): proj_w4_kernel.  Bound by streaming the packed weights, N K / 2 bytes,
// once; everything else has to stay below that.  A warp takes 16 columns as the M side of m16n8k16 and
// the rows as one or two N blocks of 8, like the bf16 kernel's transposed form.
//   * One CTA per SM owns a run of 16-column blocks.  Its 16 warps stand WN across the columns (CB blocks
//     each) and WK = 16 / WN along K, and walk K in chunks of WK x 128 inputs.
//   * Weights: every warp streams its own through a private ring of 16-byte asynchronous copies (each is
//     used once), requested before the wait for the stream's previous kernel.
//   * Rows: a chunk of them is staged once for all warps, two buffers, through registers, so that the
//     inputs can be stored in the order the unpacked weights have.
//   * A lane reads one 32-bit word = 8 consecutive inputs of a column; the four lanes of a quad hold a
//     32-block, so no product mixes two groups and the scale is applied to the fp32 sums, not to the
//     weights.
//   * Unpacking decides the rate (every weight is unpacked once per step): a word becomes four bf16 pairs
//     128 + q with a logic operation each (and a shift for three of them), from which a packed subtraction takes
//     128 + z.  Both and their difference q - z are exact in bf16, so the tensor core multiplies q - z itself: a weight
//     of zero adds nothing, and the roundings are those of the sum's own terms.
// The sums of the WK warps of a column are added in warp order: the result does not depend on timing.
// Measured, groups of 128: 1 x 2048 x 4096 3.9 us (a launch and two round trips to memory for 4 MB), 8 x 8192 x 8192
// 19.4 us (1.8 TB/s: unpacking and products bound it, not the stream; groups of 32 21.0 us).
//
// Large weights and more rows: proj_w4_tcgen05.cuh.
#pragma once
#include "common.cuh"

namespace ellm {

constexpr int kW4MaxRows = 16;

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

// CB: column blocks of a warp, WN: warps across the columns, NB: blocks of 8 rows.
template <int CB, int WN, int NB>
struct W4Shape {
    // with four blocks a warp needs about 200 registers (sums, row fragments, unpacked words): half the warps,
    // each taking two 128-input blocks of a chunk
    static constexpr int kWarps = CB == 4 ? 8 : 16;
    static constexpr int kThreads = kWarps * 32;
    static constexpr int kWK = kWarps / WN;                      // warps along K
    static constexpr int kKB = CB == 4 ? 2 : 1;                  // 128-blocks of a warp in a chunk
    static constexpr int kChunk = kWK * kKB * 128;               // inputs of a chunk
    static constexpr int kRow = kKB * 64;                        // bytes of a column in a stage
    static constexpr int kStageBytes = CB * 16 * kRow;           // a warp's weights of a chunk
    static constexpr int kXBytes = NB * 8 * kChunk * 2;          // a chunk of the rows
    static constexpr int kStages = CB == 4 ? 3 : (NB * kWK >= 32 ? 5 : 6);
    static constexpr int kRingBytes = kWarps * kStages * kStageBytes;
    static constexpr int kPartBytes = kWK * WN * CB * 16 * NB * 8 * 4;   // the warps' sums, over the drained ring
    static constexpr int kSmemBytes = (kRingBytes > kPartBytes ? kRingBytes : kPartBytes) + 2 * kXBytes;
    static_assert(kSmemBytes <= 232448, "shared memory budget");
    // 16-byte piece c of column r sits at c ^ swz(r): the 8 columns a load touches fall in different bank groups
    __device__ static constexpr int swz(int r) { return kKB == 2 ? (r & 7) : ((r >> 1) & 3); }
};

// q - z of inputs (i, i + 4), i = 0..3, of a word of 8, as bf16 pairs.  128 + q and 128 + z (z up to 127, `zero` holds it
// twice) are the bf16 numbers 0x4300 | q and 0x4300 | z.
__device__ __forceinline__ void w4_pairs(uint32_t word, uint32_t base, uint32_t zero, uint32_t (&r)[4]) {
    const uint32_t s[4] = {word, word >> 4, word >> 8, word >> 12};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xea;" : "=r"(r[i]) : "r"(s[i]), "r"(base));   // (s & mask) | base
        const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&r[i]), *reinterpret_cast<const __nv_bfloat162*>(&zero));
        r[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
}
// 128 + z twice, z being byte `gr` of four
__device__ __forceinline__ uint32_t w4_zero_pair(uint32_t z4, int gr) {
    return __byte_perm(z4, 0x43434343u, 0x4040u + 0x0101u * static_cast<uint32_t>(gr));
}

template <int CB, int WN, int NB, int GW>   // GW: 32-blocks per group (group = 32 * GW)
__global__ void __launch_bounds__(W4Shape<CB, WN, NB>::kThreads, 1) proj_w4_kernel(const W4Params p) {
    using S = W4Shape<CB, WN, NB>;
    extern __shared__ __align__(128) unsigned char smem[];
    constexpr int kGroups = 4 / GW;                                  // groups per 128 inputs
    constexpr int kXPieces = NB * 8 * S::kChunk / 8;                 // 16-byte pieces of a chunk of the rows
    constexpr int kXPer = (kXPieces + S::kThreads - 1) / S::kThreads;  // per thread
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int wn = warp % WN, wk = warp / WN;
    unsigned char* xs = smem + S::kSmemBytes - 2 * S::kXBytes;
    unsigned char* ring = smem + warp * S::kStages * S::kStageBytes;
    const uint32_t ring_addr = smem_u32(ring);
    float* part = reinterpret_cast<float*>(smem);                    // [wk][row][WN * CB * 16 columns]

    long long blk0, blk1;   // this CTA's column blocks
    if (!assign_range((p.n_cols + 15) / 16, gridDim.x, blockIdx.x, &blk0, &blk1)) return;
    const int passes = (static_cast<int>(blk1 - blk0) + WN * CB - 1) / (WN * CB);
    const int chunks = (p.k + S::kChunk - 1) / S::kChunk;
    const long long row_bytes = p.k / 2;
    const int groups_row = p.k / (32 * GW), blocks_k = p.k / 128;
    bool waited = false;
    uint32_t base;
    asm volatile("mov.u32 %0, 0x43004300;" : "=r"(base));   // (opaque: kept in a register, so that w4_pairs is one logic operation per pair)

    for (int pass = 0; pass < passes; ++pass) {
        // this warp's blocks of the pass: the pass's blocks split evenly over the WN warps
        const int pass_blk = static_cast<int>(blk0) + pass * WN * CB, pass_n = min(WN * CB, static_cast<int>(blk1) - pass_blk);
        long long c0 = 0, c1 = 0;
        assign_range(pass_n, WN, wn, &c0, &c1);
        const int cbs = static_cast<int>(c1 - c0), n_first = (pass_blk + static_cast<int>(c0)) * 16;
        const int n_last = min(p.n_cols, n_first + cbs * 16);

        // A lane copies piece lane % P of columns lane / P + (32 / P) i, P pieces to a column.
        constexpr int kP = S::kRow / 16, kColStep = 32 / kP, kCopies = S::kStageBytes / 512;
        const int pr = lane / kP, pc = lane % kP;
        const uint8_t* wsrc = p.w + (n_first + pr) * row_bytes + wk * S::kRow + pc * 16;   // of the next chunk requested
        const long long wstep = kColStep * row_bytes;
        const int wcols = n_last - n_first - pr;   // column i * kColStep + pr exists when i * kColStep < wcols
        const bool full = n_first + CB * 16 <= n_last;   // all of the warp's columns exist
        int wslot = 0, wk0 = wk * S::kKB * 128 + pc * 32;
        auto issue = [&]() {
            const uint32_t dst = ring_addr + wslot * S::kStageBytes + pr * S::kRow;
            const bool in_k = wk0 < p.k;
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                const uint32_t at = dst + i * kColStep * S::kRow + ((pc ^ S::swz(pr + i * kColStep)) << 4);
                if (full) {
                    if (in_k) cp_async_16(at, wsrc + i * wstep, 16);
                } else {   // columns that do not exist: zeros
                    const bool ok = in_k && i * kColStep < wcols;
                    cp_async_16(at, ok ? wsrc + i * wstep : p.w, ok ? 16 : 0);
                }
            }
            wsrc += S::kWK * S::kRow;
            wk0 += S::kChunk;
            wslot = wslot + 1 == S::kStages ? 0 : wslot + 1;
        };
#pragma unroll
        for (int s = 0; s < S::kStages - 1; ++s) {
            if (s < chunks) issue();
            cp_async_commit();
        }
        if (!waited) {
            asm volatile("griddepcontrol.wait;" ::: "memory");
            asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
            waited = true;
        }

        // rows of a chunk: a piece = 8 inputs of a row, stored as the pairs (i, i + 4); row r's pieces are XORed
        // with (r & 1) << 2 (a quarter-warp reads two rows' 64-byte runs).  A thread's pieces are of the same
        // inputs of different rows, or of one row when a chunk has more pieces per row than there are threads.
        constexpr int kRowPieces = S::kChunk / 8;
        static_assert(kRowPieces <= S::kThreads && S::kThreads % kRowPieces == 0 && kXPieces % kRowPieces == 0, "whole rows per sweep");
        constexpr int kRowStep = S::kThreads / kRowPieces;
        const int xm = threadIdx.x / kRowPieces, xc = threadIdx.x % kRowPieces;
        uint4 xv[kXPer];
        unsigned xlive = 0;
#pragma unroll
        for (int i = 0; i < kXPer; ++i) {
            const int m = xm + i * kRowStep;
            if (m < p.m_rows && (m % p.max_batch) < p.batch) xlive |= 1u << i;
        }
        const __nv_bfloat16* xsrc = p.a + xm * p.lda + xc * 8;
        int xk = xc * 8;
        auto x_fetch = [&]() {
#pragma unroll
            for (int i = 0; i < kXPer; ++i) {
                xv[i] = make_uint4(0u, 0u, 0u, 0u);
                if (((xlive >> i) & 1u) && xk < p.k) xv[i] = *reinterpret_cast<const uint4*>(xsrc + i * kRowStep * p.lda);
            }
            xsrc += S::kChunk;
            xk += S::kChunk;
        };
        auto x_store = [&](int buffer) {
#pragma unroll
            for (int i = 0; i < kXPer; ++i) {
                const int m = xm + i * kRowStep;
                if (m >= NB * 8) continue;
                uint4 v;
                v.x = __byte_perm(xv[i].x, xv[i].z, 0x5410);
                v.y = __byte_perm(xv[i].x, xv[i].z, 0x7632);
                v.z = __byte_perm(xv[i].y, xv[i].w, 0x5410);
                v.w = __byte_perm(xv[i].y, xv[i].w, 0x7632);
                *reinterpret_cast<uint4*>(xs + buffer * S::kXBytes + m * (S::kChunk * 2) + ((xc ^ ((m & 1) << 2)) << 4)) = v;
            }
        };
        // Scales (bf16) and zero points (bytes) of the 128 inputs of a chunk: lane (g, t) holds those of columns g
        // and g + 8 of block t % CB, the quad's lanes hand them to one another.  The next chunk's are requested
        // while the current one's are in use.  (Columns that do not exist read another one's; nothing is stored.)
        const int sblk = min(t % CB, max(cbs - 1, 0));
        const __nv_bfloat16* sptr[2];
        const uint8_t* zptr[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const long long at = static_cast<long long>(min(n_first + sblk * 16 + h * 8 + g, p.n_cols - 1)) * groups_row;
            sptr[h] = p.scales + at;
            zptr[h] = p.zeros + at;   // (only followed when there are zero points)
        }
        uint2 snew[2];
        uint32_t znew[2] = {0x08080808u, 0x08080808u};
        auto scales_fetch = [&](int block) {   // of the 128 inputs `block`
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const __nv_bfloat16* sp = sptr[h] + block * kGroups;
                const uint8_t* zp = zptr[h] + block * kGroups;
                if (kGroups == 4) {
                    snew[h] = *reinterpret_cast<const uint2*>(sp);
                    if (p.zeros) znew[h] = *reinterpret_cast<const uint32_t*>(zp);
                } else if (kGroups == 2) {
                    snew[h].x = *reinterpret_cast<const uint32_t*>(sp);
                    if (p.zeros) znew[h] = *reinterpret_cast<const uint16_t*>(zp);
                } else {
                    snew[h].x = *reinterpret_cast<const uint16_t*>(sp);
                    if (p.zeros) znew[h] = *zp;
                }
            }
        };

        float acc[CB][NB][4];
#pragma unroll
        for (int cb = 0; cb < CB; ++cb)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) acc[cb][nb][0] = acc[cb][nb][1] = acc[cb][nb][2] = acc[cb][nb][3] = 0.0f;
        if (wk * S::kKB < blocks_k) scales_fetch(wk * S::kKB);
        x_fetch();
        x_store(0);
        __syncthreads();
        // this lane's word of 32-block w in a stage, and its piece of the rows
        int woff[4 * S::kKB];
#pragma unroll
        for (int w = 0; w < 4 * S::kKB; ++w) woff[w] = g * S::kRow + ((w ^ S::swz(g)) << 4) + t * 4;
        const unsigned char* xfrag = xs + g * (S::kChunk * 2) + (((wk * S::kKB * 16 + t) ^ ((g & 1) << 2)) << 4);
        const unsigned char* xfrag_odd = xfrag + ((g & 1) ? -64 : 64);   // 32-blocks 1 and 3: the XOR of odd rows swaps neighbours
        int slot = 0;
        for (int chunk = 0; chunk < chunks; ++chunk) {
            if (chunk + 1 < chunks) x_fetch();
            if (chunk + S::kStages - 1 < chunks) issue();
            cp_async_commit();
            cp_async_wait<S::kStages - 1>();
            __syncwarp();
            const unsigned char* st = ring + slot * S::kStageBytes;
#pragma unroll
            for (int kb = 0; kb < S::kKB; ++kb) {
                const int block = (chunk * S::kWK + wk) * S::kKB + kb;
                if (block >= blocks_k) break;
                const int next = kb + 1 < S::kKB ? block + 1 : block + 1 + (S::kWK - 1) * S::kKB;   // this warp's next 128-block
                const uint2 scur[2] = {snew[0], snew[1]};
                const uint32_t zcur[2] = {znew[0], znew[1]};
                if (next < blocks_k) scales_fetch(next);
                uint32_t x[NB][4][4];
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint4 v = *reinterpret_cast<const uint4*>((w & 1 ? xfrag_odd : xfrag) + (chunk & 1) * S::kXBytes +
                                                                        nb * 8 * (S::kChunk * 2) + kb * 256 + (w >> 1) * 128);
                        x[nb][w][0] = v.x; x[nb][w][1] = v.y; x[nb][w][2] = v.z; x[nb][w][3] = v.w;
                    }
#pragma unroll
                for (int cb = 0; cb < CB; ++cb) {
                    if (cb >= cbs) break;
                    uint2 sraw[2];
                    uint32_t zraw[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int from = (lane & ~3) + cb;   // (CB <= 4: the lane of the quad that holds block cb)
                        sraw[h].x = __shfl_sync(0xffffffffu, scur[h].x, from);
                        sraw[h].y = kGroups == 4 ? __shfl_sync(0xffffffffu, scur[h].y, from) : 0u;
                        zraw[h] = p.zeros ? __shfl_sync(0xffffffffu, zcur[h], from) : 0x08080808u;
                    }
                    auto scale_of = [&](int h, int gr) {
                        const uint32_t two = gr < 2 ? sraw[h].x : sraw[h].y;
                        return __uint_as_float(gr & 1 ? two & 0xffff0000u : two << 16);
                    };
#pragma unroll
                    for (int gr = 0; gr < kGroups; ++gr) {
                        const uint32_t z0 = w4_zero_pair(zraw[0], gr), z1 = w4_zero_pair(zraw[1], gr);
                        float d[NB][4];
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) d[nb][0] = d[nb][1] = d[nb][2] = d[nb][3] = 0.0f;
#pragma unroll
                        for (int wi = 0; wi < GW; ++wi) {
                            const int w = gr * GW + wi;
                            uint32_t pl[4], ph[4];
                            w4_pairs(*reinterpret_cast<const uint32_t*>(st + woff[kb * 4 + w] + cb * 16 * S::kRow), base, z0, pl);
                            w4_pairs(*reinterpret_cast<const uint32_t*>(st + woff[kb * 4 + w] + (cb * 16 + 8) * S::kRow), base, z1, ph);
                            const uint32_t a0[4] = {pl[0], ph[0], pl[1], ph[1]}, a1[4] = {pl[2], ph[2], pl[3], ph[3]};
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb) mma_bf16_16816(d[nb], a0, x[nb][w][0], x[nb][w][1]);
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb) mma_bf16_16816(d[nb], a1, x[nb][w][2], x[nb][w][3]);
                        }
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            acc[cb][nb][0] += d[nb][0] * scale_of(0, gr);
                            acc[cb][nb][1] += d[nb][1] * scale_of(0, gr);
                            acc[cb][nb][2] += d[nb][2] * scale_of(1, gr);
                            acc[cb][nb][3] += d[nb][3] * scale_of(1, gr);
                        }
                    }
                }
            }
            __syncwarp();   // all lanes are done with the stage before it is refilled
            slot = slot + 1 == S::kStages ? 0 : slot + 1;
            if (chunk + 1 < chunks) x_store((chunk + 1) & 1);   // (that buffer was last read before the previous barrier)
            __syncthreads();
        }
        cp_async_wait<0>();
        __syncthreads();
        // ---- the warps' sums, over the ring: a lane holds columns g and g + 8 of rows 2t and 2t + 1 of every block
        constexpr int kCols = WN * CB * 16;
        float* mypart = part + wk * NB * 8 * kCols + static_cast<int>(c0) * 16;
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
            if (cb >= cbs) break;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                float* row = mypart + (nb * 8 + 2 * t) * kCols + cb * 16 + g;
                row[0] = acc[cb][nb][0];
                row[kCols] = acc[cb][nb][1];
                row[8] = acc[cb][nb][2];
                row[kCols + 8] = acc[cb][nb][3];
            }
        }
        __syncthreads();
        const int cols = min(pass_n * 16, p.n_cols - pass_blk * 16);
        for (int idx = threadIdx.x; idx < p.m_rows * kCols; idx += S::kThreads) {
            const int m = idx / kCols, j = idx % kCols, n = pass_blk * 16 + j;
            if (j >= cols || (m % p.max_batch) >= p.batch) continue;
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < S::kWK; ++w) sum += part[(w * NB * 8 + m) * kCols + j];
            if (p.residual) sum += __bfloat162float(p.residual[m * p.ldr + n]);
            p.c[m * p.ldc + n] = __float2bfloat16_rn(sum);
        }
        if (pass + 1 < passes) __syncthreads();
    }
}

}  // namespace ellm
