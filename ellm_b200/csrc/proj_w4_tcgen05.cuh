// K9: 4-bit weights on the tensor-memory unit - the form of proj_w4.cuh for large weights and for many rows.
//
//     D[n][m] = sum_k W[n][k] x[m][k]:   128 weight rows n are the M side of tcgen05.mma, the activation rows m
//     its N side (16 to 256), so that a handful of rows costs the tensor unit a handful of columns.
//
// What bounds it: up to 32 rows it should be the packed weights from HBM (0.5 byte each), with a prompt chunk the
// products.  What does today is the chain of the warp that issues them: about 1200 clocks for a 128-input block
// whatever the rows (its barriers, the products' issue, the commits), against 100 (16 rows) to 830 (208 rows) of
// products; the unpackers, about 14 instructions per 8 weights, wait for a free buffer more than half of the time.
// Measured: 13 x 28672 x 8192 59 us (117 MB of weights, 2.0 TB/s), 600 x 8192 x 8192 100 to 110 us by what L2 holds
// (731 TFLOP/s at 110).
//   warps 0-7   unpack: two groups of four, one block each in turn; a thread has one weight row.  A warp streams its
//               32 rows' packed words through a private ring of 16-byte asynchronous copies and stores the bf16 pairs
//               into tensor memory, where the MMA takes its A operand from: no shared-memory round trip and no proxy
//               fence (through shared memory, three buffers: 13 x 28672 x 8192 64 -> 76 us, 600 x 8192 x 8192 104 -> 109)
//   warp  8     TMA producer of the rows (m x 256 bytes per 128-input block)
//   warp  9     MMA issuer, owner of tensor memory
//   warps 10-13 drain / epilogue: thread = one weight row
// Tensor memory: columns [0, 256) four unpacked blocks (128 rows x 128 inputs each), [256, 512) accumulators.
// kSmall (up to 32 rows): a block holds q - z, exact in bf16, every group of a block has its own accumulator columns,
// and the drain warps add scale * accumulator to fp32 sums in registers: no rounding but the last.  Otherwise the tile
// holds (q - z) * scale rounded to bf16 (half a step per weight) and tensor memory accumulates over all of K.
// Work split: the (tile, 128-input block) units form one list, cut evenly over one CTA per SM.  A tile that falls to
// one CTA is finished there; of one cut between CTAs each writes its fp32 part, and w4_reduce_kernel adds the parts in
// list order (no atomics: the result does not depend on timing).
#pragma once
#include "proj_tcgen05.cuh"

namespace ellm {

constexpr int kWtThreads = 14 * 32;
constexpr int kWtTileN = 128;
constexpr int kWtWarpPacked = 32 * 64;                 // a warp's packed weights of a block: 2 KB
constexpr int kWtMaxStages = 8;
constexpr int kWtSmemMax = 232448;
constexpr int kWtRingSmall = 7, kWtRing = 2;           // slots of a warp's ring (kSmall / many rows)

enum { kWtWaitIn = 21, kWtWaitInEmpty = 22, kWtWaitUnpacked = 23, kWtWaitUnpackedEmpty = 24, kWtWaitAcc = 25, kWtWaitAccEmpty = 26 };

struct W4TcParams {
    const __nv_bfloat16* scales;   // [n_cols][k / group]
    const uint8_t* zeros;          // or nullptr (8)
    const __nv_bfloat16* residual;
    __nv_bfloat16* c;
    long long ldr, ldc;
    float* part;                   // [2 * CTAs][mt][128]: the parts of cut tiles (first and last of a CTA's run)
    int* status;
    unsigned long long wait_timeout_ns;
    long long units;               // tiles_n * tiles_m * blocks
    int debug_skip_load;           // test hook: block of CTA 0 the producer never loads; -1 = none
    int m_rows, batch, max_batch;
    int n_cols, blocks;            // blocks = k / 128
    int tiles_m, mt;               // rows per tile, a multiple of 16
    int stages;                    // ring of row blocks
};

// packed rings, barriers, slack to align the base to 1024
inline int w4_tc_fixed(int mt) { return (mt <= 32 ? kWtRingSmall : kWtRing) * 8 * kWtWarpPacked + 512 + 1024; }
inline int w4_tc_stages(int mt) {
    const int s = (kWtSmemMax - w4_tc_fixed(mt)) / (mt * 256), most = mt <= 32 ? 4 : kWtMaxStages;
    return s > most ? most : s;
}
inline int w4_tc_smem(int mt) { return w4_tc_fixed(mt) + w4_tc_stages(mt) * mt * 256; }

// A run of units inside one tile.
struct W4Segment {
    int tile_n, tile_m, block0, blocks;
    bool whole;   // all of the tile's blocks
    int slot;     // where its part goes otherwise
};
__device__ __forceinline__ bool w4_segment(const W4TcParams& p, long long u, long long u0, long long u1, W4Segment& s) {
    if (u >= u1) return false;
    const long long tile = u / p.blocks;
    s.block0 = static_cast<int>(u - tile * p.blocks);
    s.blocks = static_cast<int>(min(static_cast<long long>(p.blocks - s.block0), u1 - u));
    // row tiles of the same weights follow one another (a CTA with several finds the packed weights in L2)
    s.tile_m = static_cast<int>(tile % p.tiles_m);
    s.tile_n = static_cast<int>(tile / p.tiles_m);
    s.whole = s.blocks == p.blocks;
    s.slot = 2 * static_cast<int>(blockIdx.x) + (u == u0 ? 0 : 1);
    return true;
}

// 8 weights of a word as four bf16 pairs in input order, (q - z) exactly, times s2 when kScale.  16 + q is the byte
// 0x80 | q << 3 below the byte 0x41.
template <bool kScale>
__device__ __forceinline__ uint4 w4_unpack8(uint32_t word, uint32_t z16, uint32_t s2) {
    uint32_t even, odd;
    asm("lop3.b32 %0, %1, 0x78787878, %2, 0xea;" : "=r"(even) : "r"(word << 3), "r"(0x80808080u));
    asm("lop3.b32 %0, %1, 0x78787878, %2, 0xea;" : "=r"(odd) : "r"(word >> 1), "r"(0x80808080u));
    const uint32_t lo = __byte_perm(even, odd, 0x5140), hi = __byte_perm(even, odd, 0x7362);   // bytes 0..3, 4..7 in order
    uint32_t r[4] = {__byte_perm(lo, 0x41414141u, 0x4140), __byte_perm(lo, 0x41414141u, 0x4342), __byte_perm(hi, 0x41414141u, 0x4140),
                     __byte_perm(hi, 0x41414141u, 0x4342)};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&r[i]), *reinterpret_cast<const __nv_bfloat162*>(&z16));
        if (kScale) v = __hmul2(v, *reinterpret_cast<const __nv_bfloat162*>(&s2));
        r[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}

// kSmall: kMt = 16 or 32 rows per tile and kGW 32-blocks per group; else kMt = 0 (p.mt rows).
template <bool kSmall, int kMt, int kGW>
__global__ void __launch_bounds__(kWtThreads, 1)
proj_w4_tcgen05_kernel(const __grid_constant__ CUtensorMap map_x, const uint8_t* w4, const W4TcParams p) {
    extern __shared__ unsigned char smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    unsigned char* smem = smem_raw + (base - smem_u32(smem_raw));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kGroups = 4 / kGW;                       // groups per block
    const int mt = kSmall ? kMt : p.mt;
    const int stage_bytes = mt * 256;
    constexpr int kRing = kSmall ? kWtRingSmall : kWtRing;
    // [row stages][packed weights: kRing x 2 KB per unpack warp][barriers]
    const uint32_t s_in = base, s_packed = s_in + p.stages * stage_bytes, bar0 = s_packed + kRing * 8 * kWtWarpPacked;
    auto bar_in = [&](int s) { return bar0 + 8u * s; };
    auto bar_in_empty = [&](int s) { return bar0 + 8u * (kWtMaxStages + s); };
    auto bar_un = [&](int b) { return bar0 + 8u * (2 * kWtMaxStages + b); };                // unpacked block b of four
    auto bar_un_empty = [&](int b) { return bar0 + 8u * (2 * kWtMaxStages + 4 + b); };
    auto bar_acc = [&](int b) { return bar0 + 8u * (2 * kWtMaxStages + 8 + b); };
    auto bar_acc_empty = [&](int b) { return bar0 + 8u * (2 * kWtMaxStages + 10 + b); };
    const uint32_t bar_final = bar0 + 8u * (2 * kWtMaxStages + 12);
    unsigned char* tail = smem + (bar0 - base) + 8 * (2 * kWtMaxStages + 14);
    volatile int* abort_word = reinterpret_cast<volatile int*>(tail);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail + 8);

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(bar_in(s), 1);
            mbar_init(bar_in_empty(s), 1);
        }
        for (int b = 0; b < 4; ++b) {
            mbar_init(bar_un(b), 4);
            mbar_init(bar_un_empty(b), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(bar_acc(b), 1);
            mbar_init(bar_acc_empty(b), 4);
        }
        mbar_init(bar_final, 1);
        *abort_word = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (threadIdx.x == 8 * 32) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    long long u0 = 0, u1 = 0;
    assign_range(p.units, gridDim.x, blockIdx.x, &u0, &u1);
    W4Segment sg;

    if (warp < 8) {
        // =============================== unpack ===============================
        // group = warp / 4 takes every other unit of the CTA's run; this thread's row = its tensor-memory lane
        const int group = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
        unsigned char* ring = smem + (s_packed - base) + warp * kRing * kWtWarpPacked;
        // 64-byte row segments; piece c of row i sits at c ^ ((i >> 1) & 3).  A lane copies piece lane & 3 of rows
        // lane / 4 + 8 i of the warp's 32.
        const int pr = lane >> 2, pc = lane & 3;
        const uint32_t pdst = smem_u32(ring) + pr * 64 + ((pc ^ ((pr >> 1) & 3)) << 4);
        const long long row_bytes = static_cast<long long>(p.blocks) * 64, step8 = 8 * row_bytes;
        // the next unit to be requested: its block, row tile, weight row of this lane
        long long iu = u0;
        int islot = 0, iblock = 0, im = 0, in = 0;
        const uint8_t* isrc = w4;
        if (u0 < u1) {
            const long long tile = u0 / p.blocks;
            iblock = static_cast<int>(u0 - tile * p.blocks);
            im = static_cast<int>(tile % p.tiles_m);
            in = static_cast<int>(tile / p.tiles_m) * kWtTileN + (warp & 3) * 32 + pr;
            isrc = w4 + in * row_bytes + iblock * 64 + pc * 16;
        }
        auto advance = [&]() {
            ++iu;
            isrc += 64;
            if (++iblock == p.blocks) {   // the next tile: the same weights for the next row tile, or the next 128
                iblock = 0;
                isrc -= row_bytes;
                if (++im == p.tiles_m) {
                    im = 0;
                    in += kWtTileN;
                    isrc += kWtTileN * row_bytes;
                }
            }
        };
        auto issue = [&]() {
            if (iu < u1) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {   // rows that do not exist: zeros
                    const bool a = in + i * 8 < p.n_cols;
                    cp_async_16(pdst + islot * kWtWarpPacked + i * 512, a ? isrc + i * step8 : w4, a ? 16 : 0);
                }
                islot = islot + 1 == kRing ? 0 : islot + 1;
                advance();
                if (iu < u1) advance();
            }
            cp_async_commit();
        };
        if (group == 1 && iu < u1) advance();
#pragma unroll 1
        for (int i = 0; i < kRing - 1; ++i) issue();
        // zero points and scales of this thread's row, requested one of its blocks ahead
        uint32_t z_next[kGroups];
        __nv_bfloat16 s_next[kGroups];
        auto fetch = [&](int tile_n, int block) {
            const int n = min(tile_n * kWtTileN + r, p.n_cols - 1);
            const long long at = (static_cast<long long>(n) * p.blocks + block) * kGroups;
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                z_next[g] = p.zeros ? p.zeros[at + g] : 8u;
                if (!kSmall) s_next[g] = p.scales[at + g];
            }
        };
        int slot = 0;
        unsigned n_done = 0;      // units of the CTA's run
        bool ok = true;
        for (long long u = u0; ok && w4_segment(p, u, u0, u1, sg); u += sg.blocks) {
            bool have = false;    // the requested zero points are of this segment
            for (int j = 0; j < sg.blocks && ok; ++j, ++n_done) {
                if ((n_done & 1u) != static_cast<unsigned>(group)) continue;
                if (!have) fetch(sg.tile_n, sg.block0 + j);
                have = true;
                uint32_t z16[kGroups], s2[kGroups];
#pragma unroll
                for (int g = 0; g < kGroups; ++g) {
                    const __nv_bfloat162 zz = __float2bfloat162_rn(16.0f + static_cast<float>(z_next[g]));   // exact (z up to 127)
                    z16[g] = *reinterpret_cast<const uint32_t*>(&zz);
                    s2[g] = 0u;
                    if (!kSmall) {
                        const __nv_bfloat162 ss = __bfloat162bfloat162(s_next[g]);
                        s2[g] = *reinterpret_cast<const uint32_t*>(&ss);
                    }
                }
                if (j + 2 < sg.blocks) fetch(sg.tile_n, sg.block0 + j + 2);
                issue();
                cp_async_wait<kRing - 1>();
                __syncwarp();
                const unsigned char* wp = ring + slot * kWtWarpPacked + lane * 64;
                uint4 w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const uint4*>(wp + ((i ^ ((lane >> 1) & 3)) << 4));
                slot = slot + 1 == kRing ? 0 : slot + 1;
                const int b = static_cast<int>(n_done & 3);
                if ((n_done & ~1u) == 4u) asm volatile("griddepcontrol.wait;" ::: "memory");   // from here on the wait is for products (see below)
                if (lane == 0)
                    ok = mbar_wait(bar_un_empty(b), ((n_done >> 2) & 1u) ^ 1u, abort_word, p.status, kWtWaitUnpackedEmpty, p.wait_timeout_ns);
                ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;   // (also: every lane has read its packed words)
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int h = 0; h < 2; ++h) {   // 64 inputs: 32 columns
                    uint32_t pk[32];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint4& v = w[h * 2 + (i >> 2)];
                        const uint32_t word = (i & 3) == 0 ? v.x : (i & 3) == 1 ? v.y : (i & 3) == 2 ? v.z : v.w;
                        const int g = (h * 2 + (i >> 2)) / kGW;
                        const uint4 o = w4_unpack8<!kSmall>(word, z16[g], s2[g]);
                        pk[i * 4 + 0] = o.x; pk[i * 4 + 1] = o.y; pk[i * 4 + 2] = o.z; pk[i * 4 + 3] = o.w;
                    }
                    tmem_st32u(tmem + lane_base + b * 64 + h * 32, pk);
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_un(b));
            }
        }
        cp_async_wait<0>();
    } else if (warp == 8) {
        // =============================== TMA producer ===============================
        if (lane == 0) {
            bool ok = true;
            long long n_done = 0;
            int s = 0;
            uint32_t phase = 1;   // of the slot's "empty": the first round passes at once
            asm volatile("griddepcontrol.wait;" ::: "memory");   // the rows are the previous kernel's output; the weights are not
            asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
            for (long long u = u0; ok && w4_segment(p, u, u0, u1, sg); u += sg.blocks) {
                for (int j = 0; j < sg.blocks && ok; ++j, ++n_done) {
                    ok = mbar_wait(bar_in_empty(s), phase, abort_word, p.status, kWtWaitInEmpty, p.wait_timeout_ns);
                    if (!ok) break;
                    if (!(n_done == p.debug_skip_load && blockIdx.x == 0)) {
                        mbar_arrive_expect_tx(bar_in(s), static_cast<uint32_t>(stage_bytes));
                        for (int h = 0; h < 2; ++h)
                            tma_load_2d(s_in + s * stage_bytes + h * mt * 128, &map_x, bar_in(s), (sg.block0 + j) * 128 + h * 64, sg.tile_m * mt);
                    }
                    if (++s == p.stages) {
                        s = 0;
                        phase ^= 1;
                    }
                }
            }
            if (*abort_word) {   // copies still on their way into shared memory: wait (bounded, quietly) for the last of every slot
                for (int s = 0; s < p.stages; ++s) {
                    const long long last = n_done - 1 - ((n_done - 1 - s) % p.stages + p.stages) % p.stages;
                    if (last >= 0 && !(last == p.debug_skip_load && blockIdx.x == 0))
                        mbar_wait_quiet(bar_in(s), static_cast<uint32_t>((last / p.stages) & 1), 200000ull);
                }
            }
        }
        __syncwarp();
    } else if (warp == 9) {
        // =============================== MMA issuer ===============================
        // The whole warp walks the list, so that descriptors and addresses stay in uniform registers, and one elected
        // lane issues.  A block's barriers are waited for side by side, a lane each (one after the other each costs about
        // 100 clocks even when it is ready).  With one lane doing everything a block took 1100 clocks, whatever the rows.
        // The products need the rows, which are copied in once the previous kernel has finished: that is waited for ahead
        // of the first wait that has a limit, here and in the other roles, so that its time does not count against it.
        asm volatile("griddepcontrol.wait;" ::: "memory");
        bool ok = true;
        unsigned n_done = 0, n_acc = 0;   // blocks; accumulators handed over
        int s = 0;
        uint32_t phase = 0;               // of the slot's "full"
        const uint32_t idesc = umma_idesc_mn(128, static_cast<uint32_t>(mt));
        for (long long u = u0; ok && w4_segment(p, u, u0, u1, sg); u += sg.blocks) {
            for (int j = 0; j < sg.blocks && ok; ++j, ++n_done) {
                const int b = static_cast<int>(n_done & 3), half = static_cast<int>(n_done & 1);
                // (chosen without branches: three divergent ones cost 4 % of a chunk)
                const uint32_t acc_bar = kSmall ? bar_acc_empty(half) : bar_acc_empty(0);
                const uint32_t acc_par = (kSmall ? (n_done >> 1) & 1u : n_acc & 1u) ^ 1u;
                const bool on_acc = lane == 2 && (kSmall || j == 0);
                const uint32_t bar = lane == 1 ? bar_un(b) : on_acc ? acc_bar : bar_in(s);
                const uint32_t par = lane == 1 ? (n_done >> 2) & 1u : on_acc ? acc_par : phase;
                const int code = lane == 1 ? kWtWaitUnpacked : on_acc ? kWtWaitAccEmpty : kWtWaitIn;
                ok = mbar_wait(bar, par, abort_word, p.status, code, p.wait_timeout_ns);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint64_t x_desc = umma_desc(s_in + s * stage_bytes, 0, 1024);   // (a step along K only adds to its address field)
                const uint32_t x_half = static_cast<uint32_t>(mt * 128) >> 4;
                if (elect_one()) {
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) {
                        const uint32_t d = kSmall ? tmem + 256 + (half * 4 + ks / (2 * kGW)) * mt : tmem + 256;
                        const bool first = kSmall ? ks % (2 * kGW) == 0 : j == 0 && ks == 0;
                        umma_bf16_a_tmem(d, tmem + b * 64 + ks * 8, x_desc + (ks >> 2) * x_half + (ks & 3) * 2, idesc, !first);
                    }
                    umma_commit(bar_un_empty(b));
                    umma_commit(bar_in_empty(s));
                    if (kSmall) umma_commit(bar_acc(half));
                    else if (j + 1 == sg.blocks) umma_commit(bar_acc(0));
                }
                __syncwarp();
                if (++s == p.stages) {
                    s = 0;
                    phase ^= 1;
                }
            }
            ++n_acc;
        }
        if (elect_one()) {
            umma_commit(bar_final);   // every MMA has completed before tensor memory is given back
            mbar_wait_quiet(bar_final, 0, *abort_word ? 2000000ull : p.wait_timeout_ns);
        }
        __syncwarp();
    } else {
        // =============================== drain, epilogue ===============================
        const int r = (warp & 3) * 32 + lane;   // tensor-memory lane = weight row of the tile
        const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
        unsigned n_done = 0, n_acc = 0;
        bool ok = true;
        asm volatile("griddepcontrol.wait;" ::: "memory");   // also: outputs, parts and the residual belong to earlier kernels until here
        for (long long u = u0; ok && w4_segment(p, u, u0, u1, sg); u += sg.blocks) {
            const int n = sg.tile_n * kWtTileN + r, m0 = sg.tile_m * mt;
            const bool exists = n < p.n_cols;
            // rows m .. m + 15 of this weight row (the residual's values requested together)
            const bool all_live = p.batch == p.max_batch;
            auto store16 = [&](int m, float* v) {
                if (!sg.whole) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) p.part[(static_cast<long long>(sg.slot) * mt + m + i) * kWtTileN + r] = v[i];
                    return;
                }
                unsigned live = 0;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int row = m0 + m + i;
                    if (exists && row < p.m_rows && (all_live || (row % p.max_batch) < p.batch)) live |= 1u << i;
                }
                if (p.residual) {
                    __nv_bfloat16 res[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if ((live >> i) & 1u) res[i] = p.residual[(m0 + m + i) * p.ldr + n];
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if ((live >> i) & 1u) v[i] += __bfloat162float(res[i]);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if ((live >> i) & 1u) p.c[(m0 + m + i) * p.ldc + n] = __float2bfloat16_rn(v[i]);
            };
            if constexpr (kSmall) {
                float acc[kMt];
#pragma unroll
                for (int m = 0; m < kMt; ++m) acc[m] = 0.0f;
                const __nv_bfloat16* sp = p.scales + static_cast<long long>(exists ? n : p.n_cols - 1) * p.blocks * kGroups;
                float sc[kGroups], sc_next[kGroups];
                auto fetch = [&](int block) {
#pragma unroll
                    for (int g = 0; g < kGroups; ++g) sc_next[g] = __bfloat162float(sp[block * kGroups + g]);
                };
                fetch(sg.block0);
                for (int j = 0; j < sg.blocks && ok; ++j, ++n_done) {
#pragma unroll
                    for (int g = 0; g < kGroups; ++g) sc[g] = sc_next[g];
                    if (j + 1 < sg.blocks) fetch(sg.block0 + j + 1);
                    const int b = static_cast<int>(n_done & 1);
                    if (lane == 0) ok = mbar_wait(bar_acc(b), static_cast<uint32_t>((n_done >> 1) & 1), abort_word, p.status, kWtWaitAcc, p.wait_timeout_ns);
                    ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int g = 0; g < kGroups; ++g) {
#pragma unroll
                        for (int h = 0; h < kMt / 16; ++h) {
                            float v[16];
                            tmem_ld16(tmem + lane_base + 256 + (b * 4 + g) * kMt + h * 16, v);
                            tmem_wait_ld();
#pragma unroll
                            for (int m = 0; m < 16; ++m) acc[h * 16 + m] = fmaf(v[m], sc[g], acc[h * 16 + m]);
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar_acc_empty(b));
                }
                if (!ok) break;
#pragma unroll
                for (int m = 0; m < kMt; m += 16) store16(m, acc + m);
            } else {
                if (lane == 0) ok = mbar_wait(bar_acc(0), n_acc & 1u, abort_word, p.status, kWtWaitAcc, p.wait_timeout_ns);
                ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
                if (!ok) break;
                tc_fence_after();
                for (int m = 0; m < mt; m += 16) {
                    float v[16];
                    tmem_ld16(tmem + lane_base + 256 + m, v);
                    tmem_wait_ld();
                    store16(m, v);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_acc_empty(0));
                ++n_acc;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// Adds the parts of the tiles that were cut between CTAs.  One block per (tile, 8 rows); 128 threads = weight rows.
__global__ void __launch_bounds__(128) w4_reduce_kernel(const W4TcParams p, int ctas) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // (units fit 32 bits: the launch checks)
    const unsigned first = blockIdx.x * static_cast<unsigned>(p.blocks), last = first + p.blocks - 1;
    const unsigned units = static_cast<unsigned>(p.units), q = units / ctas, rem = units % ctas;
    auto cta_of = [&](unsigned u) { return u < (q + 1) * rem ? u / (q + 1) : rem + (u - (q + 1) * rem) / q; };
    const unsigned c0 = cta_of(first), c1 = cta_of(last);
    const int tile_m = static_cast<int>(blockIdx.x % p.tiles_m), n = static_cast<int>(blockIdx.x / p.tiles_m) * kWtTileN + threadIdx.x;
    const int m0 = blockIdx.y * 8, row0 = tile_m * p.mt + m0;
    const unsigned begin0 = c0 < rem ? (q + 1) * c0 : q * c0 + rem;
    // every CTA after the first begins inside this tile: its part is the first of its run
    const float* src = p.part + (static_cast<long long>(2 * c0 + (begin0 >= first ? 0 : 1)) * p.mt + m0) * kWtTileN + threadIdx.x;
    const float* rest = p.part + (static_cast<long long>(2 * (c0 + 1)) * p.mt + m0) * kWtTileN + threadIdx.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");   // (in every block: this grid's end has to imply the products')
    if (c0 == c1 || n >= p.n_cols) return;   // c0 == c1: finished by the CTA that had all of the tile
    float sum[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] = src[i * kWtTileN];
#pragma unroll 2
    for (unsigned c = c0 + 1; c <= c1; ++c, rest += 2ll * p.mt * kWtTileN)
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] += rest[i * kWtTileN];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int row = row0 + i;
        if (row >= p.m_rows || m0 + i >= p.mt || (row % p.max_batch) >= p.batch) continue;
        if (p.residual) sum[i] += __bfloat162float(p.residual[row * p.ldr + n]);
        p.c[row * p.ldc + n] = __float2bfloat16_rn(sum[i]);
    }
}

}  // namespace ellm
