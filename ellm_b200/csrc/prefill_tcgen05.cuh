// K1 (fast form): causal grouped-query flash-attention prefill on the Blackwell
// tensor cores: tcgen05.mma with accumulators in tensor memory, operands staged in
// shared memory by TMA (no cluster, no multicast), online softmax in fp32.
//
// Replaces, for chunks of many rows, the item walk of the reference's
// Attention::run (src/compiler/mul/attention.rs:85-153) and the per-row key loop
// it calls (src/kernel/generic/flash_attention.rs:60-89): chunk row r of sequence
// b is the token at position base + r and attends keys 0..=base + r.
//
// A work item is 256 packed rows of one (sequence, KV head): packed row rho = r*G + g
// (g = query head inside its group, fastest), split in two tiles of 128 rows, so
// the G query heads of a group share every K/V tile - the reference's "one KV
// head at a time" locality.  One CTA per SM walks the list of items (heaviest
// first, the next untaken one from a device counter).  Warp roles:
//   warps 0-3  softmax / correction / epilogue of tile 0 (thread = one row)
//   warps 4-7  the same for tile 1
//   warp  8    TMA producer (one lane): Q tiles once, then K_j, V_j through a ring
//   warp  9    MMA issuer (one lane) and owner of the tensor-memory allocation
// Per 128-key tile j and row tile t:  S_t = Q_t K_j^T (tensor memory) -> softmax
// threads read S_t half a row at a time, write P_t (bf16) back into the first 64
// columns of S_t (the first half's P before the second half's scores are fetched)
// and, when the running max moved by more than 2^8, rescale O_t in tensor memory ->
// O_t += P_t V_j with P_t read from tensor memory as the A operand.
// The two row tiles alternate on the tensor core, so one tile's softmax overlaps
// the other's MMAs.
//
// Every wait is bounded (about two seconds): when one runs out the kernel sets a
// status word, all roles leave their loops, tensor memory is released and the
// kernel returns; the host turns the status into ELLM_ERR_DEVICE_TIMEOUT.
//
// kExt instantiations (score_mods.cuh): scores capped and biased, a key interval per row, key tiles of a
// shared prefix ahead of the sequence's own, and any group of up to 128 query heads (a row tile holds the
// floor(128 / G) positions that fit).  An item walks the 128-key tiles from the first to the last key any of
// its rows sees; a tile that some row of a row tile does not see whole is exponentiated under per-row bit masks,
// in the same one-pass step.  The interval hulls come from a table filled by a small kernel ahead
// of this one (row_begin), or follow from the positions alone.
// What bounds it: the softmax warps.  A 128-key step of both row tiles takes about 3700 clocks plain, 5000 capped
// (six multiply-adds a score for the tanh) and 4300 biased, against 2800 for its products; an item costs about
// 11000 clocks besides its steps (queries, first tile, epilogue), which is what short documents and windows pay.
// Measured, 128-element heads: capped 16384-token prompt, 32 / 4 heads, 2.55 to 2.75 ms by the GPU's clocks (800 to 860
// TFLOP/s); 2 x 8191 tokens of documents of about 900, biased, 32 / 8 heads, 374 us; 8 x 256 rows under a capped 1024-key
// window, 64 / 8 heads, 145 us; 16 x 48 rows after 8190 shared keys, 32 / 4 heads, 159 us (650 TFLOP/s).
// An item owns all keys of its rows: a chunk of fewer items than SMs leaves the others idle (1 x 64 rows after 8190 keys is
// 8 items, 188 us capped; 1 x 16 rows after 32768 shared keys 4 items, 507 us).
//
// kExtSplit: the shared-prefix part of a decode step.  The rows are the step's query rows (chunk row =
// sequence), the keys the prefix alone, cut into `splits` runs of tiles so that every SM has work, and the
// result is one fp32 partial (O, LSE) per run; the sequences' own keys go through the split-KV kernel and its
// merge takes these partials in.  The prefix is read once per 256 query rows of a KV head instead of once per
// sequence.  A K/V tile is used by one or two CTAs only and comes from HBM: two further warps load the tiles with
// 16-byte asynchronous copies instead of the TMA producer (64 sequences of 32 / 4 heads on 32768 keys: 99 -> 94 us
// when that was introduced).  That step takes 81 us now, 134 MB of prefix and own keys: not the stream but the chain of
// a step (4000 to 5000 clocks), 10000 clocks to the first tile and 4000 of epilogue bound it - the same step on a
// prefix that stays in L2 takes as long.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cmath>
#include <type_traits>

#include "../../include/ellm_attn.h"
#include "common.cuh"
#include "score_mods.cuh"

namespace ellm {

constexpr int kTcTileRows = 128;   // rows per tile = tensor-memory lanes
constexpr int kTcTiles = 2;        // row tiles per CTA
constexpr int kTcKeys = 128;       // keys per K/V tile
constexpr int kTcStages = 5;       // ring slots, each holds one K or one V tile
constexpr int kTcTileBytes = kTcKeys * kRowBytes;          // 32 KB: two 16 KB halves of 128 rows x 128 B
constexpr int kTcHalfBytes = kTcTileBytes / 2;
constexpr int kTcThreads = (kTcTiles * 4 + 2) * 32;        // 320
constexpr int kTcLoaders = 2;                              // kExtSplit: warps that copy K/V tiles, half a tile each
constexpr int kTcSplitThreads = kTcThreads + kTcLoaders * 32;
constexpr int kTcSmemQ = 0;
constexpr int kTcSmemRing = kTcSmemQ + kTcTiles * kTcTileBytes;
constexpr int kTcSmemBar = kTcSmemRing + kTcStages * kTcTileBytes;
constexpr int kTcSmemBytes = kTcSmemBar + 256 + 1024;       // barriers + slack to align the base to 1024
constexpr float kTcRescaleThreshold = 8.0f;                 // log2 units
constexpr float kTcSumTrigger = 65536.0f;                   // a fast-path step whose row sum reaches this is redone with a rescale
#ifndef ELLM_TC_POLY_EVERY
#define ELLM_TC_POLY_EVERY 0
#endif
constexpr int kTcPolyEvery = ELLM_TC_POLY_EVERY;            // every n-th pair of a row uses the polynomial exp2 (0 = none)
constexpr int kTcPolyDiv = kTcPolyEvery > 0 ? kTcPolyEvery : 1;   // the divisor the selection below may use

struct Tcgen05Plan {
    bool ready = false;
    char why[160] = "";
    void* encode = nullptr;  // cuTensorMapEncodeTiled, fetched from the driver at run time
    int sm_count = 0;
    // the tensor maps of the last launch, reused when the next one has the same geometry
    CUtensorMap map_q, map_k, map_v, map_kn, map_vn;
    bool cached_fused = false;
    size_t cached_interval = 0, cached_batch = 0;
    long long cached_kv_rows = -1;
    const void* cached_q = nullptr;
    unsigned long long wait_timeout_ns = 2000000000ull;   // ellm_attn_set_option("tc_wait_timeout_ns")
    int debug_skip_item = -1;                              // ellm_attn_set_option("tc_debug_skip_kv_item")
    int persistent = -1;                                   // ellm_attn_set_option("tc_persistent"): -1 auto, 0 one CTA per item, 1 one CTA per SM
    int fuse_append = 1;                                   // ellm_attn_set_option("tc_fuse_append"): 0 keeps the separate append kernel
    int* sched = nullptr;                                  // the item counter and the exit counter of the one-CTA-per-SM form (the handle's)
    // kExt: any group of up to 128 heads; the tensor maps of the last such launch and what they depend on
    bool ready_ext = false;
    int4* ranges = nullptr;                                // key ranges of every row tile (the handle's), when row_begin is set
    struct ExtKey {
        long long kv_rows = -1;
        size_t interval = 0, batch = 0;
        const void *pk = nullptr, *pv = nullptr;
        long long ps1 = 0, ps2 = 0, plen = 0;
        bool operator==(const ExtKey& o) const {
            return kv_rows == o.kv_rows && interval == o.interval && batch == o.batch && pk == o.pk && pv == o.pv && ps1 == o.ps1 &&
                   ps2 == o.ps2 && plen == o.plen;
        }
    } ext_key;
    CUtensorMap ext_q, ext_k, ext_v, ext_pk, ext_pv;
};

// kExt, capped scores: the form used past the polynomial's range is off by 1e-7 of cap whatever the score, which above
// kTcCapMax would pass 1e-5 of an exponent (such chunks go to the warp-level kernel); up to kTcFixedMaxCap in log2 units the
// softmax takes 0 for the row maximum: exp2 of +-88 and sums of 2^20 such are far from the ends of fp32's range.
// (cap_in's 11th power is folded into a coefficient: it has to stay in fp32's range)
constexpr float kTcCapMax = 128.0f, kTcCapInMin = 1.0f / 4096.0f, kTcCapInMax = 2048.0f;
constexpr float kTcFixedMaxCap = 88.0f;
// kExt bits
enum { kExtOn = 1, kExtCap = 2, kExtBias = 4, kExtSplit = 8 };

struct TcExt {
    ScoreMods mods;
    const int4* ranges = nullptr;   // [batch][tiles]: (first key, end, last "lo", first "hi") of a row tile's rows; nullptr: from the positions
    int tile_pos = 0;               // positions per row tile = 128 / group
    int tiles = 0;                  // row tiles per sequence
    int prefix_tiles = 0;           // 128-key tiles of the shared prefix
    int splits = 1;                 // kExtSplit: runs of prefix tiles, each with its own partial result
    long long part_rows = 0;        // kExtSplit: rows of one partial
    float cap_coef[6] = {};         // the tanh polynomial in the product itself: coefficient of t^(2i+1), times cap_log2
    // q and the cache, for the rows recomputed key by key
    const __nv_bfloat16* q = nullptr;
    const __nv_bfloat16* k = nullptr;
    const __nv_bfloat16* v = nullptr;
    long long s0 = 0, s1 = 0, s2 = 0;
};

struct TcParams {
    void* out;              // bf16, or fp32 for a partial result over a key window

    float* lse;
    int* status;            // device word: non-zero = a bounded wait ran out
    const int32_t* positions;  // per-sequence position of chunk row 0, or nullptr (then `base` for all)
    long long base;         // position of chunk row 0
    long long key_begin;    // rows attend keys [key_begin, min(position + 1, key_end)); key_end for a uniform chunk start only
    long long key_end;
    long long n_items;      // 256-row work items of the launch = pair_tiles * kv_heads * batch
    int* sched;             // two device words, zero between launches: [0] items handed out beyond the first
                            // one per CTA, [1] CTAs that have finished; nullptr = one item per CTA (grid = n_items)
    long long max_seq;      // rows per (sequence, kv head) in the cache
    int interval, batch, max_batch;
    int q_heads, kv_heads, group;
    int pair_tiles;         // 256-row CTA tiles per (sequence, kv head) = ceil(interval * group / 256)
    int pair_major;         // CTA order: 1 = all heads of the heaviest tile first, 0 = head by head
    unsigned long long wait_timeout_ns;   // bound of every device-side wait
    int debug_skip_item;    // test hook: ring item (K_0, V_0, K_1, ...) the producer never loads; -1 = none
    float scale_log2;
};
struct TcParamsExt : TcParams {   // of the kExt instantiations
    TcExt ext;
};

// ---------------------------------------------------------------- PTX wrappers
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_arrive_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint32_t mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done;
}

// Bounded wait.  Returns false when the CTA has been told to give up (abort word set by
// any thread) or when this wait itself ran out, in which case it sets both words.
__device__ __noinline__ bool mbar_wait_slow(uint32_t bar, uint32_t parity, volatile int* abort_word, int* status,
                                            int code, unsigned long long timeout_ns) {
    const unsigned long long t0 = global_timer_ns();
    for (;;) {
        for (int i = 0; i < 256; ++i)
            if (mbar_try_wait(bar, parity)) return true;
        if (*abort_word) return false;
        if (global_timer_ns() - t0 > timeout_ns) {
            *abort_word = code;
            atomicCAS(status, 0, code);
            return false;
        }
    }
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort_word, int* status,
                                          int code, unsigned long long timeout_ns) {
    for (int i = 0; i < 64; ++i)
        if (mbar_try_wait(bar, parity)) return true;
    return mbar_wait_slow(bar, parity, abort_word, status, code, timeout_ns);
}

// True in one lane of the (converged) warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1,
                                            int c2, int c3) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
        : "memory");
}
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1,
                                            int c2, int c3, int c4) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
        : "memory");
}

// shared -> global tile store of the same box shape (rows past the map's bound are dropped)
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2, int c3) {
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];"
                 ::"l"(map), "r"(src), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
                 : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read_all() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Shared-memory matrix descriptor, 128-byte swizzle: rows of 128 bytes, 8-row groups
// `sbo` bytes apart, 64-element column blocks `lbo` bytes apart (used by MN-major operands).
__device__ __forceinline__ uint64_t umma_desc(uint32_t smem_addr, uint32_t lbo, uint32_t sbo) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((smem_addr & 0x3ffffu) >> 4);
    d |= static_cast<uint64_t>((lbo >> 4) & 0x3fffu) << 16;
    d |= static_cast<uint64_t>((sbo >> 4) & 0x3fffu) << 32;
    d |= 1ull << 46;   // descriptor version of this architecture
    d |= 2ull << 61;   // SWIZZLE_128B
    return d;
}
// Instruction descriptor: bf16 x bf16 -> fp32, M = 128, N = 128; b_mn_major selects a B
// operand whose N dimension is contiguous in shared memory.
__host__ __device__ constexpr uint32_t umma_idesc(bool b_mn_major) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((128u >> 3) << 17) |
           ((128u >> 4) << 24);
}
__device__ __forceinline__ void umma_bf16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Same with the A operand in tensor memory (128 lanes x 8 columns of packed bf16 pairs per 16-wide K step).
__device__ __forceinline__ void umma_bf16_a_tmem(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                                 uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// 32 consecutive fp32 columns of this thread's tensor-memory lane.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st32u(uint32_t taddr, const uint32_t* r);
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const float (&v)[32]) {
    tmem_st32u(taddr, reinterpret_cast<const uint32_t*>(v));
}
__device__ __forceinline__ void tmem_st32u(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
          "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
          "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st16u(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ---- packed fp32 pair arithmetic and the exp2 helpers of the softmax passes ----
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// 2^x for a pair, x <= ~8, without the exp2 unit: x = n + f with n = round(x) (magic-number
// add), 2^f from a degree-3 polynomial on [-0.5, 0.5] (max relative error 7.5e-5, below the
// bf16 rounding P gets anyway), 2^n added into the exponent field.
__device__ __forceinline__ uint64_t exp2_poly2(uint64_t x2) {
    float x0, x1;
    unpack2(x2, x0, x1);
    const uint64_t xc = pack2(fmaxf(x0, -126.0f), fmaxf(x1, -126.0f));
    const uint64_t magic = pack2(12582912.0f, 12582912.0f), neg_magic = pack2(-12582912.0f, -12582912.0f);
    const uint64_t r2 = add2(xc, magic);              // low mantissa bits now hold round(x)
    const uint64_t n2 = add2(r2, neg_magic);          // round(x) as a float
    const uint64_t f2 = fma2(n2, pack2(-1.0f, -1.0f), xc);
    uint64_t p2 = fma2(f2, pack2(0.0551716685295105f, 0.0551716685295105f), pack2(0.2426111251115799f, 0.2426111251115799f));
    p2 = fma2(p2, f2, pack2(0.6932609677314758f, 0.6932609677314758f));
    p2 = fma2(p2, f2, pack2(0.9999280571937561f, 0.9999280571937561f));
    float r0, r1, p0, p1;
    unpack2(r2, r0, r1);
    unpack2(p2, p0, p1);
    const float y0 = __int_as_float(__float_as_int(p0) + (__float_as_int(r0) << 23));
    const float y1 = __int_as_float(__float_as_int(p1) + (__float_as_int(r1) << 23));
    return pack2(y0, y1);
}

// Optional per-CTA time stamps for tuning (compiled in only with -DELLM_TC_TRACE): slot -> SM clock.
#ifdef ELLM_TC_TRACE
__device__ long long g_tc_trace[1024 * 64];
#define TC_TRACE(slot)                                                                   \
    do {                                                                                 \
        if (blockIdx.x < 1024 && (slot) < 64) g_tc_trace[blockIdx.x * 64 + (slot)] = clock64(); \
    } while (0)
#define TC_TRACE_NS(slot)                                                                \
    do {                                                                                 \
        if (blockIdx.x < 1024 && (slot) < 64) g_tc_trace[blockIdx.x * 64 + (slot)] = static_cast<long long>(global_timer_ns()); \
    } while (0)
#else
#define TC_TRACE(slot) do {} while (0)
#define TC_TRACE_NS(slot) do {} while (0)
#endif

// Status codes written by a wait that ran out (which wait gave up).
enum { kTcWaitQ = 1, kTcWaitKvFull = 2, kTcWaitKvEmpty = 3, kTcWaitSFull = 4, kTcWaitPFull = 5, kTcWaitPvDone = 6,
       kTcWaitQEmpty = 7, kTcWaitSched = 8 };

// One work item: 256 packed rows (two 128-row tiles) of one (sequence, KV head).
struct TcItem {
    int pair, kvh, b;
    long long base;      // position of the sequence's chunk row 0
    long long key_end;   // rows attend keys [key_begin, min(position + 1, key_end))
    int j0;              // first 128-key tile of the window
    int lo;              // first visible column of that tile (key_begin - 128 * j0)
    int steps[kTcTiles]; // key tiles row tile t needs (0: no valid row, or no key of the window in reach)
    int nsteps;
    bool zero_tail;
};
// kExt: key tiles of the shared prefix (counted in steps), then own tiles from j0 on; row tile t sees the own
// keys [flo, fhi) whole.
// With a distance bias the own tiles are walked from the last to the first: the nearest keys, whose scores the bias
// lowers least, set the maximum at once (from first to last a steep head's maximum leaps in every tile).
struct TcItemExt : TcItem {
    int np;
    int p0 = 0, split = 0;   // kExtSplit: first prefix tile of the item's run
    int flo[kTcTiles], fhi[kTcTiles];
};

// The items are numbered heaviest first: later row tiles have more keys.  When all heads' K/V fit
// in L2 together the order is heaviest-first over the whole launch, else head by head so that one
// head's K/V stays resident while its row tiles are worked off.  A CTA starts with item blockIdx.x
// and then takes the next item nobody has taken yet (a device counter): long items first, short
// ones fill the ends, whatever the items turn out to cost.
__device__ __forceinline__ void tc_item(const TcParams& p, long long idx, TcItem& it) {
    const int heads = p.kv_heads * p.batch;
    int head;
    if (p.pair_major) {
        it.pair = p.pair_tiles - 1 - static_cast<int>(idx / heads);
        head = static_cast<int>(idx % heads);
    } else {
        head = static_cast<int>(idx / p.pair_tiles);
        it.pair = p.pair_tiles - 1 - static_cast<int>(idx % p.pair_tiles);
    }
    it.kvh = head % p.kv_heads;
    it.b = head / p.kv_heads;
    // where this sequence's chunk starts and where its keys end
    it.base = p.positions ? static_cast<long long>(p.positions[it.b]) : p.base;
    it.key_end = p.positions ? min(it.base + p.interval, p.max_seq) : p.key_end;
    it.j0 = static_cast<int>(p.key_begin / kTcKeys);
    it.lo = static_cast<int>(p.key_begin - static_cast<long long>(it.j0) * kTcKeys);
    const int total_rows = p.interval * p.group;
    it.nsteps = 0;
#pragma unroll
    for (int t = 0; t < kTcTiles; ++t) {
        const int rho0 = (it.pair * kTcTiles + t) * kTcTileRows;
        int s = 0;
        if (rho0 < total_rows) {
            const int rho_last = min(rho0 + kTcTileRows, total_rows) - 1;
            long long kend = it.base + rho_last / p.group + 1;
            if (kend > it.key_end) kend = it.key_end;
            s = static_cast<int>((kend + kTcKeys - 1) / kTcKeys) - it.j0;
            if (s < 0) s = 0;
        }
        it.steps[t] = s;
        it.nsteps = max(it.nsteps, s);
    }
    // With per-sequence chunk starts the K/V tensor maps are bounded by the cache, not by this
    // sequence's end, so the last V tile may carry rows past key_end that hold anything; their P
    // is 0 but 0 * NaN is NaN, so the producer zeroes them before the MMA may read the tile.
    it.zero_tail = p.positions != nullptr && static_cast<long long>(it.j0 + it.nsteps) * kTcKeys > it.key_end;
}

// kExt: what row tile `tile` of sequence b needs of the sequence's own keys, without a table.
__device__ __forceinline__ int4 tc_range_of_positions(const TcParamsExt& p, int b, long long base, long long end, int tile) {
    const long long p0 = base + static_cast<long long>(tile) * p.ext.tile_pos;
    const long long p1 = min(p0 + p.ext.tile_pos, base + p.interval) - 1;
    const long long pre = p.ext.mods.prefix_lens ? p.ext.mods.prefix_lens[b] : 0;
    const long long ke = max(0ll, min(max(p1 + 1, pre), end));
    long long fhi = p0 < 0 ? 0 : min(max(p0 + 1, pre), end);
    return make_int4(0, static_cast<int>(ke), 0, static_cast<int>(max(0ll, fhi)));
}

__device__ __forceinline__ void tc_item(const TcParamsExt& p, long long idx, TcItemExt& it) {
    {
        const int heads = p.kv_heads * p.batch;
        int head;
        if (p.pair_major) {
            it.pair = p.pair_tiles - 1 - static_cast<int>(idx / heads);
            head = static_cast<int>(idx % heads);
        } else {
            head = static_cast<int>(idx / p.pair_tiles);
            it.pair = p.pair_tiles - 1 - static_cast<int>(idx % p.pair_tiles);
        }
        it.kvh = head % p.kv_heads;
        it.b = head / p.kv_heads;
        it.base = p.positions ? static_cast<long long>(p.positions[it.b]) : p.base;
        it.key_end = p.positions ? min(it.base + p.interval, p.max_seq) : p.key_end;
        it.np = p.ext.prefix_tiles;
        it.lo = 0;
        int4 r[kTcTiles];
        int j0 = 0x7fffffff;
#pragma unroll
        for (int t = 0; t < kTcTiles; ++t) {
            const int tile = it.pair * kTcTiles + t;
            r[t] = make_int4(0, 0, 0, 0);
            if (tile < p.ext.tiles)
                r[t] = p.ext.ranges ? p.ext.ranges[it.b * p.ext.tiles + tile] : tc_range_of_positions(p, it.b, it.base, it.key_end, tile);
            if (r[t].x < r[t].y) j0 = min(j0, r[t].x / kTcKeys);
            it.flo[t] = r[t].z;
            it.fhi[t] = r[t].w;
        }
        it.j0 = j0 == 0x7fffffff ? 0 : j0;
        it.nsteps = 0;
#pragma unroll
        for (int t = 0; t < kTcTiles; ++t) {
            const bool rows = it.pair * kTcTiles + t < p.ext.tiles;
            it.steps[t] = rows ? it.np + (r[t].x < r[t].y ? (r[t].y + kTcKeys - 1) / kTcKeys - it.j0 : 0) : 0;
            it.nsteps = max(it.nsteps, it.steps[t]);
        }
        if (p.ext.mods.slopes)   // walked backwards: both row tiles start at the last tile (masked for the one it lies beyond)
#pragma unroll
            for (int t = 0; t < kTcTiles; ++t)
                if (it.steps[t] > 0) it.steps[t] = it.nsteps;
        // as in tc_item, for the last own tile (a prefix tile is cut by its tensor map)
        it.zero_tail = p.positions != nullptr && it.nsteps > it.np &&
                       static_cast<long long>(it.j0 + it.nsteps - it.np) * kTcKeys > it.key_end;
    }
}

struct TcItemSplit : TcItemExt {};
__device__ __forceinline__ void tc_item(const TcParamsExt& p, long long idx, TcItemSplit& it) {
    // the runs of one (row pair, head) first, so that the items running together share a head's keys in L2
    it.split = static_cast<int>(idx % p.ext.splits);
    const int rest = static_cast<int>(idx / p.ext.splits);
    it.pair = rest % p.pair_tiles;
    it.kvh = rest / p.pair_tiles;
    it.b = 0;
    it.base = 0;
    it.key_end = 0;
    it.lo = 0;
    it.j0 = 0;
    it.zero_tail = false;
    long long a = 0, z = 0;
    assign_range(p.ext.prefix_tiles, p.ext.splits, it.split, &a, &z);
    it.p0 = static_cast<int>(a);
    it.np = it.nsteps = static_cast<int>(z - a);
#pragma unroll
    for (int t = 0; t < kTcTiles; ++t) {
        it.steps[t] = it.pair * kTcTiles + t < p.ext.tiles ? it.np : 0;
        it.flo[t] = it.fhi[t] = 0;
    }
}

// The key ranges of every row tile, from row_begin: one block per (row tile, sequence).
__global__ void __launch_bounds__(128) tc_ranges_kernel(const ScoreMods m, const int32_t* positions, long long base_all, int interval,
                                                        long long max_seq, int tile_pos, int tiles, int4* out) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ int s[4];   // first key, end, last lo, first hi
    const int tile = blockIdx.x, b = blockIdx.y;
    if (threadIdx.x == 0) { s[0] = 0x7fffffff; s[1] = 0; s[2] = 0; s[3] = 0x7fffffff; }
    __syncthreads();
    const long long base = positions ? static_cast<long long>(positions[b]) : base_all;
    const int r = tile * tile_pos + static_cast<int>(threadIdx.x);
    if (threadIdx.x < tile_pos && r < interval) {
        const long long pos = base + r;
        long long lo, hi;
        row_interval(m, b, pos, min(base + interval, max_seq), lo, hi);
        if (lo < hi) {
            atomicMin(&s[0], static_cast<int>(lo));
            atomicMax(&s[1], static_cast<int>(hi));
        }
        atomicMax(&s[2], static_cast<int>(lo));
        atomicMin(&s[3], static_cast<int>(max(0ll, hi)));
    }
    __syncthreads();
    if (threadIdx.x == 0) out[b * tiles + tile] = s[1] > 0 ? make_int4(s[0], s[1], s[2], s[3]) : make_int4(0, 0, s[2], s[3]);
}

// kExt: a row's constants for turning products into scores.
struct TcRow {
    float scale_log2, cap_in, cap_log2;
    float slope;     // times log2(e)
    float dist0;     // position minus the tile's first key
    bool ahead;      // no visible column lies beyond the row's position (uniform over the warp)
};
// One score in log2 units; column c of the tile.  The capped form here is 1 - 2 / (1 + e^(2u)) with an absolute
// error of 1e-7 cap: the chunk kernel is used up to kTcCapMax.
template <int kExt>
__device__ __forceinline__ float tc_score(const TcRow& r, float t, float c) {
    float x = (kExt & kExtCap) ? fmaf(-2.0f * r.cap_log2, fast_rcp(1.0f + fast_exp2(t * (r.cap_in * 2.0f * kLog2e))), r.cap_log2)
                               : t * r.scale_log2;
    if (kExt & kExtBias) x = fmaf(-r.slope, fabsf(r.dist0 - c), x);
    return x;
}
template <int kExt>
__device__ __forceinline__ float tc_score_in(int col, float t, const TcRow& r, int lo, int rel) {
    return col >= lo && col <= rel ? tc_score<kExt>(r, t, static_cast<float>(col)) : -INFINITY;
}
// A wait of the teardown: bounded, sets no status.
__device__ __noinline__ bool mbar_wait_quiet(uint32_t bar, uint32_t parity, unsigned long long timeout_ns) {
    const unsigned long long t0 = global_timer_ns();
    for (;;) {
        for (int i = 0; i < 64; ++i)
            if (mbar_try_wait(bar, parity)) return true;
        if (global_timer_ns() - t0 > timeout_ns) return false;
    }
}

// Rare tail of the one-pass step: a score among the row's second 64 keys leapt far above the maximum in
// use after the first 64 keys' P had gone to tensor memory.  Finds the second half's true maximum,
// rescales O_t and the stored first half of P_t to it, and recomputes the second half.  Out of line:
// its registers must not be charged to the plain step.
struct TcFixed {
    float m_used, l;
};

// kExt: ext = the row's constants and the visible columns.
template <int kExt, class... Ext>
__device__ __noinline__ TcFixed tc_fix_second_half(uint32_t tS, uint32_t tO, float scale_log2, float m_used, float l,
                                                   float first_half_sum, uint32_t* pk, const Ext... ext) {
    float mx = -INFINITY;
#pragma unroll 1
    for (int c = 0; c < 2; ++c) {
        float v[32];
        tmem_ld32(tS + 64 + c * 32, v);
        tmem_wait_ld();
        if constexpr (kExt != 0)
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = tc_score_in<kExt>(64 + c * 32 + i, v[i], ext...);
        float m0 = max3(v[0], v[1], v[2]), m1 = max3(v[3], v[4], v[5]);
#pragma unroll
        for (int i = 6; i < 30; i += 6) {
            m0 = max3(m0, v[i], v[i + 1]);
            m1 = max3(m1, v[i + 2], v[i + 3]);
            m0 = fmaxf(m0, v[i + 4]);
            m1 = fmaxf(m1, v[i + 5]);
        }
        mx = max3(mx, max3(m0, v[30], v[31]), m1);
    }
    float m_new = fmaxf(m_used, kExt != 0 ? mx : mx * scale_log2);
    // rows whose maximum did not move far keep it (their corr is 1): as in the two-pass step
    bool moved = m_new - m_used > kTcRescaleThreshold;
    if constexpr (kExt != 0) moved = moved && m_new != -INFINITY;
    float corr = moved ? fast_exp2(m_used - m_new) : 1.0f;
    if constexpr (kExt != 0)
        if (moved) {
            // The row moves by whole powers of two (to less than 1 above its maximum), so that the first half's P, rounded to
            // bf16 already, is not rounded again.  A row whose first key is in this half has nothing to bring along.
            const float by = ceilf(m_new - m_used);
            corr = by < 126.0f ? __int_as_float((127 - static_cast<int>(by)) << 23) : 0.0f;
            if (m_used != -INFINITY) m_new = m_used + by;
        }
    if (moved) m_used = m_new;
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {   // O_t: every P.V of earlier steps has completed (this step's S_t exists)
        float o[32];
        tmem_ld32(tO + c * 32, o);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] *= corr;
        tmem_st32(tO + c * 32, o);
    }
    {   // the first half of P_t, bf16 pairs in columns [0, 32)
        uint32_t q[32];
        tmem_ld32(tS, *reinterpret_cast<float(*)[32]>(&q[0]));
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const __nv_bfloat162 h = *reinterpret_cast<const __nv_bfloat162*>(&q[i]);
            q[i] = pack_bf16(__low2float(h) * corr, __high2float(h) * corr);
        }
        tmem_st32u(tS, q);
    }
    const float msub = kExt != 0 && m_used == -INFINITY ? 0.0f : m_used;
    const uint64_t scale2 = pack2(scale_log2, scale_log2), negm2 = pack2(-msub, -msub);
    uint64_t sum_a = pack2(0.0f, 0.0f), sum_b = sum_a;
#pragma unroll 1
    for (int c = 0; c < 2; ++c) {
        float v[32];
        tmem_ld32(tS + 64 + c * 32, v);
        tmem_wait_ld();
        if constexpr (kExt != 0)
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = tc_score_in<kExt>(64 + c * 32 + i, v[i], ext...);
#pragma unroll
        for (int cc = 0; cc < 16; ++cc) {
            const uint64_t x2 = kExt != 0 ? add2(pack2(v[2 * cc], v[2 * cc + 1]), negm2) : fma2(pack2(v[2 * cc], v[2 * cc + 1]), scale2, negm2);
            float x0, x1;
            unpack2(x2, x0, x1);
            const uint64_t p2 = pack2(fast_exp2(x0), fast_exp2(x1));
            if (cc & 1) sum_b = add2(sum_b, p2); else sum_a = add2(sum_a, p2);
            float p0, p1;
            unpack2(p2, p0, p1);
            pk[c * 16 + cc] = pack_bf16(p0, p1);
        }
    }
    float sa, sb;
    unpack2(add2(sum_a, sum_b), sa, sb);
    TcFixed r;
    r.m_used = m_used;
    r.l = (l + first_half_sum) * corr + (sa + sb);
    return r;
}

// 64 products of one row -> P and its sum: score, subtraction of the maximum (inside `off`), mask, exp2, rounding,
// pair by pair, so that the polynomial's multiply-adds and the exponentials are in flight together (computing all
// scores first and all exponentials after ran the two units one after the other).
//   kCap: the tanh polynomial with cap_in folded into its coefficients;  kScored: s holds scores already.
//   m0, m1: visible columns;  base, slope: the distance bias of column i is base + slope * i (kExtBias, `ahead`).
template <int kExt, bool kScored, bool kMask>
__device__ __forceinline__ float tc_exp64(const float (&s)[64], const TcRow& r, const float (&coef)[6], float base, unsigned m0, unsigned m1,
                                          uint32_t (&pk)[32]) {
    const uint64_t base2 = pack2(base, base), scale2 = pack2(r.scale_log2, r.scale_log2);
    uint64_t sum_a = pack2(0.0f, 0.0f), sum_b = sum_a;
#pragma unroll
    for (int c = 0; c < 32; ++c) {
        const int i = 2 * c;
        const uint64_t s2 = pack2(s[i], s[i + 1]);
        uint64_t add = base2, x2;
        if constexpr ((kExt & kExtBias) != 0 && !kScored) add = pack2(fmaf(r.slope, static_cast<float>(i), base), fmaf(r.slope, static_cast<float>(i + 1), base));
        if constexpr (kScored) {
            x2 = add2(s2, base2);
        } else if constexpr ((kExt & kExtCap) != 0) {
            const uint64_t v = mul2(s2, s2);
            uint64_t q = fma2(pack2(coef[5], coef[5]), v, pack2(coef[4], coef[4]));
            q = fma2(q, v, pack2(coef[3], coef[3]));
            q = fma2(q, v, pack2(coef[2], coef[2]));
            q = fma2(q, v, pack2(coef[1], coef[1]));
            q = fma2(q, v, pack2(coef[0], coef[0]));
            x2 = fma2(s2, q, add);
        } else {
            x2 = fma2(s2, scale2, add);
        }
        float x0, x1;
        unpack2(x2, x0, x1);
        if constexpr (kMask) {
            const unsigned m = c < 16 ? m0 : m1;
            x0 = (m >> (i & 31)) & 1u ? x0 : -INFINITY;
            x1 = (m >> ((i + 1) & 31)) & 1u ? x1 : -INFINITY;
        }
        const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
        if (c & 1) sum_b = add2(sum_b, pack2(p0, p1)); else sum_a = add2(sum_a, pack2(p0, p1));
        pk[c] = pack_bf16(p0, p1);
    }
    float sa, sb;
    unpack2(add2(sum_a, sum_b), sa, sb);
    return sa + sb;
}
template <int kExt>
__device__ __forceinline__ float tc_row64(float (&s)[64], const TcRow& r, const float (&coef)[6], float c0, float off, bool edge, int lo, int rel,
                                          bool valid, uint32_t (&pk)[32]) {
    unsigned m0 = ~0u, m1 = ~0u;
    if (edge) {
        const unsigned long long below = rel < 0 ? 0ull : rel >= 63 ? ~0ull : (2ull << rel) - 1ull;
        const unsigned long long from = lo <= 0 ? ~0ull : lo >= 64 ? 0ull : ~0ull << lo;
        m0 = static_cast<unsigned>(below & from);
        m1 = static_cast<unsigned>((below & from) >> 32);
    }
    const float d = r.dist0 - c0, base = (kExt & kExtBias) ? off - r.slope * d : off;
    bool direct = true;
    if constexpr ((kExt & kExtCap) != 0) {
        // Which form the warp takes follows from what its rows see alone: masked products count as 0, and lanes without a
        // row, whose queries are whatever the tile held before, have no say.
        if (edge)
#pragma unroll
            for (int i = 0; i < 64; ++i) s[i] = ((i < 32 ? m0 : m1) >> (i & 31)) & 1u ? s[i] : 0.0f;
        float a0 = max3(fabsf(s[0]), fabsf(s[1]), fabsf(s[2])), a1 = max3(fabsf(s[3]), fabsf(s[4]), fabsf(s[5]));
#pragma unroll
        for (int i = 6; i < 62; i += 4) {
            a0 = max3(a0, fabsf(s[i]), fabsf(s[i + 1]));
            a1 = max3(a1, fabsf(s[i + 2]), fabsf(s[i + 3]));
        }
        a0 = max3(a0, fabsf(s[62]), fabsf(s[63]));
        direct = __all_sync(0xffffffffu, fmaxf(a0, a1) * r.cap_in <= kTanhPolyMax || !valid);
    }
    if constexpr ((kExt & kExtBias) != 0) direct = direct && r.ahead;
    if (direct) return edge ? tc_exp64<kExt, false, true>(s, r, coef, base, m0, m1, pk) : tc_exp64<kExt, false, false>(s, r, coef, base, m0, m1, pk);
    if constexpr ((kExt & (kExtCap | kExtBias)) != 0) {   // scores past the polynomial's range, or keys past the position
#pragma unroll
        for (int i = 0; i < 64; ++i) s[i] = tc_score<kExt>(r, s[i], c0 + static_cast<float>(i));
        return tc_exp64<kExt, true, true>(s, r, coef, off, m0, m1, pk);
    }
    return 0.0f;
}

// The largest visible score of a key tile, for rows that have seen no key before it (they have l = 0 and nothing in
// O_t, so the one-pass step can go on from it).  Rolled like the two-pass step.
template <int kExt>
__device__ __forceinline__ float tc_first_max(uint32_t tS, const TcRow& r, int lo, int rel) {
    float mx = -INFINITY;
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
        float v[32];
        tmem_ld32(tS + c * 32, v);
        tmem_wait_ld();
        const int l0 = lo - c * 32, r0 = rel - c * 32;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            float x = (kExt & kExtBias) ? tc_score<kExt>(r, v[i], static_cast<float>(c * 32 + i)) : v[i];
            mx = fmaxf(mx, i >= l0 && i <= r0 ? x : -INFINITY);
        }
    }
    if constexpr ((kExt & kExtBias) == 0)
        if (mx != -INFINITY) mx = tc_score<kExt>(r, mx, 0.0f);   // the score grows with the product
    return mx;
}

// The two-pass step of a kExt row tile: the true maximum, O_t rescaled to it where it moved far, then P.  Taken when
// a score leaps far above the maximum in use.  32 columns at a time in a rolled
// loop: it is rare, and its code must not push the one-pass step's out of the instruction cache.
template <int kExt>
__device__ __forceinline__ void tc_two_pass(uint32_t tS, uint32_t tO, const TcRow& r, int lo, int rel, bool rescale_o, bool valid, float& m_used, float& l) {
    float mx = -INFINITY;
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
        float v[32];
        tmem_ld32(tS + c * 32, v);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const int col = c * 32 + i;
            mx = fmaxf(mx, col >= lo && col <= rel ? tc_score<kExt>(r, v[i], static_cast<float>(col)) : -INFINITY);
        }
    }
    const float m_new = fmaxf(m_used, mx);
    const bool need = (m_new - m_used > kTcRescaleThreshold) || (m_used == -INFINITY && m_new != -INFINITY);
    const bool rescale = __any_sync(0xffffffffu, need && valid);   // (lanes without a row hold left-overs)
    float corr = 1.0f;
    if (rescale) {
        corr = (m_used == -INFINITY) ? 0.0f : fast_exp2(m_used - m_new);
        m_used = m_new;
    }
    const float msub = (m_used == -INFINITY) ? 0.0f : m_used;
    if (rescale && rescale_o) {
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
            float o[32];
            tmem_ld32(tO + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] *= corr;
            tmem_st32(tO + c * 32, o);
        }
    }
    float sum = 0.0f;
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {   // P of 32 columns takes 16, which never overlap columns of S_t not yet read
        float v[32];
        uint32_t pk[16];
        tmem_ld32(tS + c * 32, v);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const int col = c * 32 + i;
            v[i] = fast_exp2(col >= lo && col <= rel ? tc_score<kExt>(r, v[i], static_cast<float>(col)) - msub : -INFINITY);
            sum += v[i];
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) pk[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
        tmem_st16u(tS + c * 16, pk);
    }
    l = l * corr + sum;
}

// One key tile of a kExt row tile: P_t in tensor memory on return.  fixed_max: the scores are bounded (capped, no
// bias), m_used is a constant for the whole row and nothing can leap.
template <int kExt>
__device__ __forceinline__ void tc_step_ext(uint32_t tS, uint32_t tO, const TcRow& r, const float (&coef)[6], int lo, int rel, bool edge,
                                            bool first, bool fixed_max, bool valid, float& m_used, float& l) {
    bool slow = false;
    if (!fixed_max && __any_sync(0xffffffffu, m_used == -INFINITY && valid)) {
        const float m = tc_first_max<kExt>(tS, r, edge ? lo : 0, edge ? rel : 127);
        if (m_used == -INFINITY) m_used = m;
    }
    {
        float sum0 = 0.0f;
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
            float s[64];
            tmem_ld32(tS + half * 64, *reinterpret_cast<float(*)[32]>(&s[0]));
            tmem_ld32(tS + half * 64 + 32, *reinterpret_cast<float(*)[32]>(&s[32]));
            tmem_wait_ld();
            uint32_t pk[32];
            const float sum = tc_row64<kExt>(s, r, coef, static_cast<float>(half * 64), m_used == -INFINITY ? 0.0f : -m_used, edge, lo - half * 64,
                                             rel - half * 64, valid, pk);   // (a row without any key yet: all masked)
            const bool leapt = !fixed_max && __any_sync(0xffffffffu, !(sum < kTcSumTrigger) && valid);
            if (!leapt) {
                tmem_st32u(tS + half * 32, pk);
                if (half == 0) sum0 = sum; else l += sum0 + sum;
            } else if (half == 0) {   // S_t is still intact: the whole step in two passes
                slow = true;
                break;
            } else {                  // the first half's P is already in place: bring it and O_t to the new maximum
                uint32_t redone[32];
                const TcFixed f = tc_fix_second_half<kExt>(tS, tO, 0.0f, m_used, l, sum0, redone, r, edge ? lo : 0, edge ? rel : 127);
                m_used = f.m_used;
                l = f.l;
                tmem_st32u(tS + 32, redone);
            }
        }
    }
    if (slow) tc_two_pass<kExt>(tS, tO, r, edge ? lo : 0, edge ? rel : 127, !first, valid, m_used, l);
}

// kFused: the chunk's own K/V rows come from k_new / v_new and are written into the cache here (a
// separate instantiation, so that the plain kernel carries none of its state).
// kExt: modified scores, intervals, shared prefix (map_kn / map_vn are then the prefix's maps).
template <typename OutT, bool kFused, int kExt = 0>
__global__ void __launch_bounds__((kExt & kExtSplit) ? kTcSplitThreads : kTcThreads, 1)
prefill_tcgen05_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_kn,
                       const __grid_constant__ CUtensorMap map_vn,
                       const std::conditional_t<kExt != 0, TcParamsExt, TcParams> p) {
    using Item = std::conditional_t<(kExt & kExtSplit) != 0, TcItemSplit, std::conditional_t<kExt != 0, TcItemExt, TcItem>>;
    extern __shared__ unsigned char smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    unsigned char* smem = smem_raw + (smem_base - smem_u32(smem_raw));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) { TC_TRACE_NS(0); TC_TRACE(1); }
    constexpr bool kSplit = (kExt & kExtSplit) != 0;
    if constexpr (!kSplit) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == (kTcTiles * 4) * 32) {   // the producer thread fetches the three descriptors ahead of its first copy
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_q) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
        if (kFused || kExt != 0) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_kn) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_vn) : "memory");
        }
    }

    // barriers (8 bytes each) and two words behind them
    const uint32_t bar0 = smem_base + kTcSmemBar;
    auto bar_q = [&](int t) { return bar0 + 8u * t; };
    auto bar_kv_full = [&](int s) { return bar0 + 8u * (2 + s); };
    auto bar_kv_empty = [&](int s) { return bar0 + 8u * (2 + kTcStages + s); };
    auto bar_s_full = [&](int t) { return bar0 + 8u * (2 + 2 * kTcStages + t); };
    auto bar_p_full = [&](int t) { return bar0 + 8u * (4 + 2 * kTcStages + t); };
    auto bar_pv_done = [&](int t) { return bar0 + 8u * (6 + 2 * kTcStages + t); };
    auto bar_q_empty = [&](int t) { return bar0 + 8u * (8 + 2 * kTcStages + t); };
    const uint32_t bar_tail = bar0 + 8u * (10 + 2 * kTcStages);
    const uint32_t bar_final = bar0 + 8u * (11 + 2 * kTcStages);
    auto bar_sched_full = [&](int s) { return bar0 + 8u * (12 + 2 * kTcStages + s); };    // the item list's two-slot mailbox
    auto bar_sched_empty = [&](int s) { return bar0 + 8u * (14 + 2 * kTcStages + s); };
    constexpr int kNumBars = 16 + 2 * kTcStages;
    static_assert(8 * kNumBars + 24 <= 256, "the barrier block is 256 bytes");
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kTcSmemBar + 8 * kNumBars);
    volatile int* abort_word = reinterpret_cast<volatile int*>(smem + kTcSmemBar + 8 * kNumBars + 8);
    volatile int* sched_idx = reinterpret_cast<volatile int*>(smem + kTcSmemBar + 8 * kNumBars + 16);   // [2]

    if (threadIdx.x == 0) {
        for (int t = 0; t < kTcTiles; ++t) {
            mbar_init(bar_q(t), 1);
            mbar_init(bar_q_empty(t), kSplit ? kTcTileRows / 32 : 1);   // (kExtSplit: the softmax warps, done with it as staging space)
            mbar_init(bar_s_full(t), 1);
            mbar_init(bar_p_full(t), kTcTileRows / 32);   // one arrival per softmax warp
            mbar_init(bar_pv_done(t), 1);
        }
        for (int s = 0; s < kTcStages; ++s) {
            mbar_init(bar_kv_full(s), kSplit ? kTcLoaders : 1);
            mbar_init(bar_kv_empty(s), 1);
        }
        mbar_init(bar_tail, 1);
        mbar_init(bar_final, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar_sched_full(i), 1);
            mbar_init(bar_sched_empty(i), 1 + kTcTiles * 4 + (kSplit ? kTcLoaders : 0));   // the MMA thread, every softmax and loader warp
        }
        *abort_word = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kTcTiles * 4 + 1) {  // the MMA warp owns tensor memory: all 512 columns
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // columns: S_0 [0,128), S_1 [128,256), O_0 [256,384), O_1 [384,512)

    // Launched as a programmatic dependent, the set-up above ran while the stream's previous kernel
    // was still at work; everything below reads or writes what that kernel may have touched.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // the split-KV kernel behind this one reads nothing that this one writes: from here on it may run, and only
    // its end waits for this grid's.  What older kernels wrote is visible here; the fence passes that on.
    if constexpr (kSplit) {
        __threadfence();
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    }
    if (threadIdx.x == 0) TC_TRACE(2);
    const int total_rows = p.interval * p.group;
    const int n_items = static_cast<int>(p.n_items);
    // the k-th item of this CTA as the producer publishes it (n_items = no more)
    auto take_item = [&](long long k, bool& ok, int code) -> int {
        ok = mbar_wait(bar_sched_full(static_cast<int>(k & 1)), static_cast<uint32_t>((k >> 1) & 1), abort_word, p.status, code, p.wait_timeout_ns);
        const int idx = ok ? sched_idx[k & 1] : n_items;
        return idx;
    };

    // Every role walks the same list of items.  What carries over from one item to the next are the
    // barriers' phases, so each role counts what it has pushed through them so far: ring items,
    // key steps per row tile, Q loads per row tile.
    if (warp < kTcTiles * 4) {
        // =============================== softmax / correction / epilogue ===============================
        const int t = warp >> 2;
        const int row = (warp & 3) * 32 + lane;                 // row of the tile = tensor-memory lane
        const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t tS = tmem + lane_base + t * 128;
        const uint32_t tO = tmem + lane_base + 256 + t * 128;
        int steps_done = 0;     // key steps of this row tile over all items so far
        bool ok = true;
        Item it;
        int redo_item = -1;        // kExt: the last item with rows of this warp to be computed again, and which
        unsigned redo_rows = 0;
        int n_traced = 0;
        for (long long k = 0; ok; ++k) {
            int idx = n_items;
            if (lane == 0) idx = take_item(k, ok, kTcWaitSched);
            idx = __shfl_sync(0xffffffffu, idx, 0);
            ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
            if (!ok) break;
            if (lane == 0) mbar_arrive(bar_sched_empty(static_cast<int>(k & 1)));
            if (idx >= n_items) break;
            tc_item(p, idx, it);
            const int tr = 8 + 8 * n_traced + 4 * t;   // trace slots of this item and tile
            ++n_traced;
            int rho = (it.pair * kTcTiles + t) * kTcTileRows + row;
            if constexpr (kExt != 0)   // a row tile holds whole positions
                rho = row < p.ext.tile_pos * p.group ? (it.pair * kTcTiles + t) * p.ext.tile_pos * p.group + row : total_rows;
            const bool valid = rho < total_rows;
            const int pos = valid ? rho / p.group : 0, g = valid ? rho % p.group : 0;
            // kExt: the row's interval of own keys, its constants
            int row_lo = 0, row_hi = 0;
            TcRow xr{};
            float coef[6] = {};
            bool fixed_max = false;
            if constexpr (kExt != 0) {
                if ((kExt & kExtSplit) == 0 && valid) {
                    long long a, z;
                    row_interval(p.ext.mods, it.b, it.base + pos, it.key_end, a, z);
                    row_lo = static_cast<int>(a);
                    row_hi = static_cast<int>(z);
                }
                xr.scale_log2 = p.scale_log2;
                xr.cap_in = p.ext.mods.cap_in;
                xr.cap_log2 = p.ext.mods.cap_log2;
                if ((kExt & kExtBias) && valid) xr.slope = p.ext.mods.slopes[it.kvh * p.group + g] * kLog2e;
                if constexpr ((kExt & kExtCap) != 0)
#pragma unroll
                    for (int i = 0; i < 6; ++i) coef[i] = p.ext.cap_coef[i];
                // capped scores lie in +-cap: with 2^(cap log2 e) far inside fp32's (and bf16's) range the softmax needs no maximum
                fixed_max = (kExt & kExtCap) && !(kExt & kExtBias) && p.ext.mods.cap_log2 <= kTcFixedMaxCap;
            }
            const long long lim = valid ? min(it.base + pos, it.key_end - 1) : -1;   // last key this row may see
            const long long tile_min_lim = min(it.base + ((it.pair * kTcTiles + t) * kTcTileRows) / p.group, it.key_end - 1);
            const int my_steps = it.steps[t];
            long long row_index = (static_cast<long long>(pos) * p.max_batch + it.b) * p.q_heads + it.kvh * p.group + g;
            if constexpr ((kExt & kExtSplit) != 0) row_index += it.split * p.ext.part_rows;
            float m_used = kExt != 0 && fixed_max ? 0.0f : -INFINITY, l = 0.0f;
            for (int j = 0; j < my_steps && ok; ++j) {
                // lane 0 polls the barrier, the warp follows (32 pollers per warp only add shared-memory traffic)
                ok = lane == 0 ? mbar_wait(bar_s_full(t), (steps_done + j) & 1, abort_word, p.status, kTcWaitSFull, p.wait_timeout_ns) : true;
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                if (j == 0 && (warp & 3) == 0 && lane == 0) TC_TRACE(tr);
                tc_fence_after();
                long long key0 = static_cast<long long>(it.j0 + j) * kTcKeys;
                int lo = j == 0 ? it.lo : 0;                           // columns below it lie before the key window
                bool edge = key0 + kTcKeys - 1 > tile_min_lim || lo > 0;   // the causal edge (or the window's start) crosses this tile
                const long long dlim = lim - key0;                     // last column this row may see
                int rel = dlim < 0 ? -1 : (dlim > 127 ? 127 : static_cast<int>(dlim));
                if constexpr (kExt != 0) {
                    if (j < it.np) {   // a tile of the shared prefix: seen whole, up to its end
                        const long long left = p.ext.mods.plen - static_cast<long long>(it.p0 + j) * kTcKeys;
                        lo = 0;
                        rel = left < kTcKeys ? static_cast<int>(left) - 1 : kTcKeys - 1;
                        edge = left < kTcKeys;
                        xr.ahead = true;
                    } else {
                        key0 = static_cast<long long>((kExt & kExtBias) ? it.j0 + it.nsteps - 1 - j : it.j0 + j - it.np) * kTcKeys;
                        lo = min(max(row_lo - static_cast<int>(key0), 0), kTcKeys);
                        rel = min(max(row_hi - static_cast<int>(key0), 0), kTcKeys) - 1;
                        xr.ahead = p.ext.mods.prefix_lens == nullptr ||
                                   key0 + kTcKeys - 1 <= it.base + (it.pair * kTcTiles + t) * static_cast<long long>(p.ext.tile_pos);
                        edge = static_cast<int>(key0) < it.flo[t] || static_cast<int>(key0) + kTcKeys > it.fhi[t];
                    }
                    xr.dist0 = static_cast<float>(static_cast<int>(it.base + pos - key0));
                }
                if constexpr (kExt != 0) {
                    tc_step_ext<kExt>(tS, tO, xr, coef, lo, rel, edge, j == 0, fixed_max, valid, m_used, l);
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar_p_full(t));
                    continue;
                }
                // Fast path (every step but the first, unless a score leaps far above the maximum in use):
                // exponentiate against the maximum already in use, in one pass.  P is held in registers
                // until the step's row sum has shown that nothing leapt - then it is consistent with O
                // and l as they stand and goes to tensor memory as is.  Otherwise S_t is still intact and
                // the two-pass slow path below redoes the step with a rescale of O_t.
                bool slow = (j == 0) || edge;
                if (!slow) {
                    // Half a row at a time: the first 64 keys' P goes to tensor memory (over columns of S_t
                    // that have been read) before the second 64 scores are fetched, so that a thread holds 64
                    // scores and 32 packed P values at most.
                    const uint64_t scale2 = pack2(p.scale_log2, p.scale_log2), negm2 = pack2(-m_used, -m_used);
                    uint32_t pk[32];
                    float half_sum[2];
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        float s[64];
                        tmem_ld32(tS + half * 64, *reinterpret_cast<float(*)[32]>(&s[0]));
                        tmem_ld32(tS + half * 64 + 32, *reinterpret_cast<float(*)[32]>(&s[32]));
                        tmem_wait_ld();
                        uint64_t sum_a = pack2(0.0f, 0.0f), sum_b = sum_a;
#pragma unroll
                        for (int cc = 0; cc < 32; ++cc) {
                            const uint64_t x2 = fma2(pack2(s[2 * cc], s[2 * cc + 1]), scale2, negm2);
                            uint64_t p2;
                            if (kTcPolyEvery > 0 && (cc % kTcPolyDiv) == kTcPolyDiv - 1) {
                                p2 = exp2_poly2(x2);
                            } else {
                                float x0, x1;
                                unpack2(x2, x0, x1);
                                p2 = pack2(fast_exp2(x0), fast_exp2(x1));
                            }
                            if (cc & 1) sum_b = add2(sum_b, p2); else sum_a = add2(sum_a, p2);
                            float p0, p1;
                            unpack2(p2, p0, p1);
                            pk[cc] = pack_bf16(p0, p1);
                        }
                        float sa, sb;
                        unpack2(add2(sum_a, sum_b), sa, sb);
                        half_sum[half] = sa + sb;
                        // No row maximum is tracked here.  A score far above the maximum in use shows up as a huge
                        // term of the sum (2^16 and more: one key 16 octaves above, or infinity).
                        const bool leapt = __any_sync(0xffffffffu, !(half_sum[half] < kTcSumTrigger));
                        if (half == 0) {
                            if (leapt) {   // S_t is still intact: the whole step the slow way
                                slow = true;
                                break;
                            }
                            tmem_st32u(tS, pk);
                        } else {
                            if (leapt) {   // the first half's P is already in place: bring it and O_t to the new maximum
                                uint32_t redone[32];   // (addressable only here: pk itself stays in registers)
                                const TcFixed f = tc_fix_second_half<0>(tS, tO, p.scale_log2, m_used, l, half_sum[0], redone);
                                m_used = f.m_used;
                                l = f.l;
#pragma unroll
                                for (int i = 0; i < 32; ++i) pk[i] = redone[i];
                            } else {
                                l += half_sum[0] + half_sum[1];
                            }
                            tmem_st32u(tS + 32, pk);
                            tmem_wait_st();
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(bar_p_full(t));
                        }
                    }
                }
                if (slow) {
                    // pass 1 over S_t: row maximum (3-input max, two chains per 32-column chunk).  The
                    // scores are read again in pass 2 rather than kept: tensor-memory reads are cheap and
                    // 128 live registers per thread are not.
                    float mx = -INFINITY;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float s[64];
                        tmem_ld32(tS + h * 64, *reinterpret_cast<float(*)[32]>(&s[0]));
                        tmem_ld32(tS + h * 64 + 32, *reinterpret_cast<float(*)[32]>(&s[32]));
                        tmem_wait_ld();
                        if (edge) {
#pragma unroll
                            for (int c = 0; c < 64; ++c) s[c] = (h * 64 + c <= rel && h * 64 + c >= lo) ? s[c] : -INFINITY;
                        }
                        float m0 = max3(s[0], s[1], s[2]), m1 = max3(s[3], s[4], s[5]);
                        float m2 = max3(s[6], s[7], s[8]), m3 = max3(s[9], s[10], s[11]);
#pragma unroll
                        for (int c = 12; c < 60; c += 8) {
                            m0 = max3(m0, s[c], s[c + 1]);
                            m1 = max3(m1, s[c + 2], s[c + 3]);
                            m2 = max3(m2, s[c + 4], s[c + 5]);
                            m3 = max3(m3, s[c + 6], s[c + 7]);
                        }
                        m0 = max3(m0, s[60], s[61]);
                        m1 = max3(m1, s[62], s[63]);
                        mx = max3(mx, fmaxf(m0, m1), fmaxf(m2, m3));
                    }
                    const float m_new = fmaxf(m_used, mx * p.scale_log2);
                    // rescale O only when the maximum moved far enough to matter; otherwise keep
                    // exponentiating against the stale maximum (O and l stay consistent with it)
                    const bool need = (m_new - m_used > kTcRescaleThreshold) || (m_used == -INFINITY && m_new != -INFINITY);
                    const bool rescale = __any_sync(0xffffffffu, need);
                    float corr = 1.0f;
                    if (rescale) {
                        corr = (m_used == -INFINITY) ? 0.0f : fast_exp2(m_used - m_new);
                        m_used = m_new;
                    }
                    const float msub = (m_used == -INFINITY) ? 0.0f : m_used;
                    // S_t(j) complete implies P.V(t, j-1) complete (MMAs of one thread finish in issue
                    // order), so O_t can be rescaled and the columns of S_t can take P_t right away.
                    if (rescale && j > 0) {   // before any P.V of this step may start
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            float o[32];
                            tmem_ld32(tO + c * 32, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] *= corr;
                            tmem_st32(tO + c * 32, o);
                        }
                    }
                    // pass 2: p = exp2(s * scale - m) on packed pairs; P row -> tensor memory as bf16
                    // pairs (k, k+1) per 32-bit column, 64 columns, over the first half of S_t.
                    {
                        const uint64_t scale2 = pack2(p.scale_log2, p.scale_log2), negm2 = pack2(-msub, -msub);
                        uint64_t sum_a = pack2(0.0f, 0.0f), sum_b = sum_a;
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            // keys [64*half, 64*half+64) of S sit in columns [64*half, +64); their P goes to
                            // columns [32*half, +32), which never overlap a half of S not yet read
                            float s[64];
                            tmem_ld32(tS + half * 64, *reinterpret_cast<float(*)[32]>(&s[0]));
                            tmem_ld32(tS + half * 64 + 32, *reinterpret_cast<float(*)[32]>(&s[32]));
                            tmem_wait_ld();
                            if (edge) {
#pragma unroll
                                for (int c = 0; c < 64; ++c) s[c] = (half * 64 + c <= rel && half * 64 + c >= lo) ? s[c] : -INFINITY;
                            }
                            uint32_t pk[32];
#pragma unroll
                            for (int cc = 0; cc < 32; ++cc) {
                                const int c = half * 32 + cc;
                                const uint64_t x2 = fma2(pack2(s[2 * cc], s[2 * cc + 1]), scale2, negm2);
                                uint64_t p2;
                                if (kTcPolyEvery > 0 && (c % kTcPolyDiv) == kTcPolyDiv - 1) {
                                    p2 = exp2_poly2(x2);
                                } else {
                                    float x0, x1;
                                    unpack2(x2, x0, x1);
                                    p2 = pack2(fast_exp2(x0), fast_exp2(x1));
                                }
                                if (c & 1) sum_b = add2(sum_b, p2); else sum_a = add2(sum_a, p2);
                                float p0, p1;
                                unpack2(p2, p0, p1);
                                pk[cc] = pack_bf16(p0, p1);
                            }
                            tmem_st32u(tS + half * 32, pk);
                            tmem_wait_st();
                            tc_fence_before();
                            __syncwarp();
                            if (half == 1 && lane == 0) mbar_arrive(bar_p_full(t));
                        }
                        float sa, sb;
                        unpack2(add2(sum_a, sum_b), sa, sb);
                        l = l * corr + (sa + sb);
                    }
                }
            }
            if ((warp & 3) == 0 && lane == 0) TC_TRACE(tr + 1);
            if (ok && my_steps > 0) {
                ok = mbar_wait(bar_pv_done(t), (steps_done + my_steps - 1) & 1, abort_word, p.status, kTcWaitPvDone, p.wait_timeout_ns);
                ok = __all_sync(0xffffffffu, ok);
            }
            if (!ok) break;
            if ((warp & 3) == 0 && lane == 0) TC_TRACE(tr + 2);
            OutT* orow = reinterpret_cast<OutT*>(p.out) + row_index * kHeadDim;
            if (my_steps > 0) {
                tc_fence_after();
                float inv = (l > 0.0f) ? 1.0f / l : 0.0f;
                bool bad = false;   // kExt: the row is not finite (see exact_row)
                if constexpr (kExt != 0) {
                    if (!(l < INFINITY)) bad = true;
                }
                if constexpr (kSplit) {
                    // A thread's row is 512 bytes: 16-byte stores of 32 threads would touch 32 lines each.  The warp turns
                    // 64 columns of its 32 rows over in its quarter of the Q tile (which this item's products are done
                    // with) and stores whole 256-byte runs.  Piece c of row r sits at c ^ (r & 15).
                    unsigned char* stage = smem + kTcSmemQ + t * kTcTileBytes + (warp & 3) * (kTcTileBytes / 4);
                    const unsigned live = __ballot_sync(0xffffffffu, valid);
#pragma unroll 1
                    for (int h = 0; h < 2; ++h) {
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float o[32];
                            tmem_ld32(tO + h * 64 + c * 32, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                *reinterpret_cast<float4*>(stage + lane * 256 + (((c * 8 + i) ^ (lane & 15)) << 4)) =
                                    make_float4(o[i * 4 + 0] * inv, o[i * 4 + 1] * inv, o[i * 4 + 2] * inv, o[i * 4 + 3] * inv);
                        }
                        __syncwarp();
#pragma unroll 4
                        for (int i = 0; i < 16; ++i) {
                            const int r = 2 * i + (lane >> 4), c = lane & 15;
                            const float4 v = *reinterpret_cast<const float4*>(stage + r * 256 + ((c ^ (r & 15)) << 4));
                            const long long at = __shfl_sync(0xffffffffu, row_index, r);
                            if ((live >> r) & 1u) *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + at * kHeadDim + h * 64 + c * 4) = v;
                        }
                        __syncwarp();
                    }
                    fence_async_smem();   // before the next item's Q may be copied in
                    if (valid && p.lse) p.lse[row_index] = (m_used + log2f(l)) * kLn2;
                } else {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float o[32];
                    tmem_ld32(tO + c * 32, o);
                    tmem_wait_ld();
                    if constexpr (kExt != 0) {
                        if (l == 0.0f) {   // sees nothing: zeros, whatever the masked rows of V were
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = 0.0f;
                        }
                        float big = 0.0f;   // 0 * x is 0 for a finite x, NaN otherwise
#pragma unroll
                        for (int i = 0; i < 32; ++i) big = fmaf(o[i], 0.0f, big);
                        bad |= !(big == 0.0f);
                    }
                    if (valid) {
                        if constexpr (sizeof(OutT) == 4) {
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                *reinterpret_cast<float4*>(orow + c * 32 + i * 4) =
                                    make_float4(o[i * 4 + 0] * inv, o[i * 4 + 1] * inv, o[i * 4 + 2] * inv, o[i * 4 + 3] * inv);
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                uint4 v;
                                v.x = pack_bf16(o[i * 8 + 0] * inv, o[i * 8 + 1] * inv);
                                v.y = pack_bf16(o[i * 8 + 2] * inv, o[i * 8 + 3] * inv);
                                v.z = pack_bf16(o[i * 8 + 4] * inv, o[i * 8 + 5] * inv);
                                v.w = pack_bf16(o[i * 8 + 6] * inv, o[i * 8 + 7] * inv);
                                *reinterpret_cast<uint4*>(orow + c * 32 + i * 8) = v;
                            }
                        }
                    }
                }
                if (valid && p.lse) p.lse[row_index] = (m_used + log2f(l)) * kLn2;
                }
                if constexpr (kExt != 0 && sizeof(OutT) == 2) {
                    // These rows are computed again once the list is done: doing it here would keep the other roles in
                    // their bounded waits.  The warp's items with such rows form a chain through the rows' own outputs.
                    const unsigned redo = __ballot_sync(0xffffffffu, bad && valid);
                    __syncwarp();   // each lane's stores of its own row, before other lanes store the same row
                    if (redo) {
                        const long long r_index = __shfl_sync(0xffffffffu, row_index, __ffs(redo) - 1);
                        if (lane == 0)
                            *reinterpret_cast<int2*>(reinterpret_cast<__nv_bfloat16*>(p.out) + r_index * kHeadDim) =
                                make_int2(redo_item, static_cast<int>(redo_rows));
                        redo_item = idx;
                        redo_rows = redo;
                    }
                }
                // the next item's first P.V overwrites O_t: its P is only handed over by these same
                // threads, after the reads above have completed
                tc_fence_before();
            } else if (valid) {
                // no key of the window lies in reach of this tile's rows: an empty partial result
                if constexpr (sizeof(OutT) == 4) {
                    for (int i = 0; i < 32; ++i) *reinterpret_cast<float4*>(orow + i * 4) = make_float4(0.f, 0.f, 0.f, 0.f);
                } else {
                    for (int i = 0; i < 16; ++i) *reinterpret_cast<uint4*>(orow + i * 8) = make_uint4(0u, 0u, 0u, 0u);
                }
                if (p.lse) p.lse[row_index] = -INFINITY;
            }
            if constexpr (kSplit) {
                __syncwarp();
                if (lane == 0 && my_steps > 0) mbar_arrive(bar_q_empty(t));
            }
            steps_done += my_steps;
            if ((warp & 3) == 0 && lane == 0) TC_TRACE(tr + 3);
        }
        if constexpr (kExt != 0 && !kSplit && sizeof(OutT) == 2) {
            // Rare: the rows that came out not finite, key by key (see exact_row), one row at a time, the whole warp on
            // it.  Nothing waits for this warp any more but the block's last barrier.
            while (ok && redo_item >= 0) {
                tc_item(p, redo_item, it);
                const int rho0 = (it.pair * kTcTiles + t) * p.ext.tile_pos * p.group + (warp & 3) * 32;   // of lane 0
                auto row_at = [&](int rho) { return (static_cast<long long>(rho / p.group) * p.max_batch + it.b) * p.q_heads + it.kvh * p.group + rho % p.group; };
                __nv_bfloat16* const out = reinterpret_cast<__nv_bfloat16*>(p.out);
                int2 link = make_int2(-1, 0);
                if (lane == 0) link = *reinterpret_cast<const int2*>(out + row_at(rho0 + __ffs(redo_rows) - 1) * kHeadDim);   // (written by this lane)
                link.x = __shfl_sync(0xffffffffu, link.x, 0);
                link.y = __shfl_sync(0xffffffffu, link.y, 0);
                const ScoreMods& m = p.ext.mods;
                for (unsigned rows = redo_rows; rows; rows &= rows - 1) {
                    const int rho = rho0 + __ffs(rows) - 1, head = it.kvh * p.group + rho % p.group;
                    const long long r_index = row_at(rho), r_pos = it.base + rho / p.group;
                    long long lo, hi;
                    row_interval(m, it.b, r_pos, it.key_end, lo, hi);
                    exact_row(m, p.ext.q + r_index * kHeadDim, p.ext.k + it.b * p.ext.s0 + it.kvh * p.ext.s1,
                              p.ext.v + it.b * p.ext.s0 + it.kvh * p.ext.s1, p.ext.s2, m.pk + it.kvh * m.ps1, m.pv + it.kvh * m.ps1, r_pos, lo, hi,
                              m.slopes ? m.slopes[head] * kLog2e : 0.0f, out + r_index * kHeadDim, p.lse ? p.lse + r_index : nullptr, lane);
                }
                redo_item = link.x;
                redo_rows = static_cast<unsigned>(link.y);
            }
        }
    } else if (warp == kTcTiles * 4) {
        // =============================== TMA producer ===============================
        if (lane == 0) {
            bool ok = true;
            long long ring_n = 0;                   // ring items requested so far (K_0, V_0, K_1, ... of every item)
            int q_loads[kTcTiles] = {0, 0};
            int tails = 0;                          // tiles cleaned up so far
            bool tail_pending = false;
            // fused append: tiles waiting to be stored into the cache, per ring slot
            bool store_pending[kTcStages] = {};
            long long store_ring[kTcStages] = {};
            int store_key0[kTcStages] = {};
            int store_head[kTcStages] = {};
            // waits until the slot's tile has landed, stores it to the cache rows it holds and waits until the
            // store has read the slot (so that the slot can be refilled)
            auto flush_store = [&](int slot) -> bool {
                const long long r = store_ring[slot];
                if (!mbar_wait(bar_kv_full(slot), static_cast<uint32_t>((r / kTcStages) & 1), abort_word, p.status, kTcWaitKvFull, p.wait_timeout_ns))
                    return false;
                const int hd = store_head[slot];
                const CUtensorMap* map = (hd >> 30) ? &map_v : &map_k;
                for (int h = 0; h < 2; ++h)
                    tma_store_4d(map, smem_base + kTcSmemRing + slot * kTcTileBytes + h * kTcHalfBytes, h * 64, store_key0[slot],
                                 hd & 0xffff, (hd >> 16) & 0x3fff);
                bulk_commit();
                bulk_wait_read_all();
                store_pending[slot] = false;
                return true;
            };
            Item it;
            for (long long k = 0; ok; ++k) {
                // this CTA's k-th item: its own block index first, then whatever comes next on the list
                long long idx = blockIdx.x;
                if (k > 0) idx = p.sched ? static_cast<long long>(gridDim.x) + atomicAdd(p.sched, 1) : p.n_items;
                if (idx > p.n_items) idx = p.n_items;
                ok = mbar_wait(bar_sched_empty(static_cast<int>(k & 1)), static_cast<uint32_t>(((k >> 1) & 1) ^ 1), abort_word, p.status,
                               kTcWaitSched, p.wait_timeout_ns);
                if (!ok) break;
                sched_idx[k & 1] = static_cast<int>(idx);
                mbar_arrive(bar_sched_full(static_cast<int>(k & 1)));   // releases the word above to the waiters
                if (idx >= p.n_items) break;
                tc_item(p, idx, it);
                for (int t = 0; t < kTcTiles && ok; ++t) {
                    if (it.steps[t] == 0) continue;
                    // the previous item's last Q.K^T of this row tile has finished with the Q tile
                    ok = mbar_wait(bar_q_empty(t), (q_loads[t] & 1) ^ 1, abort_word, p.status, kTcWaitQEmpty, p.wait_timeout_ns);
                    if (!ok) break;
                    int pos0 = (it.pair * kTcTiles + t) * kTcTileRows / p.group;
                    uint32_t q_bytes = kTcTileBytes;
                    if constexpr (kExt != 0) {
                        pos0 = (it.pair * kTcTiles + t) * p.ext.tile_pos;
                        q_bytes = static_cast<uint32_t>(p.ext.tile_pos * p.group) * kRowBytes;
                    }
                    mbar_arrive_expect_tx(bar_q(t), q_bytes);
                    for (int h = 0; h < 2; ++h)
                        tma_load_5d(smem_base + kTcSmemQ + t * kTcTileBytes + h * kTcHalfBytes, &map_q, bar_q(t), h * 64, 0,
                                    pos0, it.kvh, it.b);
                    ++q_loads[t];
                }
                for (int item = 0; !kSplit && item < 2 * it.nsteps && ok; ++item, ++ring_n) {  // K_0, V_0, K_1, V_1, ...
                    const int slot = static_cast<int>(ring_n % kTcStages);
                    const uint32_t round_par = static_cast<uint32_t>((ring_n / kTcStages) & 1);
                    if constexpr (kFused) {
                        // a tile of the chunk's own rows that waits in this slot to be written into the cache
                        // goes out first (it landed long ago: the slot has been consumed since)
                        if (store_pending[slot]) ok = flush_store(slot);
                        if (!ok) break;
                    }
                    ok = mbar_wait(bar_kv_empty(slot), round_par ^ 1, abort_word, p.status, kTcWaitKvEmpty, p.wait_timeout_ns);
                    if (!ok) break;
                    if (ring_n == p.debug_skip_item) continue;   // test hook: this item's barrier is never signalled
                    const int key0 = (it.j0 + (item >> 1)) * kTcKeys;
                    if constexpr (kFused) {
                        // Key tiles at or past the chunk's start hold the chunk's own rows, which are not in the
                        // cache yet - they come from k_new / v_new (row = key - chunk start).  Exactly one item
                        // writes such a tile into the cache: the one whose rows include the tile's first token.
                        const bool from_new = key0 >= p.base;
                        const CUtensorMap* map = from_new ? ((item & 1) ? &map_vn : &map_kn) : ((item & 1) ? &map_v : &map_k);
                        const int row0 = from_new ? key0 - static_cast<int>(p.base) : key0;
                        mbar_arrive_expect_tx(bar_kv_full(slot), kTcTileBytes);
                        for (int h = 0; h < 2; ++h)
                            tma_load_4d(smem_base + kTcSmemRing + slot * kTcTileBytes + h * kTcHalfBytes, map, bar_kv_full(slot),
                                        h * 64, row0, it.kvh, it.b);
                        if (from_new && (static_cast<long long>(row0 / kTcKeys) * p.group) / 2 == it.pair) {
                            store_pending[slot] = true;
                            store_ring[slot] = ring_n;
                            store_key0[slot] = key0;
                            store_head[slot] = it.kvh | (it.b << 16) | ((item & 1) << 30);
                        }
                    } else {
                        const CUtensorMap* map = (item & 1) ? &map_v : &map_k;
                        int row0 = key0, seq = it.b;
                        if constexpr (kExt != 0) {
                            if ((item >> 1) < it.np) {
                                map = (item & 1) ? &map_vn : &map_kn;
                                row0 = (it.p0 + (item >> 1)) * kTcKeys;
                                seq = 0;
                            } else {
                                row0 = (kExt & kExtBias) ? (it.j0 + it.nsteps - 1 - (item >> 1)) * kTcKeys : row0 - it.np * kTcKeys;
                            }
                        }
                        // The V tile with rows past the sequence's end (the last one, the first where the keys are walked
                        // backwards) lands on a barrier of the producer's own; it is cleaned up and only then signalled.
                        const bool tail = it.zero_tail && item == ((kExt & kExtBias) ? 1 : 2 * it.nsteps - 1);
                        const uint32_t landed = tail ? bar_tail : bar_kv_full(slot);
                        mbar_arrive_expect_tx(landed, kTcTileBytes);
                        for (int h = 0; h < 2; ++h)
                            tma_load_4d(smem_base + kTcSmemRing + slot * kTcTileBytes + h * kTcHalfBytes, map, landed, h * 64, row0, it.kvh, seq);
                        if (tail) {
                            ok = mbar_wait(bar_tail, static_cast<uint32_t>(tails & 1), abort_word, p.status, kTcWaitKvFull, p.wait_timeout_ns);
                            if (!ok) {
                                tail_pending = true;
                                break;
                            }
                            // a 128-byte row of either half holds one key; the swizzle only permutes inside a row
                            const int first = static_cast<int>(it.key_end - static_cast<long long>(row0));
                            unsigned char* tile = smem + kTcSmemRing + slot * kTcTileBytes;
                            for (int r = first * 8; r < kTcKeys * 8; ++r) {
                                *reinterpret_cast<uint4*>(tile + r * 16) = make_uint4(0u, 0u, 0u, 0u);
                                *reinterpret_cast<uint4*>(tile + kTcHalfBytes + r * 16) = make_uint4(0u, 0u, 0u, 0u);
                            }
                            fence_async_smem();
                            mbar_arrive(bar_kv_full(slot));
                            ++tails;
                        }
                    }
                }
            }
            if (kFused) {
                for (int s = 0; s < kTcStages && ok; ++s)
                    if (store_pending[s]) ok = flush_store(s);
                bulk_wait_all();   // the cache rows are written before the kernel ends
            }
            if (*abort_word) {
                // a wait ran out somewhere: copies this thread requested may still be on their way into
                // shared memory.  Wait (bounded, quietly) for the barrier of every slot it armed last.
                for (int s = 0; s < kTcStages; ++s) {
                    const long long last = ring_n - 1 - ((ring_n - 1 - s) % kTcStages + kTcStages) % kTcStages;   // last item of slot s
                    if (last >= 0 && last != p.debug_skip_item)
                        mbar_wait_quiet(bar_kv_full(s), static_cast<uint32_t>((last / kTcStages) & 1), 200000ull);
                }
                for (int t = 0; t < kTcTiles; ++t)
                    if (q_loads[t] > 0) mbar_wait_quiet(bar_q(t), static_cast<uint32_t>((q_loads[t] - 1) & 1), 200000ull);
                if (tail_pending) mbar_wait_quiet(bar_tail, static_cast<uint32_t>(tails & 1), 200000ull);
            }
        }
        __syncwarp();
    } else if (kSplit && warp >= kTcTiles * 4 + 2) {
        // =============================== K/V loaders (kExtSplit) ===============================
        // Loader warp w copies rows [64 w, 64 w + 64) of every tile, 16 bytes a lane, a row's 256 contiguous bytes by
        // 16 lanes, into the layout a TMA box of 128-byte swizzled rows has.  Up to four tiles are in flight.  A tile is
        // signalled, after the fence that makes it visible to the MMAs, when the copies of three later ones are
        // out, or at once when there is no free slot to copy into: then the copies are ahead of the MMAs anyway.
        if constexpr (kSplit) {
            constexpr int kAhead = 3;
            const int half = warp - (kTcTiles * 4 + 2);
            const int rlane = lane >> 4, chunk = lane & 15;
            uint32_t off[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                off[i] = (chunk >> 3) * kTcHalfBytes + (half * 64 + 2 * i + rlane) * 128 + (((chunk & 7) ^ (2 * i + rlane)) << 4);
            long long ring_n = 0, signalled = 0;
            auto signal_upto = [&](long long n) {   // the copies of tiles < n have landed
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                for (; signalled < n; ++signalled)
                    if (lane == 0 && signalled != p.debug_skip_item) mbar_arrive(bar_kv_full(static_cast<int>(signalled % kTcStages)));
            };
            bool ok = true;
            Item it;
            for (long long k = 0; ok; ++k) {
                int idx = n_items;
                if (lane == 0) idx = take_item(k, ok, kTcWaitSched);
                idx = __shfl_sync(0xffffffffu, idx, 0);
                ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
                if (!ok) break;
                if (lane == 0) mbar_arrive(bar_sched_empty(static_cast<int>(k & 1)));
                if (idx >= n_items) break;
                tc_item(p, idx, it);
                const ScoreMods& m = p.ext.mods;
                for (int item = 0; item < 2 * it.nsteps; ++item, ++ring_n) {
                    const int slot = static_cast<int>(ring_n % kTcStages);
                    const uint32_t par = static_cast<uint32_t>(((ring_n / kTcStages) & 1) ^ 1);
                    if (signalled < ring_n && !__shfl_sync(0xffffffffu, lane == 0 ? mbar_try_wait(bar_kv_empty(slot), par) : 0u, 0)) {
                        cp_async_wait<0>();
                        signal_upto(ring_n);
                    }
                    if (lane == 0)
                        ok = mbar_wait(bar_kv_empty(slot), par, abort_word, p.status, kTcWaitKvEmpty, p.wait_timeout_ns);
                    ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
                    if (!ok) break;
                    const long long row0 = static_cast<long long>(it.p0 + (item >> 1)) * kTcKeys + half * 64 + rlane;
                    const __nv_bfloat16* src = ((item & 1) ? m.pv : m.pk) + it.kvh * m.ps1 + row0 * m.ps2 + chunk * 8;
                    const uint32_t dst = smem_base + kTcSmemRing + slot * kTcTileBytes;
                    const long long left = m.plen - row0;   // row 2 i of this lane exists when 2 i < left
                    if (left >= 64) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) cp_async_16(dst + off[i & 3] + (i >> 2) * 1024, src + i * 2 * m.ps2, 16);
                    } else {
#pragma unroll 4
                        for (int i = 0; i < 32; ++i) cp_async_16(dst + off[i & 3] + (i >> 2) * 1024, 2 * i < left ? src + i * 2 * m.ps2 : m.pk, 2 * i < left ? 16 : 0);
                    }
                    cp_async_commit();
                    if (item == 0) {   // the item's first K tile: everything waits for it
                        cp_async_wait<0>();
                        signal_upto(ring_n + 1);
                        continue;
                    }
                    cp_async_wait<kAhead>();
                    if (ring_n - kAhead + 1 > signalled) signal_upto(ring_n - kAhead + 1);
                }
                if (!ok) break;
                cp_async_wait<0>();
                signal_upto(ring_n);
            }
            cp_async_wait<0>();   // (a wait that ran out: nothing of this warp's is in flight when the block ends)
        }
    } else if (kExt != 0) {
        // =============================== MMA issuer, kExt ===============================
        // The same order of products as below.  The whole warp walks the list and one elected lane issues: addresses
        // and descriptors then stay in uniform registers.  Issued by a lane of a divergent branch a product costs the
        // issuing thread about 90 clocks, and the 32 of a step were what the step took.
        if constexpr (kExt != 0) {
            bool ok = true;
            constexpr uint32_t idesc_qk = umma_idesc(false), idesc_pv = umma_idesc(true);
            auto wait = [&](uint32_t bar, uint32_t par, int code) -> bool {
                return __all_sync(0xffffffffu, mbar_wait(bar, par, abort_word, p.status, code, p.wait_timeout_ns)) != 0;
            };
            int slot_k = 0, slot_v = 0;              // ring slots of the next K and V tile to be used ...
            int ring_slot = 0;                       // ... which follow one another in the ring
            uint32_t ring_par = 0;
            auto next_slot = [&]() {
                if (++ring_slot == kTcStages) {
                    ring_slot = 0;
                    ring_par ^= 1;
                }
            };
            unsigned steps_done[kTcTiles] = {0, 0}, q_loads[kTcTiles] = {0, 0};
            Item it;
            for (long long k = 0; ok; ++k) {
                int idx = n_items;
                if (lane == 0) idx = take_item(k, ok, kTcWaitSched);
                idx = __shfl_sync(0xffffffffu, idx, 0);
                ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
                if (!ok) break;
                if (lane == 0) mbar_arrive(bar_sched_empty(static_cast<int>(k & 1)));
                if (idx >= n_items) break;
                tc_item(p, idx, it);
                const int nsteps = it.nsteps;
                auto wait_tile = [&]() -> bool {   // the next tile of the ring
                    return wait(bar_kv_full(ring_slot), ring_par, kTcWaitKvFull);
                };
                auto issue_qk = [&](int t, int slot, bool last) {
                    const uint64_t q_desc = umma_desc(smem_base + kTcSmemQ + t * kTcTileBytes, 0, 1024);
                    const uint64_t k_desc = umma_desc(smem_base + kTcSmemRing + slot * kTcTileBytes, 0, 1024);
                    if (elect_one()) {
#pragma unroll
                        for (int ks = 0; ks < 8; ++ks) {
                            const uint32_t off = ((ks >> 2) * kTcHalfBytes + (ks & 3) * 32) >> 4;
                            umma_bf16(tmem + t * 128, q_desc + off, k_desc + off, idesc_qk, ks > 0);
                        }
                        umma_commit(bar_s_full(t));
                        if (!kSplit && last) umma_commit(bar_q_empty(t));   // this item reads Q_t no more
                    }
                    __syncwarp();
                };
                auto issue_pv = [&](int t, int slot, bool first) {
                    const uint64_t v_desc = umma_desc(smem_base + kTcSmemRing + slot * kTcTileBytes, kTcHalfBytes, 1024);
                    if (elect_one()) {
#pragma unroll
                        for (int ks = 0; ks < 8; ++ks)
                            umma_bf16_a_tmem(tmem + 256 + t * 128, tmem + t * 128 + ks * 8, v_desc + ((ks * 16 * 128) >> 4), idesc_pv, !(first && ks == 0));
                        umma_commit(bar_pv_done(t));
                    }
                    __syncwarp();
                };
                for (int t = 0; t < kTcTiles && ok; ++t)
                    if (it.steps[t] > 0) ok = wait(bar_q(t), q_loads[t] & 1u, kTcWaitQ);
                if (ok && nsteps > 0) {
                    ok = wait_tile();
                    if (ok) {
                        tc_fence_after();
                        for (int t = 0; t < kTcTiles; ++t)
                            if (it.steps[t] > 0) issue_qk(t, ring_slot, it.steps[t] == 1);
                        if (elect_one()) umma_commit(bar_kv_empty(ring_slot));
                        __syncwarp();
                        next_slot();
                    }
                }
                for (int j = 0; j < nsteps && ok; ++j) {
                    bool have_v = false, have_k = false;
                    for (int t = 0; t < kTcTiles && ok; ++t) {
                        if (j >= it.steps[t]) continue;
                        ok = wait(bar_p_full(t), (steps_done[t] + j) & 1u, kTcWaitPFull);
                        if (!ok) break;
                        if (!have_v) {
                            ok = wait_tile();
                            if (!ok) break;
                            slot_v = ring_slot;
                            next_slot();
                            have_v = true;
                        }
                        tc_fence_after();
                        issue_pv(t, slot_v, j == 0);
                        if (j + 1 < it.steps[t]) {
                            if (!have_k) {
                                ok = wait_tile();
                                if (!ok) break;
                                slot_k = ring_slot;
                                next_slot();
                                have_k = true;
                                tc_fence_after();
                            }
                            issue_qk(t, slot_k, j + 2 == it.steps[t]);
                        }
                    }
                    if (!ok) break;
                    if (elect_one()) {
                        umma_commit(bar_kv_empty(slot_v));                      // V_j free once every MMA so far is done
                        if (j + 1 < nsteps) umma_commit(bar_kv_empty(slot_k));  // and K_{j+1}
                    }
                    __syncwarp();
                }
                if (!ok) break;
                for (int t = 0; t < kTcTiles; ++t) {
                    steps_done[t] += it.steps[t];
                    if (it.steps[t] > 0) ++q_loads[t];
                }
            }
            if (elect_one()) {
                umma_commit(bar_final);   // every MMA issued above has completed before tensor memory is given back
                mbar_wait_quiet(bar_final, 0, *abort_word ? 2000000ull : p.wait_timeout_ns);
            }
            __syncwarp();
        }
    } else {
        // =============================== MMA issuer ===============================
        // One thread issues every MMA, one GEMM after the other: two issuing threads were tried and
        // lost 20 % because their GEMMs interleave on the tensor pipe and both finish late.
        if (lane == 0) {
            bool ok = true;
            constexpr uint32_t idesc_qk = umma_idesc(false), idesc_pv = umma_idesc(true);
            auto issue_qk = [&](int t, int slot) {  // S_t = Q_t K^T: 8 steps of 16 over head_dim
                const uint32_t q_addr = smem_base + kTcSmemQ + t * kTcTileBytes;
                const uint32_t k_addr = smem_base + kTcSmemRing + slot * kTcTileBytes;
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) {
                    const uint32_t off = (ks >> 2) * kTcHalfBytes + (ks & 3) * 32;
                    umma_bf16(tmem + t * 128, umma_desc(q_addr + off, 0, 1024), umma_desc(k_addr + off, 0, 1024), idesc_qk,
                              ks > 0);
                }
                umma_commit(bar_s_full(t));
            };
            // O_t += P_t V for keys [64*half, 64*half + 64): 4 steps of 16 keys
            auto issue_pv_half = [&](int t, int slot, bool first, int half) {
                const uint32_t v_addr = smem_base + kTcSmemRing + slot * kTcTileBytes;
#pragma unroll
                for (int k4 = 0; k4 < 4; ++k4) {
                    const int ks = half * 4 + k4;
                    const uint32_t b_off = ks * 16 * 128;  // 16 key rows of 128 bytes
                    umma_bf16_a_tmem(tmem + 256 + t * 128, tmem + t * 128 + ks * 8,
                                     umma_desc(v_addr + b_off, kTcHalfBytes, 1024), idesc_pv, !(first && ks == 0));
                }
                if (half == 1) umma_commit(bar_pv_done(t));
            };
            long long ring_c = 0;                  // ring items of all earlier work items
            int steps_done[kTcTiles] = {0, 0};
            int q_loads[kTcTiles] = {0, 0};
            Item it;
            for (long long k = 0; ok; ++k) {
                const int idx = take_item(k, ok, kTcWaitSched);
                if (!ok) break;
                mbar_arrive(bar_sched_empty(static_cast<int>(k & 1)));
                if (idx >= n_items) break;
                tc_item(p, idx, it);
                const int nsteps = it.nsteps;
                // ring item i of this work item: K_(i/2) for even i, V_(i/2) for odd i
                auto wait_item = [&](int item) {
                    const long long r = ring_c + item;
                    return mbar_wait(bar_kv_full(static_cast<int>(r % kTcStages)), static_cast<uint32_t>((r / kTcStages) & 1), abort_word,
                                     p.status, kTcWaitKvFull, p.wait_timeout_ns);
                };
                auto slot_of = [&](int item) { return static_cast<int>((ring_c + item) % kTcStages); };
                for (int t = 0; t < kTcTiles && ok; ++t)
                    if (it.steps[t] > 0) ok = mbar_wait(bar_q(t), static_cast<uint32_t>(q_loads[t] & 1), abort_word, p.status, kTcWaitQ, p.wait_timeout_ns);
                if (ok && nsteps > 0) {
                    ok = wait_item(0);
                    if (ok) {
                        tc_fence_after();
                        for (int t = 0; t < kTcTiles; ++t)
                            if (it.steps[t] > 0) {
                                issue_qk(t, slot_of(0));
                                if (it.steps[t] == 1) umma_commit(bar_q_empty(t));   // this item reads Q_t no more
                            }
                        umma_commit(bar_kv_empty(slot_of(0)));
                    }
                }
                for (int j = 0; j < nsteps && ok; ++j) {
                    const int item_v = 2 * j + 1, slot_v = slot_of(item_v);
                    const int item_k = 2 * j + 2, slot_k = slot_of(item_k);
                    bool have_v = false, have_k = false;
                    for (int t = 0; t < kTcTiles && ok; ++t) {
                        if (j >= it.steps[t]) continue;
                        ok = mbar_wait(bar_p_full(t), static_cast<uint32_t>((steps_done[t] + j) & 1), abort_word, p.status, kTcWaitPFull,
                                       p.wait_timeout_ns);
                        if (!ok) break;
                        if (!have_v) {
                            ok = wait_item(item_v);
                            if (!ok) break;
                            have_v = true;
                        }
                        tc_fence_after();
                        issue_pv_half(t, slot_v, j == 0, 0);
                        issue_pv_half(t, slot_v, j == 0, 1);
                        if (j + 1 < it.steps[t]) {
                            if (!have_k) {
                                ok = wait_item(item_k);
                                if (!ok) break;
                                have_k = true;
                                tc_fence_after();
                            }
                            issue_qk(t, slot_k);
                            if (j + 2 == it.steps[t]) umma_commit(bar_q_empty(t));
                        }
                    }
                    if (!ok) break;
                    umma_commit(bar_kv_empty(slot_v));                      // V_j free once every MMA so far is done
                    if (j + 1 < nsteps) umma_commit(bar_kv_empty(slot_k));  // and K_{j+1}
                }
                if (!ok) break;
                ring_c += 2 * nsteps;
                for (int t = 0; t < kTcTiles; ++t) {
                    steps_done[t] += it.steps[t];
                    if (it.steps[t] > 0) ++q_loads[t];
                }
            }
            // every MMA issued above has completed before tensor memory is given back
            umma_commit(bar_final);
            mbar_wait_quiet(bar_final, 0, *abort_word ? 2000000ull : p.wait_timeout_ns);
        }
        __syncwarp();
    }

    // teardown: every role gets here (all waits are bounded)
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0) { TC_TRACE(3); TC_TRACE_NS(4); }
    if (threadIdx.x == 0 && p.sched) {
        // the last CTA to leave puts the two words back to zero for the next launch
        __threadfence();
        if (atomicAdd(p.sched + 1, 1) == static_cast<int>(gridDim.x) - 1) {
            p.sched[0] = 0;
            p.sched[1] = 0;
            __threadfence();
        }
    }
    if (warp == kTcTiles * 4 + 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// ---------------------------------------------------------------- host side
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline void tcgen05_plan_init(Tcgen05Plan& plan, const ellm_attn_desc& d, int sm_count) {
    plan.ready = false;
    plan.sm_count = sm_count;
    const size_t group = d.q_heads / d.kv_heads;
    plan.ready_ext = false;
    if (group > 128) {
        snprintf(plan.why, sizeof(plan.why), "query heads per KV head (%zu) must divide 128", group);
        return;
    }
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qres) != cudaSuccess || !fn ||
        qres != cudaDriverEntryPointSuccess) {
        cudaGetLastError();
        snprintf(plan.why, sizeof(plan.why), "driver does not export cuTensorMapEncodeTiled");
        return;
    }
    if (cudaFuncSetAttribute(prefill_tcgen05_kernel<__nv_bfloat16, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kTcSmemBytes) != cudaSuccess ||
        cudaFuncSetAttribute(prefill_tcgen05_kernel<__nv_bfloat16, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kTcSmemBytes) != cudaSuccess ||
        cudaFuncSetAttribute(prefill_tcgen05_kernel<float, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kTcSmemBytes) != cudaSuccess) {
        snprintf(plan.why, sizeof(plan.why), "cannot reserve %d bytes of shared memory: %s", kTcSmemBytes,
                 cudaGetErrorString(cudaGetLastError()));
        return;
    }
    if (cudaFuncSetAttribute(prefill_tcgen05_kernel<__nv_bfloat16, false, kExtOn>, cudaFuncAttributeMaxDynamicSharedMemorySize, kTcSmemBytes) != cudaSuccess ||
        cudaFuncSetAttribute(prefill_tcgen05_kernel<__nv_bfloat16, false, kExtOn | kExtCap>, cudaFuncAttributeMaxDynamicSharedMemorySize, kTcSmemBytes) != cudaSuccess ||
        cudaFuncSetAttribute(prefill_tcgen05_kernel<__nv_bfloat16, false, kExtOn | kExtBias>, cudaFuncAttributeMaxDynamicSharedMemorySize, kTcSmemBytes) != cudaSuccess ||
        cudaFuncSetAttribute(prefill_tcgen05_kernel<__nv_bfloat16, false, kExtOn | kExtCap | kExtBias>, cudaFuncAttributeMaxDynamicSharedMemorySize, kTcSmemBytes) != cudaSuccess) {
        snprintf(plan.why, sizeof(plan.why), "cannot reserve %d bytes of shared memory: %s", kTcSmemBytes,
                 cudaGetErrorString(cudaGetLastError()));
        return;
    }
    if (cudaFuncSetAttribute(prefill_tcgen05_kernel<float, false, kExtOn | kExtSplit>, cudaFuncAttributeMaxDynamicSharedMemorySize, kTcSmemBytes) != cudaSuccess) {
        snprintf(plan.why, sizeof(plan.why), "cannot reserve %d bytes of shared memory: %s", kTcSmemBytes,
                 cudaGetErrorString(cudaGetLastError()));
        return;
    }
    plan.encode = fn;
    plan.ready_ext = true;
    if (128 % group != 0) {   // the plain instantiations pack rows without regard to positions
        snprintf(plan.why, sizeof(plan.why), "query heads per KV head (%zu) must divide 128", group);
        return;
    }
    plan.ready = true;
}

// AUTO picks this kernel for every chunk of at least 16 packed rows (rows x query heads of a
// group); a shorter chunk leaves more than 7/8 of a 128-row tile empty and goes to the warp-level kernel.
inline bool tcgen05_prefers(const Tcgen05Plan& plan, size_t interval, int group) {
    return plan.ready && interval * static_cast<size_t>(group) >= 16;
}

// The append can ride in the kernel when the chunk starts on a 128-key tile boundary with one start
// for all sequences and the whole key range is attended: then every key tile holds either cache rows
// only or new rows only.
inline bool tcgen05_can_fuse_append(const Tcgen05Plan& plan, const ellm_attn_desc& d, const int32_t* positions,
                                    size_t position_index, size_t batch, long long key_begin, long long key_end) {
    return plan.ready && plan.fuse_append && d.k_new && d.v_new && !positions && position_index % kTcKeys == 0 && key_begin == 0 &&
           key_end >= static_cast<long long>(d.max_seq) && batch < 16384 && d.kv_heads < 65536 &&
           (d.max_batch * d.kv_heads * 256) % 16 == 0;
}

// With a uniform chunk start the K/V tensor maps are bounded at min(position_index + interval,
// key_end) so that TMA zero-fills rows the chunk must not read; with per-sequence starts
// (positions != nullptr) they are bounded by the cache and the kernel zeroes the tail itself.
// out_f32 != nullptr writes an fp32 partial result there instead of bf16 to d.out.
inline int launch_prefill_tcgen05(Tcgen05Plan& plan, const ellm_attn_desc& d, const int32_t* positions,
                                  size_t position_index, size_t interval, size_t batch, long long key_begin,
                                  long long key_end, float* out_f32, float* lse, int* status, cudaStream_t stream,
                                  bool fused_append = false) {
    if (!plan.ready) return ELLM_ERR_UNSUPPORTED;
    const int group = static_cast<int>(d.q_heads / d.kv_heads);
    // per-sequence chunk starts: the maps can only be bounded by the cache itself
    long long kv_rows = positions ? static_cast<long long>(d.max_seq) : static_cast<long long>(position_index + interval);
    if (kv_rows > key_end) kv_rows = key_end;
    if (kv_rows > static_cast<long long>(d.max_seq)) kv_rows = static_cast<long long>(d.max_seq);
    if (kv_rows <= 0 || key_begin < 0 || (positions && key_begin != 0)) {
        snprintf(plan.why, sizeof(plan.why), "empty key window, or a window start together with per-sequence positions");
        return ELLM_ERR_UNSUPPORTED;
    }
    EncodeTiledFn encode = reinterpret_cast<EncodeTiledFn>(plan.encode);
    CUtensorMap& map_q = plan.map_q;
    CUtensorMap& map_k = plan.map_k;
    CUtensorMap& map_v = plan.map_v;
    // the buffers, head counts and strides are fixed for the handle: the maps depend only on these
    const bool reuse = plan.cached_kv_rows == kv_rows && plan.cached_interval == interval && plan.cached_batch == batch &&
                       plan.cached_q == d.q && plan.cached_fused == fused_append;
    plan.cached_kv_rows = -1;
    if (!reuse) {
        // q viewed as [head_dim, g, chunk row, kv head, sequence]; a box is 64 x G x (128/G) packed rows
        cuuint64_t dims[5] = {128, static_cast<cuuint64_t>(group), interval, d.kv_heads, d.max_batch};
        cuuint64_t strides[4] = {256, d.max_batch * d.q_heads * 256, static_cast<cuuint64_t>(group) * 256, d.q_heads * 256};
        cuuint32_t box[5] = {64, static_cast<cuuint32_t>(group), static_cast<cuuint32_t>(128 / group), 1, 1};
        cuuint32_t es[5] = {1, 1, 1, 1, 1};
        if (encode(&map_q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<void*>(d.q), dims, strides, box, es,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
            snprintf(plan.why, sizeof(plan.why), "cuTensorMapEncodeTiled(q) failed");
            return ELLM_ERR_UNSUPPORTED;
        }
    }
    for (int which = 0; which < 2 && !reuse; ++which) {
        cuuint64_t dims[4] = {128, static_cast<cuuint64_t>(kv_rows), d.kv_heads, batch};
        cuuint64_t strides[3] = {d.kv_strides[2] * 2, d.kv_strides[1] * 2, d.kv_strides[0] * 2};
        cuuint32_t box[4] = {64, 128, 1, 1};
        cuuint32_t es[4] = {1, 1, 1, 1};
        if (encode(which ? &map_v : &map_k, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, which ? d.v_cache : d.k_cache, dims,
                   strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
            snprintf(plan.why, sizeof(plan.why), "cuTensorMapEncodeTiled(k/v) failed");
            return ELLM_ERR_UNSUPPORTED;
        }
    }
    if (fused_append && !reuse) {
        // the chunk's new rows [chunk row, sequence, kv head, 128] seen as (128, chunk row, kv head, sequence):
        // the same box as a cache tile, so a tile of new rows lands in shared memory exactly like a cache tile
        for (int which = 0; which < 2; ++which) {
            cuuint64_t dims[4] = {128, interval, d.kv_heads, batch};
            cuuint64_t strides[3] = {d.max_batch * d.kv_heads * 256, 256, d.kv_heads * 256};
            cuuint32_t box[4] = {64, 128, 1, 1};
            cuuint32_t es[4] = {1, 1, 1, 1};
            if (encode(which ? &plan.map_vn : &plan.map_kn, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                       const_cast<void*>(which ? d.v_new : d.k_new), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                       CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
                snprintf(plan.why, sizeof(plan.why), "cuTensorMapEncodeTiled(k_new / v_new) failed");
                return ELLM_ERR_UNSUPPORTED;
            }
        }
    }
    plan.cached_fused = fused_append;
    plan.cached_kv_rows = kv_rows;
    plan.cached_interval = interval;
    plan.cached_batch = batch;
    plan.cached_q = d.q;
    TcParams p;
    p.out = out_f32 ? static_cast<void*>(out_f32) : d.out;
    p.key_begin = key_begin;
    p.key_end = kv_rows;
    p.lse = lse;
    p.status = status;
    p.base = static_cast<long long>(position_index);
    p.positions = positions;
    p.max_seq = static_cast<long long>(d.max_seq);
    p.wait_timeout_ns = plan.wait_timeout_ns;
    p.debug_skip_item = plan.debug_skip_item;
    p.interval = static_cast<int>(interval);
    p.batch = static_cast<int>(batch);
    p.max_batch = static_cast<int>(d.max_batch);
    p.q_heads = static_cast<int>(d.q_heads);
    p.kv_heads = static_cast<int>(d.kv_heads);
    p.group = group;
    p.pair_tiles = static_cast<int>((interval * group + kTcTiles * kTcTileRows - 1) / (kTcTiles * kTcTileRows));
    p.scale_log2 = d.scale * kLog2e;
    const unsigned long long items = static_cast<unsigned long long>(p.pair_tiles) * p.kv_heads * p.batch;
    if (items > 0x7fffffffull) {
        snprintf(plan.why, sizeof(plan.why), "too many row tiles for one launch");
        return ELLM_ERR_UNSUPPORTED;
    }
    p.n_items = static_cast<long long>(items);
    // One CTA per SM walking the item list (no second wave that starts from nothing, the set-up paid
    // once), or one CTA per item taken by the hardware in block order.
    const bool persistent = plan.sched != nullptr && (plan.persistent < 0 ? true : plan.persistent != 0);
    const unsigned long long ctas = persistent ? std::min<unsigned long long>(items, static_cast<unsigned long long>(plan.sm_count)) : items;
    p.sched = persistent ? plan.sched : nullptr;
    // K and V rows this launch can touch, all heads and sequences together
    const unsigned long long kv_bytes = 2ull * static_cast<unsigned long long>(kv_rows) * 256ull * d.kv_heads * batch;
    p.pair_major = kv_bytes <= (96ull << 20) ? 1 : 0;
    // a programmatic dependent of the stream's previous kernel: set-up overlaps that kernel's tail
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(ctas));
    cfg.blockDim = dim3(kTcThreads);
    cfg.dynamicSmemBytes = kTcSmemBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    // without the fused append the two extra maps are never used; any valid map will do
    const CUtensorMap& map_kn = fused_append ? plan.map_kn : map_k;
    const CUtensorMap& map_vn = fused_append ? plan.map_vn : map_v;
    if (fused_append && out_f32) {
        snprintf(plan.why, sizeof(plan.why), "the fused append comes with bf16 output only");
        return ELLM_ERR_UNSUPPORTED;
    }
    const cudaError_t e =
        out_f32        ? cudaLaunchKernelEx(&cfg, prefill_tcgen05_kernel<float, false>, map_q, map_k, map_v, map_kn, map_vn, p)
        : fused_append ? cudaLaunchKernelEx(&cfg, prefill_tcgen05_kernel<__nv_bfloat16, true>, map_q, map_k, map_v, map_kn, map_vn, p)
                       : cudaLaunchKernelEx(&cfg, prefill_tcgen05_kernel<__nv_bfloat16, false>, map_q, map_k, map_v, map_kn, map_vn, p);
    return e == cudaSuccess ? ELLM_OK : ELLM_ERR_CUDA;
}

// A K or V tensor map: boxes of 128 rows x 64 columns.
inline bool tcgen05_kv_map(const Tcgen05Plan& plan, CUtensorMap* map, const void* base, long long rows, size_t heads, size_t s_pos,
                           size_t s_head, size_t s_seq, size_t seqs) {
    cuuint64_t dims[4] = {128, static_cast<cuuint64_t>(rows), heads, seqs};
    cuuint64_t strides[3] = {s_pos * 2, s_head * 2, s_seq * 2};
    cuuint32_t box[4] = {64, 128, 1, 1};
    cuuint32_t es[4] = {1, 1, 1, 1};
    return reinterpret_cast<EncodeTiledFn>(plan.encode)(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box,
                                                        es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Runs of prefix tiles a decode step of `batch` sequences is cut into: one CTA per SM over all row pairs and heads.
inline int prefix_splits(const Tcgen05Plan& plan, size_t batch, size_t q_heads, size_t kv_heads, long long prefix_tiles) {
    const size_t tile_pos = 128 / (q_heads / kv_heads);
    const size_t pairs = (batch + kTcTiles * tile_pos - 1) / (kTcTiles * tile_pos);
    const long long s = static_cast<long long>(plan.sm_count / (pairs * kv_heads));
    return static_cast<int>(std::max(1ll, std::min(s, prefix_tiles)));
}

// The shared-prefix part of a decode step: part_o [splits][batch * q_heads][128] fp32, part_lse [splits][batch * q_heads].
inline int launch_prefix_split(Tcgen05Plan& plan, const ellm_attn_desc& d, const ScoreMods& mods, size_t batch, int splits, float* part_o,
                               float* part_lse, int* status, cudaStream_t stream) {
    const int group = static_cast<int>(d.q_heads / d.kv_heads);
    const int tile_pos = 128 / group;
    Tcgen05Plan::ExtKey key;
    key.batch = batch;
    key.pk = mods.pk; key.pv = mods.pv; key.ps1 = mods.ps1; key.ps2 = mods.ps2; key.plen = mods.plen;
    if (!(plan.ext_key == key)) {
        plan.ext_key = Tcgen05Plan::ExtKey();
        // the query rows of the step as a chunk of `batch` positions of one sequence
        cuuint64_t dims[5] = {128, static_cast<cuuint64_t>(group), batch, d.kv_heads, 1};
        cuuint64_t strides[4] = {256, d.q_heads * 256, static_cast<cuuint64_t>(group) * 256, d.q_heads * 256};
        cuuint32_t box[5] = {64, static_cast<cuuint32_t>(group), static_cast<cuuint32_t>(tile_pos), 1, 1};
        cuuint32_t es[5] = {1, 1, 1, 1, 1};
        if (reinterpret_cast<EncodeTiledFn>(plan.encode)(&plan.ext_q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<void*>(d.q), dims, strides,
                                                         box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                                         CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS ||
            !tcgen05_kv_map(plan, &plan.ext_pk, mods.pk, mods.plen, d.kv_heads, mods.ps2, mods.ps1, mods.ps1, 1) ||
            !tcgen05_kv_map(plan, &plan.ext_pv, mods.pv, mods.plen, d.kv_heads, mods.ps2, mods.ps1, mods.ps1, 1)) {
            snprintf(plan.why, sizeof(plan.why), "cuTensorMapEncodeTiled failed");
            return ELLM_ERR_UNSUPPORTED;
        }
        plan.ext_key = key;
    }
    TcParamsExt p{};
    p.out = part_o;
    p.lse = part_lse;
    p.status = status;
    p.interval = static_cast<int>(batch);
    p.batch = p.max_batch = 1;
    p.q_heads = static_cast<int>(d.q_heads);
    p.kv_heads = static_cast<int>(d.kv_heads);
    p.group = group;
    p.wait_timeout_ns = plan.wait_timeout_ns;
    p.debug_skip_item = plan.debug_skip_item;
    p.scale_log2 = d.scale * kLog2e;
    p.ext.mods = mods;
    p.ext.tile_pos = tile_pos;
    p.ext.tiles = static_cast<int>((batch + tile_pos - 1) / tile_pos);
    p.ext.prefix_tiles = static_cast<int>((mods.plen + kTcKeys - 1) / kTcKeys);
    p.ext.splits = splits;
    p.ext.part_rows = static_cast<long long>(batch * d.q_heads);
    p.pair_tiles = (p.ext.tiles + kTcTiles - 1) / kTcTiles;
    p.n_items = static_cast<long long>(p.pair_tiles) * p.kv_heads * splits;
    if (p.n_items > 0x7fffffffll) return ELLM_ERR_UNSUPPORTED;
    const bool persistent = plan.sched != nullptr && plan.persistent != 0;
    p.sched = persistent ? plan.sched : nullptr;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(persistent ? std::min<long long>(p.n_items, plan.sm_count) : p.n_items));
    cfg.blockDim = dim3(kTcSplitThreads);
    cfg.dynamicSmemBytes = kTcSmemBytes;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, prefill_tcgen05_kernel<float, false, kExtOn | kExtSplit>, plan.ext_q, plan.ext_pk,
                                             plan.ext_pv, plan.ext_pk, plan.ext_pv, p);
    return e == cudaSuccess ? ELLM_OK : ELLM_ERR_CUDA;
}

inline bool tcgen05_takes_cap(const ScoreMods& m) {
    return m.cap_log2 == 0.0f || (m.cap_log2 <= kTcCapMax * kLog2e && m.cap_in >= kTcCapInMin && m.cap_in <= kTcCapInMax);
}

// A chunk with modified scores, row intervals or a shared prefix (bf16 result).
inline int launch_prefill_tcgen05_ext(Tcgen05Plan& plan, const ellm_attn_desc& d, const ScoreMods& mods, const int32_t* positions,
                                      size_t position_index, size_t interval, size_t batch, float* lse, int* status,
                                      cudaStream_t stream) {
    if (!plan.ready_ext) return ELLM_ERR_UNSUPPORTED;
    const int group = static_cast<int>(d.q_heads / d.kv_heads);
    const int tile_pos = 128 / group;
    long long kv_rows = positions ? static_cast<long long>(d.max_seq) : static_cast<long long>(position_index + interval);
    kv_rows = std::min(kv_rows, static_cast<long long>(d.max_seq));
    EncodeTiledFn encode = reinterpret_cast<EncodeTiledFn>(plan.encode);
    Tcgen05Plan::ExtKey key;
    key.kv_rows = kv_rows; key.interval = interval; key.batch = batch;
    key.pk = mods.pk; key.pv = mods.pv; key.ps1 = mods.ps1; key.ps2 = mods.ps2; key.plen = mods.plen;
    if (!(plan.ext_key == key)) {
        plan.ext_key = Tcgen05Plan::ExtKey();
        const cuuint32_t es[5] = {1, 1, 1, 1, 1};
        {
            cuuint64_t dims[5] = {128, static_cast<cuuint64_t>(group), interval, d.kv_heads, d.max_batch};
            cuuint64_t strides[4] = {256, d.max_batch * d.q_heads * 256, static_cast<cuuint64_t>(group) * 256, d.q_heads * 256};
            cuuint32_t box[5] = {64, static_cast<cuuint32_t>(group), static_cast<cuuint32_t>(tile_pos), 1, 1};
            if (encode(&plan.ext_q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<void*>(d.q), dims, strides, box, es,
                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
                snprintf(plan.why, sizeof(plan.why), "cuTensorMapEncodeTiled(q) failed");
                return ELLM_ERR_UNSUPPORTED;
            }
        }
        auto kv_map = [&](CUtensorMap* map, const void* base, long long rows, size_t s_pos, size_t s_head, size_t s_seq, size_t seqs) {
            return tcgen05_kv_map(plan, map, base, rows, d.kv_heads, s_pos, s_head, s_seq, seqs);
        };
        if (!kv_map(&plan.ext_k, d.k_cache, kv_rows, d.kv_strides[2], d.kv_strides[1], d.kv_strides[0], batch) ||
            !kv_map(&plan.ext_v, d.v_cache, kv_rows, d.kv_strides[2], d.kv_strides[1], d.kv_strides[0], batch) ||
            (mods.plen > 0 && (!kv_map(&plan.ext_pk, mods.pk, mods.plen, mods.ps2, mods.ps1, mods.ps1, 1) ||
                               !kv_map(&plan.ext_pv, mods.pv, mods.plen, mods.ps2, mods.ps1, mods.ps1, 1)))) {
            snprintf(plan.why, sizeof(plan.why), "cuTensorMapEncodeTiled(k/v) failed");
            return ELLM_ERR_UNSUPPORTED;
        }
        if (mods.plen == 0) {   // never read; any valid map will do
            plan.ext_pk = plan.ext_k;
            plan.ext_pv = plan.ext_v;
        }
        plan.ext_key = key;
    }
    TcParamsExt p{};
    p.out = d.out;
    p.lse = lse;
    p.status = status;
    p.positions = positions;
    p.base = static_cast<long long>(position_index);
    p.key_begin = 0;
    p.key_end = kv_rows;
    p.max_seq = static_cast<long long>(d.max_seq);
    p.interval = static_cast<int>(interval);
    p.batch = static_cast<int>(batch);
    p.max_batch = static_cast<int>(d.max_batch);
    p.q_heads = static_cast<int>(d.q_heads);
    p.kv_heads = static_cast<int>(d.kv_heads);
    p.group = group;
    p.wait_timeout_ns = plan.wait_timeout_ns;
    p.debug_skip_item = plan.debug_skip_item;
    p.scale_log2 = d.scale * kLog2e;
    p.ext.mods = mods;
    p.ext.tile_pos = tile_pos;
    p.ext.tiles = static_cast<int>((interval + tile_pos - 1) / tile_pos);
    p.ext.prefix_tiles = static_cast<int>((mods.plen + kTcKeys - 1) / kTcKeys);
    const float c[6] = {kTanhC0, kTanhC1, kTanhC2, kTanhC3, kTanhC4, kTanhC5};
    for (int i = 0; i < 6; ++i) p.ext.cap_coef[i] = static_cast<float>(c[i] * std::pow(static_cast<double>(mods.cap_in), 2 * i + 1) * mods.cap_log2);
    p.ext.q = static_cast<const __nv_bfloat16*>(d.q);
    p.ext.k = static_cast<const __nv_bfloat16*>(d.k_cache);
    p.ext.v = static_cast<const __nv_bfloat16*>(d.v_cache);
    p.ext.s0 = d.kv_strides[0]; p.ext.s1 = d.kv_strides[1]; p.ext.s2 = d.kv_strides[2];
    p.pair_tiles = (p.ext.tiles + kTcTiles - 1) / kTcTiles;
    const unsigned long long items = static_cast<unsigned long long>(p.pair_tiles) * p.kv_heads * p.batch;
    if (items > 0x7fffffffull || batch > 65535) {
        snprintf(plan.why, sizeof(plan.why), "too many row tiles for one launch");
        return ELLM_ERR_UNSUPPORTED;
    }
    p.n_items = static_cast<long long>(items);
    const bool persistent = plan.sched != nullptr && (plan.persistent < 0 ? true : plan.persistent != 0);
    p.sched = persistent ? plan.sched : nullptr;
    const unsigned long long kv_bytes = 2ull * (static_cast<unsigned long long>(kv_rows) * batch + mods.plen) * 256ull * d.kv_heads;
    p.pair_major = kv_bytes <= (96ull << 20) ? 1 : 0;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (mods.row_begin) {
        p.ext.ranges = plan.ranges;
        cfg.gridDim = dim3(static_cast<unsigned>(p.ext.tiles), static_cast<unsigned>(batch));
        cfg.blockDim = dim3(128);
        if (cudaLaunchKernelEx(&cfg, tc_ranges_kernel, mods, positions, p.base, p.interval, p.max_seq, tile_pos, p.ext.tiles, plan.ranges) != cudaSuccess)
            return ELLM_ERR_CUDA;
    }
    cfg.gridDim = dim3(static_cast<unsigned>(persistent ? std::min<unsigned long long>(items, static_cast<unsigned long long>(plan.sm_count)) : items));
    cfg.blockDim = dim3(kTcThreads);
    cfg.dynamicSmemBytes = kTcSmemBytes;
    auto launch = [&](auto kernel) { return cudaLaunchKernelEx(&cfg, kernel, plan.ext_q, plan.ext_k, plan.ext_v, plan.ext_pk, plan.ext_pv, p); };
    const bool cap = mods.cap_log2 != 0.0f, bias = mods.slopes != nullptr;
    const cudaError_t e = cap && bias ? launch(prefill_tcgen05_kernel<__nv_bfloat16, false, kExtOn | kExtCap | kExtBias>)
                          : cap       ? launch(prefill_tcgen05_kernel<__nv_bfloat16, false, kExtOn | kExtCap>)
                          : bias      ? launch(prefill_tcgen05_kernel<__nv_bfloat16, false, kExtOn | kExtBias>)
                                      : launch(prefill_tcgen05_kernel<__nv_bfloat16, false, kExtOn>);
    return e == cudaSuccess ? ELLM_OK : ELLM_ERR_CUDA;
}

}  // namespace ellm
