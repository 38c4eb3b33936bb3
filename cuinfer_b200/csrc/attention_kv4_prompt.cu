// Prompt attention over the cache that is held in 4 bits (kv4.cuh) on the 5th-generation tensor cores: bfloat16, head size 64 or 128.
//
//   * A CTA has an SM alone and owns two tiles of 128 rows (query token x query head of one kv head) that walk the same 64-key tiles:
//     what taking a key tile apart costs is shared by 256 rows.
//   * Eight warps take the codes apart, four the keys and four the values (four for both were the bottleneck: 2 450 cycles a key tile).  A warp's
//     lanes read 16 bytes of codes each straight from global memory, a tile ahead (through bulk copies into shared memory the copies' barriers took
//     as long as the arithmetic), and write bfloat16 numbers into
//     the tiles that the tensor cores read (128-byte swizzle).  step * (code - zero) is exact in bfloat16, so these are the cache's
//     numbers.  Keys are a K-major operand, [key][value column]; values too, but transposed, [value column][key]: a word of value codes
//     holds two neighbouring keys of a column, which is the order that operand has.
//   * S = Q K^T and O += P V are `tcgen05.mma.cta_group::1.kind::f16`, S, P and O in tensor memory (2 x (64 + 64 + 128) columns), issued by one
//     thread; S of key tile j + 1 is computed while the softmax warps take the exponentials of tile j.
//   * Eight softmax warps, a thread per row: running maximum in base 2 that is raised when it grows by more than 8 (or at all over the
//     first 256 keys); P goes back over its scores in bfloat16, which rounds each weight once (2^-8 of it), the sum is of the weights before that.
//   * Rows see the keys up to their position, the last `window` of them, and none of a page that the block table does not name.  A value that is not
//     a number must not reach rows that do not see its key (0 x NaN is NaN): it is written as zero, and where a CTA has met one, its rows look
//     through the words of the values that they see at the end.
//
// Which two tiles: neighbours where there are more CTAs than SMs (they see almost the same keys); else tile i and the last but i of a
// request (`folded`), so that all CTAs of a launch that fits the GPU at once have the same work.
//
// Where a launch would leave SMs without work, the key tiles of a CTA are cut over several (`gridDim.z`); each then writes its rows' maximum, sum and
// weighted values, 32-bit, to scratch memory that the caller brings, and a second kernel joins them: three portions of up to 500 tokens behind up to
// 3 500 others (72 CTAs without) took 116 us, 62 so.
//
// Every mbarrier wait is bounded; on a time-out the kernel raises the error flag, stops, frees its tensor memory and returns.
#include "kv4.cuh"
#include "mma_utils.cuh"
#include "tcgen05_utils.cuh"

namespace cib {
namespace kv4p {

using namespace kv4;

constexpr int kM = 128;               // rows of a tile
constexpr int kN = 64;                // keys of a tile
constexpr int kSoftWarps = 8;         // four to a row tile
constexpr int kTakeWarps = 4;         // take the keys apart, and as many the values
constexpr int kMmaWarp = kSoftWarps + 2 * kTakeWarps;          // two of them: one for each row tile
constexpr int kThreads = (kMmaWarp + 2) * 32;
// Registers a thread: the launch gives every warp 96 (18 warps take the place of 20); the softmax warps get 24 of each taking warp's.
constexpr int kLaunchRegs = 96, kSoftRegs = 120, kTakeRegs = 72;
static_assert(kSoftWarps * kSoftRegs + 2 * kTakeWarps * kTakeRegs == (kSoftWarps + 2 * kTakeWarps) * kLaunchRegs, "no warp may wait for registers that are not there");
constexpr int kTmemCols = 512;        // per row tile: S of even key tiles | S of odd ones | O

constexpr uint32_t kMinus2p127 = 0xff00ff00u, k2p127 = 0x7f007f00u, k2p123 = 0x7d007d00u, k64 = 0x42804280u;

__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) { return fma_bf16x2(a, b, 0x80008000u); }
template <int N>
struct alignas(N * 4) Words {
    uint32_t w[N];
};

__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// umma_desc_k_major_sw128 of an address in shared memory
__device__ __forceinline__ uint64_t desc_k_major(uint32_t addr) {
    return (uint64_t)((addr & 0x3ffff) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// Loads that stay where they are written, a tile ahead of their use (the compiler moved plain ones down to it: 59 us for a prompt of 2 048 tokens
// instead of 53).
__device__ __forceinline__ void fetch(Words<4>& x, const Words<4>* p) {
    asm volatile("ld.global.nc.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x.w[0]), "=r"(x.w[1]), "=r"(x.w[2]), "=r"(x.w[3]) : "l"(p));
}
__device__ __forceinline__ void fetch(Words<2>& x, const Words<2>* p) { asm volatile("ld.global.nc.v2.b32 {%0, %1}, [%2];" : "=r"(x.w[0]), "=r"(x.w[1]) : "l"(p)); }
__device__ __forceinline__ void fetch(Words<1>& x, const Words<1>* p) { asm volatile("ld.global.nc.b32 %0, [%1];" : "=r"(x.w[0]) : "l"(p)); }
// D = F32, A = B = BF16, both K-major, M = 128
__host__ __device__ constexpr uint32_t idesc(int n) { return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24); }
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a_tmem), "l"(b), "r"(id), "r"(acc) : "memory");
}
__device__ __forceinline__ void tst32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
          "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
          "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
// two 32-bit numbers at a time
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ void tst_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <int D>
struct Smem {
    static constexpr int kPanels = D / 64;                         // 64-column panels of a query or key row
    static constexpr int kQ = kPanels * kM * 128, kK = kPanels * kN * 128, kV = D * 128;
    static constexpr int kBars = 2 * kQ + 2 * kK + 2 * kV;
    static constexpr int kTotal = kBars + 256 + 1024;
};

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
attention_prompt_kernel(const __nv_bfloat16* __restrict__ q, int q_stride, __nv_bfloat16* __restrict__ out, int out_stride,
                        const unsigned char* __restrict__ cache, int num_pages, int page_size, const int* __restrict__ block_table, int table_stride, int table_cols,
                        const int* __restrict__ query_start_loc, const int* __restrict__ seq_lens, int num_requests, int least_query, int nq, int nkv,
                        float scale_log2, int window, int folded, float* __restrict__ part_o, float* __restrict__ part_ml, int num_tokens, int* __restrict__ error_flag) {
    constexpr int NG = D / kGroup, HG = NG / 2;
    constexpr int kBytes = block_bytes(D);
    using S = Smem<D>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* sQ = base;                                       // two row tiles
    unsigned char* sK = base + 2 * S::kQ;                           // key tile j in buffer j % 2
    unsigned char* sV = sK + 2 * S::kK;
    uint64_t* bars = reinterpret_cast<uint64_t*>(base + S::kBars);
    uint64_t* k_full = bars;            // [2] a key tile is in shared memory (the taking warps arrive)
    uint64_t* v_full = bars + 2;        // [2] its values are
    uint64_t* s_full = bars + 4;        // [row tile][2] S of a key tile is in tensor memory: its keys' buffer is free
    uint64_t* p_ready = bars + 8;       // [row tile][2] P is (the softmax warps arrive)
    uint64_t* pv_done = bars + 12;      // [row tile][2] O includes a key tile: its values' buffer is free
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 16);
    __shared__ int s_req, s_pair, s_abort, s_q0, s_n, s_seq;
    // Which of a key tile's blocks the table does not name, tile j at j % 4: written when every row is through with tile j - 4.  Of a row tile that
    // walks tile j - 2 its S says so (P V of tile j - 4 was issued before it); of one that ends earlier, P of tile j - 4.
    __shared__ int s_missing[4];
    __shared__ int s_odd;               // a value that is not a number has been met

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int kvh = blockIdx.x;         // heads vary fastest: every head's longest tiles start before any shorter ones
    const int g = nq / nkv;

    if (warp == 0) {
        // which request and which of its pairs of row tiles, 32 requests at a time
        int t = gridDim.y - 1 - blockIdx.y;     // later (longer) tiles first
        int req = num_requests, pair = 0;
        for (int r0 = 0; r0 < num_requests; r0 += 32) {
            const int r = r0 + lane;
            int pairs = 0;
            if (r < num_requests) {
                const int n = query_start_loc[r + 1] - query_start_loc[r];
                pairs = n < least_query ? 0 : (n * g + 2 * kM - 1) / (2 * kM);
            }
            int upto = pairs;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int o = __shfl_up_sync(0xffffffffu, upto, d);
                if (lane >= d) upto += o;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, r < num_requests && t < upto);
            if (hit) {
                const int first = __ffs(hit) - 1;
                req = r0 + first;
                pair = t - (__shfl_sync(0xffffffffu, upto, first) - __shfl_sync(0xffffffffu, pairs, first));
                break;
            }
            t -= __shfl_sync(0xffffffffu, upto, 31);
        }
        if (lane == 0) {
            s_req = req, s_pair = pair, s_abort = 0;
            s_odd = 0;
            if (req < num_requests) {
                s_q0 = query_start_loc[req];
                s_n = query_start_loc[req + 1] - query_start_loc[req];
                s_seq = seq_lens[req];
            }
        }
    } else if (warp == 1 && lane < 16) {
        mbar_init(&bars[lane], lane < 4 ? kTakeWarps : lane >= 8 && lane < 12 ? 4 : 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (tid < 4) s_missing[tid] = 0;
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem_u32(tmem_slot)), "r"((uint32_t)kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    griddep_wait();          // queries and this step's keys and values come from the kernel before
    griddep_launch();
    const uint32_t tmem = *tmem_slot;
    const int r = s_req;
    const bool active = r < num_requests;

    // the two row tiles: first rows, and how many key tiles they walk from k_lo on (the second may be absent: no rows)
    int q0 = 0, n = 0, seq_len = 0, rows_total = 0, k_lo = 0;
    int row0[2] = {0, 0}, tiles[2] = {0, 0};
    bool has[2] = {false, false};
    if (active) {
        q0 = s_q0, n = s_n, seq_len = s_seq;
        rows_total = n * g;
        const int row_tiles = (rows_total + kM - 1) / kM;
        const int a = folded ? s_pair : 2 * s_pair, b = folded ? row_tiles - 1 - s_pair : 2 * s_pair + 1;
        row0[0] = a * kM, row0[1] = b * kM;
        has[0] = true, has[1] = b < row_tiles && b != a;
        if (window > 0) k_lo = max(0, max(0, seq_len - n + row0[0] / g) - window + 1) / kN * kN;       // (a window may be 2^31 - 1)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int last = min(row0[t] + kM, rows_total) - 1;
            const int keys = seq_len - n + last / g + 1;              // that the tile's last row sees, from the first on
            tiles[t] = has[t] && keys > k_lo ? (keys - k_lo + kN - 1) / kN : 0;
        }
    }
    if (gridDim.z > 1) {                        // this CTA's share of the key tiles
        const int share = (max(tiles[0], tiles[1]) + (int)gridDim.z - 1) / (int)gridDim.z, j0 = (int)blockIdx.z * share;
        k_lo += j0 * kN;
#pragma unroll
        for (int t = 0; t < 2; ++t) tiles[t] = min(max(tiles[t] - j0, 0), share);
    }
    const int most = max(tiles[0], tiles[1]);

    if (active && warp < kSoftWarps) {
        // ---- the query tiles: row = token_local * g + head_in_group, swizzled 64-column panels ----
        const int t = warp >> 2;
        constexpr int kChunks = D / 8, kPer = kM * kChunks / 128;
        if (has[t]) {
#pragma unroll 8
            for (int u = 0; u < kPer; ++u) {
                const int idx = (tid & 127) + u * 128;
                const int row = idx / kChunks, c = idx % kChunks;
                const int grow = row0[t] + row;
                uint4 v = make_uint4(0, 0, 0, 0);
                if (grow < rows_total) {
                    const int tl = grow / g, hi = grow - tl * g;
                    v = *reinterpret_cast<const uint4*>(q + (size_t)(q0 + tl) * q_stride + (size_t)(kvh * g + hi) * D + c * 8);
                }
                *reinterpret_cast<uint4*>(sQ + t * S::kQ + (c >> 3) * (kM * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = v;
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp < kSoftWarps || warp >= kMmaWarp) asm volatile("bar.sync 10, %0;" ::"r"((kSoftWarps + 2) * 32) : "memory");

    auto wait_all = [&](uint64_t* bar, uint32_t parity, int code) {
        bool ok = mbar_try_wait(bar, parity) || (*(volatile int*)&s_abort == 0 && mbar_wait(bar, parity));
        if (!ok && lane == 0) { atomicExch(error_flag, code); *(volatile int*)&s_abort = 1; }
        return __all_sync(0xffffffffu, ok) != 0;
    };

    if (active && warp >= kMmaWarp) {
        // ---- the MMAs: a warp for each row tile walks its loop, one lane issues (one warp for both was busy for 2 350 of 2 450 cycles a key
        // tile).  Addresses are broadcast, so that the compiler knows them to be the warp's and keeps them in uniform registers (out of
        // per-thread ones an MMA took 72 cycles to issue) ----
        const int t = __shfl_sync(0xffffffffu, warp - kMmaWarp, 0);
        const int my_tiles = t == 0 ? tiles[0] : tiles[1];
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0) + t * 256;
        const uint32_t aq = __shfl_sync(0xffffffffu, tc_smem_u32(sQ), 0) + t * S::kQ, ak = __shfl_sync(0xffffffffu, tc_smem_u32(sK), 0), av = __shfl_sync(0xffffffffu, tc_smem_u32(sV), 0);
        const bool elected = elect_one();
        auto issue_s = [&](int j) {
            const int b = j & 1;
            if (elected) {
                const uint64_t qd = desc_k_major(aq), kd = desc_k_major(ak + b * S::kK);
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint64_t q_off = (uint64_t)(((k >> 2) * (kM * 128) + (k & 3) * 32) >> 4), k_off = (uint64_t)(((k >> 2) * (kN * 128) + (k & 3) * 32) >> 4);
                    umma_bf16(tm + (uint32_t)(b * kN), qd + q_off, kd + k_off, idesc(kN), k != 0);
                }
                umma_commit(&s_full[t * 2 + b]);
            }
            __syncwarp();
        };
        bool ok = true;
        if (my_tiles > 0) {
            ok = wait_all(&k_full[0], 0, 51);
            if (ok) {
                tcgen05_fence_after();
                issue_s(0);
            }
        }
        for (int j = 0; j < my_tiles && ok; ++j) {
            const int b = j & 1;
            const uint32_t parity = (j >> 1) & 1;
            if (j + 1 < my_tiles) {
                // S(j + 1) overwrites S and P of tile j - 1: P V(j - 1) was issued before, and the tensor pipe runs what one thread issues in order
                ok = wait_all(&k_full[(j + 1) & 1], ((j + 1) >> 1) & 1, 52);
                if (!ok) break;
                tcgen05_fence_after();
                issue_s(j + 1);
            }
            ok = wait_all(&v_full[b], parity, 53) && wait_all(&p_ready[t * 2 + b], parity, 54);
            if (!ok) break;
            tcgen05_fence_after();
            if (elected) {
                const uint64_t vd = desc_k_major(av + b * S::kV);
#pragma unroll
                for (int k = 0; k < kN / 16; ++k)
                    mma_ts(tm + (uint32_t)(2 * kN), tm + (uint32_t)(b * kN + k * 8), vd + (uint64_t)(k * 32 >> 4), idesc(D), j > 0 || k != 0);
                umma_commit(&pv_done[t * 2 + b]);
            }
            __syncwarp();
        }
    } else if (active && warp >= kSoftWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTakeRegs));
        // ---- taking the codes apart: warps 0-3 of these the keys, 4-7 the values ----
        const int take = (warp - kSoftWarps) & 3;
        const bool values = warp >= kSoftWarps + kTakeWarps;
        const int* table = block_table + (size_t)r * table_stride;
        const int per_page = page_size / kBlock;
        // the number of block `block` of key tile j, or -1 (no such tile, behind the last key, or not named by the table)
        auto lookup = [&](int j, int block) {
            const int b = (k_lo + j * kN) / kBlock + block, index = b / per_page;
            if (j >= most || b * kBlock >= seq_len || index >= table_cols) return -1;
            const int page = __ldg(table + index);
            return page >= 0 && page < num_pages ? (page * nkv + kvh) * per_page + (b - index * per_page) : -1;
        };
        // a tile's buffer is free when both row tiles are through with tile j - 2
        auto free_again = [&](uint64_t* bars2, int j, int code) {
            const uint32_t parity = (uint32_t)(((j >> 1) - 1) & 1);
            return (j - 2 < 0 || j - 2 >= tiles[0] || wait_all(&bars2[j & 1], parity, code)) && (j - 2 < 0 || j - 2 >= tiles[1] || wait_all(&bars2[2 + (j & 1)], parity, code + 1));
        };
        if (!values) {
            // a warp has one of the tile's four blocks; lane = (token, quarter), tokens in the order 0 4 1 5 2 6 3 7 so that the 16-byte stores
            // of eight lanes meet in no bank
            const int quarter = lane & 3, token = ((lane >> 3) & 3) + ((lane >> 2) & 1) * 4;
            struct Codes {
                Words<NG> c[2];
                Words<HG> w[2];
                int id;
            };
            int ids = lookup(lane, take), ids_next = -1;            // lane l: this warp's block of tile 32 n + l
            auto load = [&](int j) {
                Codes x;
                if ((j & 31) == 0 && j != 0) ids = ids_next;
                if ((j & 31) == 16) ids_next = lookup((j & ~31) + 32 + lane, take);
                x.id = __shfl_sync(0xffffffffu, ids, j & 31);
                const unsigned char* kb = cache + (size_t)max(x.id, 0) * kBytes;       // (a block that is not there: any other, its scores are replaced)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    fetch(x.c[h], reinterpret_cast<const Words<NG>*>(kb) + (token + 8 * h) * 4 + quarter);
                    fetch(x.w[h], reinterpret_cast<const Words<HG>*>(kb + key_words_at(D)) + token + 8 * h);
                }
                return x;
            };
            Codes next = load(0);
            for (int j = 0; j < most; ++j) {
                const int b = j & 1;
                const Codes x = next;
                if (j + 1 < most) next = load(j + 1);
                if (!free_again(s_full, j, 55)) break;
                // a row tile that has no tile j - 2 any more may still be at its last two (no later phase of these barriers follows)
                bool through = true;
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    if (j - 4 >= 0 && j - 4 < tiles[t] && j - 2 >= tiles[t]) through = through && wait_all(&p_ready[2 * t + b], (uint32_t)((j >> 1) & 1), 63);
                if (!through) break;
                if (lane == 0) {
                    if (x.id < 0 && k_lo + j * kN + take * kBlock < seq_len) atomicOr(&s_missing[j & 3], 1 << take);
                    else atomicAnd(&s_missing[j & 3], ~(1 << take));
                }
                unsigned char* kt = sK + b * S::kK;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int row = take * kBlock + token + 8 * h;
#pragma unroll
                    for (int k = 0; k < NG; ++k) {
                        const uint32_t w = k & 1 ? __byte_perm(x.w[h].w[k >> 1], 0, 0x3232) : __byte_perm(x.w[h].w[k >> 1], 0, 0x1010);
                        const uint32_t zero = mul_bf16x2(w & 0x000f000fu, kMinus2p127), step = mul_bf16x2(w & 0xfff0fff0u, k64);
                        const uint32_t lo = x.c[h].w[k], hi = lo >> 8;
                        uint4 v;
                        v.x = mul_bf16x2(fma_bf16x2(lo & 0x000f000fu, k2p127, zero), step);
                        v.y = mul_bf16x2(fma_bf16x2(lo & 0x00f000f0u, k2p123, zero), step);
                        v.z = mul_bf16x2(fma_bf16x2(hi & 0x000f000fu, k2p127, zero), step);
                        v.w = mul_bf16x2(fma_bf16x2(hi & 0x00f000f0u, k2p123, zero), step);
                        *reinterpret_cast<uint4*>(kt + (k >> 1) * (kN * 128) + row * 128 + ((((k & 1) * 4 + quarter) ^ (row & 7)) << 4)) = v;
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&k_full[b]);
            }
        } else {
            // lane = (eight keys, eighth of a group); a warp has half of the eighths and half of the groups
            const int octet = lane & 7, eighth = (take >> 1) * 4 + (lane >> 3), g0 = (take & 1) * HG;
            struct Codes {
                Words<HG> c[4], w[4];
                int id;
            };
            // lanes 4 i .. 4 i + 3: the blocks of tile 8 n + i
            int ids = lookup(lane >> 2, lane & 3), ids_next = -1;
            auto load = [&](int j) {
                Codes x;
                if ((j & 7) == 0 && j != 0) ids = ids_next;
                if ((j & 7) == 4) ids_next = lookup((j & ~7) + 8 + (lane >> 2), lane & 3);
                x.id = __shfl_sync(0xffffffffu, ids, (j & 7) * 4 + (octet >> 1));
                const unsigned char* vb = cache + (size_t)max(x.id, 0) * kBytes;
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    fetch(x.c[p], reinterpret_cast<const Words<HG>*>(vb + value_codes_at(D)) + (((octet & 1) * 8 + eighth) * 4 + p) * 2 + (take & 1));
                    fetch(x.w[p], reinterpret_cast<const Words<HG>*>(vb + value_words_at(D)) + ((octet & 1) * 4 + p) * 2 + (take & 1));
                }
                return x;
            };
            Codes next = load(0);
            for (int j = 0; j < most; ++j) {
                const int b = j & 1;
                const int key0 = k_lo + j * kN;
                Codes x = next;
                if (j + 1 < most) next = load(j + 1);
                if (key0 + kN > seq_len || __any_sync(0xffffffffu, x.id < 0)) {      // keys behind the last one, and of no page: their weights are zero
#pragma unroll
                    for (int p = 0; p < 4; ++p) {
                        const int key = key0 + octet * 8 + 2 * p;
                        const uint32_t keep = x.id < 0 ? 0u : (key < seq_len ? 0xffffu : 0u) | (key + 1 < seq_len ? 0xffff0000u : 0u);
#pragma unroll
                        for (int k = 0; k < HG; ++k) x.w[p].w[k] &= keep;
                    }
                }
                uint32_t odd = 0;                                   // a sign bit is set where a word is not a number
#pragma unroll
                for (int p = 0; p < 4; ++p)
#pragma unroll
                    for (int k = 0; k < HG; ++k) odd |= (x.w[p].w[k] & 0x7f807f80u) + 0x00800080u;
                if (odd & 0x80008000u) {
                    atomicExch(&s_odd, 1);
#pragma unroll
                    for (int p = 0; p < 4; ++p)
#pragma unroll
                        for (int k = 0; k < HG; ++k) {
                            const uint32_t at = ((x.w[p].w[k] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
                            x.w[p].w[k] &= (at & 0x8000u ? 0u : 0xffffu) | (at & 0x80000000u ? 0u : 0xffff0000u);
                        }
                }
                if (!free_again(pv_done, j, 57)) break;
                unsigned char* vt = sV + b * S::kV;
#pragma unroll
                for (int k = 0; k < HG; ++k) {
                    uint32_t v[4][4];                               // [column][pair of keys]
#pragma unroll
                    for (int p = 0; p < 4; ++p) {
                        const uint32_t w = x.w[p].w[k], zero = mul_bf16x2(w & 0x000f000fu, kMinus2p127), step = mul_bf16x2(w & 0xfff0fff0u, k64);
                        const uint32_t lo = x.c[p].w[k], hi = lo >> 8;
                        v[0][p] = mul_bf16x2(fma_bf16x2(lo & 0x000f000fu, k2p127, zero), step);
                        v[1][p] = mul_bf16x2(fma_bf16x2(lo & 0x00f000f0u, k2p123, zero), step);
                        v[2][p] = mul_bf16x2(fma_bf16x2(hi & 0x000f000fu, k2p127, zero), step);
                        v[3][p] = mul_bf16x2(fma_bf16x2(hi & 0x00f000f0u, k2p123, zero), step);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int row = (g0 + k) * kGroup + eighth * 4 + i;
                        *reinterpret_cast<uint4*>(vt + row * 128 + ((octet ^ (row & 7)) << 4)) = make_uint4(v[i][0], v[i][1], v[i][2], v[i][3]);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&v_full[b]);
            }
        }
    } else if (active && warp < kSoftWarps) {
        // ---- softmax: a thread per row (TMEM lane 32 * (warp % 4) + lane) ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
        const int t = warp >> 2;
        const int my_tiles = tiles[t];
        const int row_local = tid & 127;
        const int grow = row0[t] + row_local;
        const bool row_ok = has[t] && grow < rows_total;
        const int pos = row_ok ? seq_len - n + grow / g : -1;
        const uint32_t lane_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(t * 256), o_addr = lane_addr + 2 * kN;
        float m_used = -INFINITY, l = 0.f;
        bool ok = true;
        for (int j = 0; j < my_tiles; ++j) {
            const int b = j & 1;
            const int key0 = k_lo + j * kN;
            ok = wait_all(&s_full[t * 2 + b], (uint32_t)((j >> 1) & 1), 59);
            if (!ok) break;
            tcgen05_fence_after();
            const int missing = *(volatile int*)&s_missing[j & 3];
            const bool need_mask = key0 + kN - 1 > pos || window > 0 || missing != 0;
            const int hi = pos - key0;                              // columns <= hi are visible ...
            const int lo = window > 0 ? hi - window : -1;           // ... and > lo
            uint32_t v[2][32];
            tmem_ld_32x32b_x32(lane_addr + (uint32_t)(b * kN), v[0]);
            tmem_ld_32x32b_x32(lane_addr + (uint32_t)(b * kN + 32), v[1]);
            tmem_ld_wait();
            if (need_mask) {
#pragma unroll
                for (int e = 0; e < kN; ++e)
                    if (!(e <= hi && e > lo) || ((missing >> (e / kBlock)) & 1)) v[e / 32][e % 32] = __float_as_uint(-INFINITY);
            }
            // P = 2^(s * scale - m), two at a time: a packed multiply-add, two ex2, a packed addition and a conversion.  From the fifth tile on m is
            // taken as it is and the tile's maximum found meanwhile; where it is more than 8 above m, the weights are computed again.
            float part[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            auto largest = [&]() {
#pragma unroll
                for (int e = 0; e < kN; e += 2)
                    part[(e >> 1) & 3] = max3(part[(e >> 1) & 3], __uint_as_float(v[e / 32][e % 32]), __uint_as_float(v[e / 32][e % 32 + 1]));
                return fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])) * scale_log2;
            };
            float corr = 1.f;
            bool rescale = false;
            auto raise = [&](float mx, float by) {
                if (mx > m_used + by || (m_used == -INFINITY && mx != -INFINITY)) {
                    corr = m_used == -INFINITY ? 0.f : exp2f(m_used - mx);
                    m_used = mx;
                    l *= corr;
                    rescale = j > 0;
                }
            };
            const uint64_t scale2 = pack2(scale_log2, scale_log2);
            uint32_t p[32];
            float2 sum;
            auto weights = [&]() {
                const float m_eff = m_used == -INFINITY ? 0.f : m_used;
                const uint64_t minus_m = pack2(-m_eff, -m_eff);
                uint64_t sums[2] = {0, 0};
#pragma unroll
                for (int e = 0; e < kN; e += 2) {
                    const float2 x = unpack2(fma2(pack2(__uint_as_float(v[e / 32][e % 32]), __uint_as_float(v[e / 32][e % 32 + 1])), scale2, minus_m));
                    float2 y;
                    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y.x) : "f"(x.x));
                    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y.y) : "f"(x.y));
                    sums[(e >> 1) & 1] = add2(sums[(e >> 1) & 1], pack2(y.x, y.y));
                    p[e / 2] = pack_bf16(y.x, y.y);
                }
                sum = unpack2(add2(sums[0], sums[1]));
            };
            if (j < 256 / kN) {
                raise(largest(), 0.f);
                weights();
            } else {
                weights();
                const float mx = largest();
                if (__any_sync(0xffffffffu, mx > m_used + 8.f || (m_used == -INFINITY && mx != -INFINITY))) {
                    raise(mx, 8.f);
                    weights();
                }
            }
            l += sum.x + sum.y;
            if (j > 0 && __any_sync(0xffffffffu, rescale)) {
                ok = wait_all(&pv_done[t * 2 + (b ^ 1)], (uint32_t)(((j - 1) >> 1) & 1), 60);
                if (!ok) break;
                tcgen05_fence_after();
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    uint32_t o[32];
                    tmem_ld_32x32b_x32(o_addr + (uint32_t)c, o);
                    tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                    tst32(o_addr + (uint32_t)c, o);
                }
            }
            tst32(lane_addr + (uint32_t)(b * kN), p);
            tst_wait();
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_ready[t * 2 + b]);
        }
        // every thread waits for the last P V itself: behind it no MMA reads this tile's shared or tensor memory
        if (ok && my_tiles > 0) ok = wait_all(&pv_done[t * 2 + ((my_tiles - 1) & 1)], (uint32_t)(((my_tiles - 1) >> 1) & 1), 62);
        tcgen05_fence_after();
        unsigned char* stage = sQ + t * S::kQ;                      // (every S has read the queries)
        constexpr int kPieces = D / 8;                              // 16-byte pieces of a row
        if (*(volatile int*)&s_abort == 0 && has[t]) {
            const bool whole = gridDim.z == 1;
            const float f = !whole ? 1.f : l == 0.f ? 0.f : __fdividef(1.f, l);
            unsigned bad = 0;                           // groups whose sum holds a value that is not a number
            if (*(volatile int*)&s_odd && row_ok) {
                const int* table = block_table + (size_t)r * table_stride;
                for (int key = window > 0 ? max(0, pos - window + 1) : 0; key <= pos && key / page_size < table_cols; ++key) {
                    const int page = table[key / page_size];
                    if (page < 0 || page >= num_pages) continue;
                    const unsigned char* block = cache + ((size_t)(page * nkv + kvh) * (page_size / kBlock) + key % page_size / kBlock) * kBytes;
                    const uint16_t* words = reinterpret_cast<const uint16_t*>(block + value_words_at(D)) + ((key % kBlock) >> 1) * NG * 2 + (key & 1);
                    for (int k = 0; k < NG; ++k)
                        if ((words[2 * k] & 0x7f80u) == 0x7f80u) bad |= 1u << k;
                }
            }
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                uint32_t o[32];
                if (my_tiles > 0) {
                    tmem_ld_32x32b_x32(o_addr + (uint32_t)c, o);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = 0;
                }
                const float ff = (bad >> (c / kGroup)) & 1u ? NAN : f;
                if (!whole) {
                    if (row_ok) {
                        const int tl = grow / g;
                        const size_t at = ((size_t)blockIdx.z * num_tokens + q0 + tl) * nq + kvh * g + (grow - tl * g);
                        if (c == 0) part_ml[at * 2] = m_used, part_ml[at * 2 + 1] = l;
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            *reinterpret_cast<float4*>(part_o + at * D + c + e) = make_float4(__uint_as_float(o[e]) * ff, __uint_as_float(o[e + 1]) * ff,
                                                                                          __uint_as_float(o[e + 2]) * ff, __uint_as_float(o[e + 3]) * ff);
                    }
                    continue;
                }
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                    uint4 pk;
                    pk.x = pack_bf16(__uint_as_float(o[e]) * ff, __uint_as_float(o[e + 1]) * ff);
                    pk.y = pack_bf16(__uint_as_float(o[e + 2]) * ff, __uint_as_float(o[e + 3]) * ff);
                    pk.z = pack_bf16(__uint_as_float(o[e + 4]) * ff, __uint_as_float(o[e + 5]) * ff);
                    pk.w = pack_bf16(__uint_as_float(o[e + 6]) * ff, __uint_as_float(o[e + 7]) * ff);
                    const int piece = (c + e) >> 3;
                    *reinterpret_cast<uint4*>(stage + row_local * (D * 2) + ((piece ^ (row_local & (kPieces - 1))) << 4)) = pk;
                }
            }
        }
        asm volatile("bar.sync %0, 128;" ::"r"(11 + t) : "memory");
        if (*(volatile int*)&s_abort == 0 && has[t] && gridDim.z == 1) {
#pragma unroll
            for (int u = 0; u < kM * kPieces / 128; ++u) {
                const int idx = row_local + u * 128;
                const int row = idx / kPieces, c = idx % kPieces;
                const int grow_out = row0[t] + row;
                if (grow_out < rows_total) {
                    const uint4 pk = *reinterpret_cast<const uint4*>(stage + row * (D * 2) + ((c ^ (row & (kPieces - 1))) << 4));
                    const int tl = grow_out / g, hh = grow_out - tl * g;
                    *reinterpret_cast<uint4*>(out + (size_t)(q0 + tl) * out_stride + (size_t)(kvh * g + hh) * D + c * 8) = pk;
                }
            }
        }
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)kTmemCols) : "memory");
}

// A warp per (token, query head): joins the shares of the keys.
template <int D>
__global__ void __launch_bounds__(128)
attention_prompt_merge_kernel(__nv_bfloat16* __restrict__ out, int out_stride, const int* __restrict__ query_start_loc, int num_requests, int least_query, int nq,
                              int shares, int num_tokens, const float* __restrict__ part_o, const float* __restrict__ part_ml) {
    const int lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int t = (int)(item / nq), head = (int)(item - (long long)t * nq);
    if (t >= num_tokens) return;                                   // (no barrier follows)
    int before = 0;                                                // the request of this row: the last one that starts at or before it
    for (int r0 = 0; r0 <= num_requests; r0 += 32) {
        const int r = r0 + lane;
        before += __popc(__ballot_sync(0xffffffffu, r <= num_requests && query_start_loc[min(r, num_requests)] <= t));
    }
    griddep_wait();
    griddep_launch();
    const int r = before - 1;
    if (r < 0 || r >= num_requests || query_start_loc[r + 1] - query_start_loc[r] < least_query) return;
    constexpr int E = D / 32;
    float M = -INFINITY, L = 0.f, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    for (int z = 0; z < shares; ++z) M = fmaxf(M, part_ml[(((size_t)z * num_tokens + t) * nq + head) * 2]);
    for (int z = 0; z < shares; ++z) {
        const size_t at = ((size_t)z * num_tokens + t) * nq + head;
        const float m = part_ml[at * 2];
        const float f = m == -INFINITY ? 0.f : exp2f(m - M);
        L += part_ml[at * 2 + 1] * f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] += part_o[at * D + lane * E + e] * f;
    }
    const float f = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int e = 0; e < E; e += 2)
        *reinterpret_cast<uint32_t*>(out + (size_t)t * out_stride + (size_t)head * D + lane * E + e) = pack_bf16(o[e] * f, o[e + 1] * f);
}

// The registers that a launch gives a thread: the split among the warps counts on them.
template <typename Kernel>
static int launch_registers(Kernel kernel) {
    cudaFuncAttributes a;
    return cudaFuncGetAttributes(&a, kernel) == cudaSuccess ? a.numRegs : -1;
}

}  // namespace kv4p
}  // namespace cib

using namespace cib;

extern "C" int cib_attention_kv4_prompt_supports(int d, int page_size) { return kv4::sizes_ok(d, page_size) && (d == 64 || d == 128); }

// num_pairs = sum over requests of ceil(tokens_r * (nq / nkv) / 256), or more: CTAs that find none leave.  least_query: requests that bring
// fewer tokens are left as they are.  shares: how many CTAs share the keys of a pair of row tiles; scratch: shares * num_tokens * nq * (d + 2) floats where
// there are several.
extern "C" int cib_attention_kv4_prompt(const void* q, int q_stride, void* out, int out_stride, const void* cache, int num_pages, int page_size,
                                        const int* block_table, int table_stride, int table_cols, const int* query_start_loc, const int* seq_lens, int num_requests,
                                        int num_tokens, int num_pairs, int folded, int shares, int least_query, int nq, int nkv, int d, float scale, int window, float* scratch, int* error_flag,
                                        cudaStream_t stream) {
    CIB_REQUIRE(cib_attention_kv4_prompt_supports(d, page_size), "attention_kv4_prompt: head size %d (64 or 128), page size %d (a multiple of 16) are not taken", d, page_size);
    CIB_REQUIRE(num_requests >= 0 && nq > 0 && nkv > 0 && nq % nkv == 0 && num_pairs >= 0 && num_pairs <= 65535, "attention_kv4_prompt: bad sizes");
    CIB_REQUIRE(num_pages > 0 && table_stride > 0 && table_cols > 0 && cache != nullptr && ((uintptr_t)cache % 16) == 0, "attention_kv4_prompt: bad cache geometry");
    CIB_REQUIRE((long long)num_pages * nkv * (page_size / kv4::kBlock) < (1ll << 31), "attention_kv4_prompt: more than 2^31 blocks");
    CIB_REQUIRE(q_stride % 8 == 0 && ((uintptr_t)q % 16) == 0 && out_stride % 8 == 0 && ((uintptr_t)out % 16) == 0, "attention_kv4_prompt: rows must be 16-byte aligned");
    CIB_REQUIRE(shares >= 1 && shares <= 65535 && (shares == 1 || (scratch != nullptr && (uintptr_t)scratch % 16 == 0)), "attention_kv4_prompt: %d shares need scratch", shares);
    CIB_REQUIRE((long long)num_tokens * nq < (1ll << 31), "attention_kv4_prompt: too many rows");
    CIB_REQUIRE(window >= 0 && error_flag != nullptr, "attention_kv4_prompt: window must be >= 0, error flag given");
    if (num_requests == 0 || num_pairs == 0) return 0;
    const float scale_log2 = scale * 1.4426950408889634f;
    float* part_ml = shares > 1 ? scratch + (size_t)shares * num_tokens * nq * d : nullptr;
#define CIB_KV4_PROMPT(DV)                                                                                                                          \
    if (d == DV) {                                                                                                                                  \
        static SmemLimit limit;                                                                                                                     \
        if (int rc = raise_smem_limit(limit, kv4p::attention_prompt_kernel<DV>, kv4p::Smem<DV>::kTotal, "attention_kv4_prompt")) return rc;         \
        static const int regs = kv4p::launch_registers(kv4p::attention_prompt_kernel<DV>);                                                          \
        CIB_REQUIRE(regs == kv4p::kLaunchRegs, "attention_kv4_prompt: built with %d registers a thread, laid out for %d", regs, kv4p::kLaunchRegs); \
        cudaError_t e = launch_pdl(kv4p::attention_prompt_kernel<DV>, dim3(nkv, num_pairs, shares), dim3(kv4p::kThreads),                           \
                                   (size_t)kv4p::Smem<DV>::kTotal, stream, prompt_pdl(), (const __nv_bfloat16*)q, q_stride, (__nv_bfloat16*)out,    \
                                   out_stride, (const unsigned char*)cache, num_pages, page_size, block_table, table_stride, table_cols, query_start_loc, \
                                   seq_lens, num_requests, least_query, nq, nkv, scale_log2, window, folded, scratch, part_ml, num_tokens,          \
                                   error_flag);                                                                                                     \
        if (e == cudaSuccess && shares > 1)                                                                                                         \
            e = launch_pdl(kv4p::attention_prompt_merge_kernel<DV>, dim3((unsigned)(((long long)num_tokens * nq + 3) / 4)), dim3(128), 0, stream,   \
                           prompt_pdl(), (__nv_bfloat16*)out, out_stride, query_start_loc, num_requests, least_query, nq, shares, num_tokens,       \
                           scratch, part_ml);                                                                                                       \
        CIB_REQUIRE(e == cudaSuccess, "attention_kv4_prompt: launch failed: %s", cudaGetErrorString(e));                                            \
        return 0;                                                                                                                                   \
    }
    CIB_KV4_PROMPT(64)
    CIB_KV4_PROMPT(128)
#undef CIB_KV4_PROMPT
    return -1;
}
