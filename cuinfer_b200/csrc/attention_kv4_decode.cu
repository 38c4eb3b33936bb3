// Attention of single tokens over the cache that is held in 4 bits (kv4.cuh): bfloat16, head size 64, 128 or 256.
//
// Decode is a stream of the cache through the SMs: 9/8 D bytes a token and kv head.  The 16-token blocks of a (request, kv head) are
// split over `splits` CTAs and inside a CTA over four warps; a warp copies two blocks at a time into a private ring
// of shared memory (a block is one contiguous piece: one `cp.async.bulk` each, counted on an mbarrier) and multiplies them with up to
// eight query heads by mma.m16n8k16 with the quantised operand as A (16 keys, or 16 value columns) and the heads as the 8 columns:
//
//   scores   S^T[key, head] = sum over groups g of step[key, g] * (sum of code q) - sum over g of step zero sum_g(q)
//   values   O^T[column, head] += sum over keys of (code - zero) * (p step),  p = 2^(s - m)
//
// What bounds such a kernel is taking the codes apart: the integer pipe does one operation in two cycles of a scheduler.  A bfloat16 whose
// bits are v < 256 is v 2^-133 (its subnormals and the first normal binade are one linear range), so four bits of a word are an
// operand as they stand: a code masked out of bits 0-3 is c 2^-133, out of bits 4-7 16 c 2^-133, and one shift by 8 serves
// the other two: 5 operations for 8 codes, where placing each code under an exponent took 7.  The queries are multiplied by a power of
// two a head, so that their largest lies in [2^126, 2^127), and by 1/16 against the codes of bits 4-7; the scores take it back.
// The zero points of all groups are one more MMA (two at head size 256) with step * zero (four bits times four) against the sums of q, which are
// split into four bfloat16 parts.  All operands of the scores are exact.  For the values one fused multiply-add on the other pipe gives (code - zero) 2^-6,
// also exact; only p * step is rounded, once: p enters that product as two bfloat16 parts.  The weights come out of the scores with keys as rows
// and go in with keys as the summed index: an 8 x 8 transposition in registers (movmatrix) for 8 keys and part.
//
// A running maximum and sum per head in base 2, in 32 bits; the warps of a CTA are merged in shared memory.
//
// Few (request, head block)s of moderate length: a cluster of up to eight CTAs shares the blocks of each, the partial results stay in the CTAs' shared memory
// and every CTA reads its share of the columns from all of them (distributed shared memory).  No list, no scratch, no second kernel: 8 requests of
// 4 096 tokens took 18.4 + 7.4 us with those, 18.8 so; one of 300 10.7 in one CTA a head, 7.8 so.
//
// Else the work of a launch is one list: the blocks of request 0, head block 0, then head block 1, .. , request 1, .., in units of `unit`
// blocks.  The launch has as many CTAs as the GPU holds at once and every CTA takes the same number of consecutive units, found from the
// lengths on the device: requests of any lengths end together, and a recorded launch fits whatever lengths it is replayed with.
// What a CTA has of a (request, head block) goes straight to the output if it is all of it; else it is a partial result: its first or its
// last piece, so two places a CTA in scratch memory that the caller brings hold them all, and a second kernel joins them (nothing global is
// counted or kept, so any number of launches may run at once).  64 requests of 1 024 to 8 192 tokens, 32 heads over 8: equal numbers of
// splits for every request left the SMs idle a third of the time.
#include "kv4.cuh"
#include "mma_utils.cuh"
#include "tcgen05_utils.cuh"

#include <cooperative_groups.h>

namespace cib {
namespace kv4 {

constexpr int kDecWarps = 4;
constexpr int kDecStages = 3;
constexpr int kDecCluster = 8;       // CTAs that share a (request, head block), at most
constexpr int kDecHeads = 8;         // query heads of a CTA: the columns of an MMA

template <int D>
constexpr int stage_bytes() { return 2 * block_bytes(D); }
template <int D>
constexpr int ring_bytes() { return kDecWarps * kDecStages * stage_bytes<D>(); }

// The blocks [first, first + count) of a request that its last token sees.
struct Span {
    int first, count;
};
__device__ __forceinline__ Span span_of(int seq_len, int window) {
    const int lo = window > 0 ? max(0, seq_len - window) : 0;
    const int first = lo / kBlock;
    return {first, max(0, (int)(((long long)seq_len + kBlock - 1) / kBlock) - first)};
}
// Units of a request for each head block; a single token without keys has one too (its row is zero), other requests none.
__device__ __forceinline__ int units_of(int r, const int* query_start_loc, const int* seq_lens, int window, int unit) {
    if (query_start_loc[r + 1] - query_start_loc[r] != 1) return 0;
    return max(1, (span_of(seq_lens[r], window).count + unit - 1) / unit);
}
// Where the list of units stands: a warp sums up the requests' units and finds the request that unit `at` of head block 0.. lies in.
struct Place {
    long long total, before;         // all units; those of the requests in front of `request`
    int request;
};
__device__ __forceinline__ Place warp_find(long long at_part, int parts, int num_requests, const int* query_start_loc, const int* seq_lens, int window,
                                           int unit, int head_blocks) {
    const int lane = threadIdx.x & 31;
    Place p{0, 0, num_requests};
    for (int r0 = 0; r0 < num_requests; r0 += 32) {
        const int r = r0 + lane;
        long long n = r < num_requests ? (long long)units_of(r, query_start_loc, seq_lens, window, unit) * head_blocks : 0;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) n += __shfl_xor_sync(0xffffffffu, n, d);
        p.total += n;
    }
    const long long share = (p.total + parts - 1) / parts, at = at_part * share;
    long long before = 0;
    for (int r0 = 0; r0 < num_requests && at < p.total; r0 += 32) {
        const int r = r0 + lane;
        long long upto = r < num_requests ? (long long)units_of(r, query_start_loc, seq_lens, window, unit) * head_blocks : 0;
        const long long own = upto;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const long long o = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += o;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, before + upto > at);
        if (hit) {
            const int first = __ffs(hit) - 1;
            p.request = r0 + first;
            p.before = before + __shfl_sync(0xffffffffu, upto - own, first);
            break;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return p;
}

template <int N>
struct alignas(N * 4) Words {
    uint32_t w[N];
};
__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) { return fma_bf16x2(a, b, 0x80008000u); }     // (+ -0)
// pairs of bfloat16 constants
constexpr uint32_t k2p127 = 0x7f007f00u, kMinus2p127 = 0xff00ff00u, k2p123 = 0x7d007d00u;
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
    return r;
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same onto zero
__device__ __forceinline__ void mma16816_0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(tc_smem_u32(dst)), "l"(src), "r"(bytes), "r"(tc_smem_u32(bar)) : "memory");
}

// CLUSTER: gridDim.x CTAs, one cluster, for each (request, head block) blockIdx.y; else the list.
template <int D, bool CLUSTER>
__global__ void __launch_bounds__(kDecWarps * 32, D > 128 ? 2 : 4)
attention_decode_kernel(const __nv_bfloat16* __restrict__ q, int q_stride, __nv_bfloat16* __restrict__ out, int out_stride,
                        const unsigned char* __restrict__ cache, int num_pages, int page_size, const int* __restrict__ block_table, int table_stride, int table_cols,
                        const int* __restrict__ query_start_loc, const int* __restrict__ seq_lens, int num_requests, int nq, int nkv, float scale_log2, int window,
                        int unit, float* __restrict__ part_o, float* __restrict__ part_ml, int* __restrict__ error_flag) {
    constexpr int NG = D / kGroup;
    constexpr int kBytes = block_bytes(D);
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ uint64_t s_full[kDecWarps * kDecStages];
    __shared__ Place s_place;
    __shared__ int s_failed;         // a wait ran out: no further piece of the list is begun
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane & 3, row = lane >> 2;
    const int g = nq / nkv, blocks_per_kv = (g + kDecHeads - 1) / kDecHeads, head_blocks = nkv * blocks_per_kv;

    if (lane < kDecStages) mbar_init(&s_full[warp * kDecStages + lane], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (threadIdx.x == 0) s_failed = 0;
    if (!CLUSTER && warp == 0) {
        const Place p = warp_find(blockIdx.x, gridDim.x, num_requests, query_start_loc, seq_lens, window, unit, head_blocks);
        if (lane == 0) s_place = p;
    }
    __syncthreads();
    griddep_wait();          // queries and this step's keys and values come from the kernel before
    griddep_launch();
    const int per_page = page_size / kBlock;
    unsigned char* ring = smem + warp * kDecStages * stage_bytes<D>();
    uint64_t* full = s_full + warp * kDecStages;
    int st = 0;                      // the ring stage that is read next, and the parity of its barrier
    uint32_t parity = 0;
    long long share = 0, to = 1, before = 0, at = 0;
    int r = CLUSTER ? (int)blockIdx.y / head_blocks : 0;
    if (!CLUSTER) {
        const Place place = s_place;
        share = (place.total + gridDim.x - 1) / gridDim.x;
        at = blockIdx.x * share, to = min(place.total, at + share);
        before = place.before, r = place.request;
    }
    const long long from = at;

    while (at < to) {
    int hblock, u0, u1, step = unit;                              // units of `step` blocks
    bool first_piece = true, alone = true;
    if constexpr (CLUSTER) {
        if (query_start_loc[r + 1] - query_start_loc[r] != 1) return;          // (the whole cluster)
        hblock = (int)blockIdx.y - r * head_blocks;
        // equal shares in steps of two blocks, and two for every warp at least
        const int blocks = span_of(seq_lens[r], window).count, mine = (blocks + (int)gridDim.x - 1) / (int)gridDim.x;
        step = max(2 * kDecWarps, (mine + 1) / 2 * 2);
        u0 = min((int)blockIdx.x, (blocks + step - 1) / step), u1 = u0 + 1;
        at = to;
    } else {
        int units = units_of(r, query_start_loc, seq_lens, window, unit);
        while (at >= before + (long long)units * head_blocks) {
            before += (long long)units * head_blocks;
            units = units_of(++r, query_start_loc, seq_lens, window, unit);
        }
        const int local = (int)(at - before);
        hblock = local / units, u0 = local - hblock * units;
        u1 = (int)min((long long)units, u0 + (to - at));
        first_piece = at == from;
        at += u1 - u0;
        alone = u0 == 0 && u1 == units;
    }
    const int kvh = hblock / blocks_per_kv, hb = hblock - kvh * blocks_per_kv;
    const int head0 = kvh * g + hb * kDecHeads, nh = min(kDecHeads, g - hb * kDecHeads);
    const int token = query_start_loc[r];
    const int seq_len = seq_lens[r];
    const Span span = span_of(seq_len, window);
    const int begin = span.first + min(span.count, u0 * step), end = span.first + min(span.count, u1 * step);
    const int lo = window > 0 ? max(0, seq_len - window) : 0;
    const int* table = block_table + (size_t)r * table_stride;

    // this warp's pairs of blocks: begin + 2 (i * warps + warp), i = 0 .. count - 1
    const int pairs = (end - begin + 1) / 2;
    const int count = pairs > warp ? (pairs - warp + kDecWarps - 1) / kDecWarps : 0;
    // lanes 2 j and 2 j + 1 look up the blocks of pair 16 n + j, a batch of 16 pairs ahead of its use
    auto lookup = [&](int batch) {
        const int i = batch * 16 + (lane >> 1);
        const int b = begin + 2 * (i * kDecWarps + warp) + (lane & 1);
        if (i >= count || b >= end) return -1;
        const int index = b / per_page;
        if (index >= table_cols) return -1;
        const int page = table[index];
        return page >= 0 && page < num_pages ? (page * nkv + kvh) * per_page + (b - index * per_page) : -1;
    };
    int ids = lookup(0), ids_next = lookup(1);
    uint32_t named = __ballot_sync(0xffffffffu, ids >= 0);       // two bits a pair of the batch: which of its blocks the table names
    uint32_t present = 0;                                        // the same of the pairs on their way, the oldest in the lowest bits
    int fill = st;
    auto request = [&](int i, int in_flight) {
        if (i != 0 && (i & 15) == 0) {
            ids = ids_next;
            ids_next = lookup((i >> 4) + 1);
            named = __ballot_sync(0xffffffffu, ids >= 0);
        }
        const uint32_t here = (named >> (2 * (i & 15))) & 3u;
        present |= here << (2 * in_flight);
        if (lane == 0) mbar_expect_tx(&full[fill], __popc(here) * kBytes);
        __syncwarp();
        if ((lane >> 1) == (i & 15) && ids >= 0)
            bulk_load(ring + fill * stage_bytes<D>() + (lane & 1) * kBytes, cache + (size_t)ids * kBytes, kBytes, &full[fill]);
        fill = fill == kDecStages - 1 ? 0 : fill + 1;
    };
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kDecStages - 2; ++i)
        if (i < count) request(i, i);

    // ---- queries: the B operand, head = column `row`; a lane has values 32 g + 8 quad .. + 7 of every group ----
    uint32_t qf[NG][4];
    float largest = 0.f;
    {
        const __nv_bfloat16* qp = q + (size_t)token * q_stride + (size_t)(head0 + row) * D + 8 * quad;
#pragma unroll
        for (int k = 0; k < NG; ++k) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (row < nh) v = *reinterpret_cast<const uint4*>(qp + k * kGroup);
            qf[k][0] = v.x, qf[k][1] = v.y, qf[k][2] = v.z, qf[k][3] = v.w;
#pragma unroll
            for (int u = 0; u < 4; ++u) largest = fmaxf(largest, fmaxf(fabsf(__uint_as_float(qf[k][u] << 16)), fabsf(__uint_as_float(qf[k][u] & 0xffff0000u))));
        }
    }
    largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
    largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
    // 2^-e for the head's largest |q| in [2^e, 2^(e + 1)); e = 0 for a head of zeros and one that is not finite
    const int exponent = largest > 1.1754944e-38f && largest < INFINITY ? (int)(__float_as_uint(largest) >> 23) - 127 : 0;
    const float down = __uint_as_float((uint32_t)(127 - exponent) << 23), tiny = exponent == 127 ? 5.877472e-39f : down;
    // minus half the sums of the scaled queries in bfloat16 parts: the B operand of the zero points.  The summed index runs over (part,
    // group pair): quads hold part quad / kPairs of a pair, then the parts behind those.  Four pairs leave room for two parts in an MMA, which
    // are 16 bits of a sum that may have 24: their last two parts are an MMA of their own.
    constexpr int kPairs = NG / 2, kSums = kPairs == 4 ? 4 : 2;
    uint32_t sums[kSums] = {};
    const int my_pair = quad % kPairs;
#pragma unroll
    for (int k = 0; k < NG; ++k) {
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float a = __uint_as_float(qf[k][u] << 16) * tiny, c = __uint_as_float(qf[k][u] & 0xffff0000u) * tiny;
            sum += a + c;
            const float up = u & 1 ? 5.3169119831396635e+36f : 8.507059173023462e+37f;       // 2^122 against 16 c, 2^126 against c
            qf[k][u] = pack_bf16(a * up, c * up);
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        float rest = -0.5f * sum;
        uint32_t part[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const __nv_bfloat16 h = __float2bfloat16_rn(rest);
            part[u] = __bfloat16_as_ushort(h);
            rest -= __bfloat162float(h);
        }
        constexpr int kFirst = 4 / kPairs;                      // parts in the first half of the index
        if ((k >> 1) == my_pair) {
            const int p0 = quad / kPairs, p1 = kFirst + p0;
            const uint32_t a = p0 == 0 ? part[0] : p0 == 1 ? part[1] : p0 == 2 ? part[2] : part[3];
            const uint32_t b = p1 == 1 ? part[1] : p1 == 2 ? part[2] : p1 == 3 ? part[3] : 0u;
            sums[0] |= a << (16 * (k & 1));
            sums[1] |= b << (16 * (k & 1));
            if constexpr (kSums == 4) sums[2] |= part[2] << (16 * (k & 1)), sums[3] |= part[3] << (16 * (k & 1));
        }
    }
    // a sum of products stands for 2^(-7 - e) of the score; of heads 2 quad and 2 quad + 1 (column c is held by lanes 4 c ..)
    float back[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) back[e] = scale_log2 * 128.f * (1.f / __shfl_sync(0xffffffffu, down, 4 * (2 * quad + e)));

    float o[2 * NG][4];
#pragma unroll
    for (int i = 0; i < 2 * NG; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    // ---- scores of the 32 keys of a stage, scaled; keys that are not seen: -inf, and their values' words cleared (what lies where no token
    // has been written may be anything) ----
    auto scores = [&](unsigned char* stage, int block0, uint32_t here, float (&s)[2][4]) {
        const bool whole = here == 3u && block0 * kBlock >= lo && (block0 + 2) * kBlock <= seq_len;
        if (!whole) {
            const int key = block0 * kBlock + lane;
            if (!((here >> (lane >> 4)) & 1u) || key < lo || key >= seq_len) {
                uint16_t* words = reinterpret_cast<uint16_t*>(stage + (lane >> 4) * kBytes + value_words_at(D)) + ((lane & 15) >> 1) * NG * 2 + (lane & 1);
#pragma unroll
                for (int k = 0; k < NG; ++k) words[2 * k] = 0;
            }
            __syncwarp();
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const unsigned char* block = stage + b * kBytes;
            const Words<NG> c0 = reinterpret_cast<const Words<NG>*>(block)[lane], c1 = reinterpret_cast<const Words<NG>*>(block)[32 + lane];
            const uint32_t* words = reinterpret_cast<const uint32_t*>(block + key_words_at(D));
            const Words<kPairs> w0 = reinterpret_cast<const Words<kPairs>*>(words)[row], w1 = reinterpret_cast<const Words<kPairs>*>(words)[row + 8];
            {
                const uint32_t a = words[row * kPairs + my_pair], c = words[(row + 8) * kPairs + my_pair];
                const uint32_t za = mul_bf16x2(mul_bf16x2(a & 0x000f000fu, k2p127), a & 0xfff0fff0u);
                const uint32_t zc = mul_bf16x2(mul_bf16x2(c & 0x000f000fu, k2p127), c & 0xfff0fff0u);
                mma16816_0(s[b], za, zc, za, zc, sums[0], sums[1]);
                if constexpr (kSums == 4) mma16816(s[b], za, zc, za, zc, sums[2], sums[3]);
            }
#pragma unroll
            for (int k = 0; k < NG; ++k) {
                float acc[4];
                const uint32_t x0 = c0.w[k], x1 = c1.w[k], y0 = x0 >> 8, y1 = x1 >> 8;
                mma16816_0(acc, x0 & 0x000f000fu, x1 & 0x000f000fu, x0 & 0x00f000f0u, x1 & 0x00f000f0u, qf[k][0], qf[k][1]);
                mma16816(acc, y0 & 0x000f000fu, y1 & 0x000f000fu, y0 & 0x00f000f0u, y1 & 0x00f000f0u, qf[k][2], qf[k][3]);
                const uint32_t a = w0.w[k >> 1], c = w1.w[k >> 1];
                const float sa = __uint_as_float((k & 1 ? a : a << 16) & 0xfff00000u), sc = __uint_as_float((k & 1 ? c : c << 16) & 0xfff00000u);
                s[b][0] = fmaf(sa, acc[0], s[b][0]);
                s[b][1] = fmaf(sa, acc[1], s[b][1]);
                s[b][2] = fmaf(sc, acc[2], s[b][2]);
                s[b][3] = fmaf(sc, acc[3], s[b][3]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) s[b][e] *= back[e & 1];
        }
        if (!whole) {
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int key = (block0 + b) * kBlock + row + 8 * h;
                    if (!((here >> b) & 1u) || key < lo || key >= seq_len) s[b][2 * h] = s[b][2 * h + 1] = -INFINITY;
                }
        }
    };
    // ---- O += (p step) (code - zero) of a stage.  p enters as two bfloat16 parts, so that only p * step is rounded (2^-8 of it; what the parts
    // leave out is 2^-16) ----
    auto values = [&](const unsigned char* stage, const uint32_t (&ph)[2][2], const uint32_t (&pl)[2][2]) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const unsigned char* block = stage + b * kBytes;
            const Words<NG>* words = reinterpret_cast<const Words<NG>*>(block + value_words_at(D));
            const Words<NG> z0 = words[quad], z1 = words[4 + quad];
            const Words<NG>* codes = reinterpret_cast<const Words<NG>*>(block + value_codes_at(D));
            const Words<NG> v0 = codes[lane], v1 = codes[32 + lane];
#pragma unroll
            for (int k = 0; k < NG; ++k) {
                const uint32_t sa = z0.w[k] & 0xfff0fff0u, sc = z1.w[k] & 0xfff0fff0u;
                const uint32_t b0 = fma_bf16x2(ph[b][0], sa, mul_bf16x2(pl[b][0], sa)), b1 = fma_bf16x2(ph[b][1], sc, mul_bf16x2(pl[b][1], sc));
                const uint32_t za = mul_bf16x2(z0.w[k] & 0x000f000fu, kMinus2p127), zc = mul_bf16x2(z1.w[k] & 0x000f000fu, kMinus2p127);
                uint32_t x0 = v0.w[k], x1 = v1.w[k];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    mma16816(o[2 * k + t], fma_bf16x2(x0 & 0x000f000fu, k2p127, za), fma_bf16x2(x0 & 0x00f000f0u, k2p123, za),
                             fma_bf16x2(x1 & 0x000f000fu, k2p127, zc), fma_bf16x2(x1 & 0x00f000f0u, k2p123, zc), b0, b1);
                    x0 >>= 8, x1 >>= 8;
                }
            }
        }
    };
    // weights of a stage's scores: running maximum (heads 2 quad, e = 0, and 2 quad + 1), sums, and the transposed parts of p
    auto weigh = [&](const float (&s)[2][4], uint32_t (&ph)[2][2], uint32_t (&pl)[2][2]) {
        float top[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float x = fmaxf(fmaxf(s[0][e], s[0][2 + e]), fmaxf(s[1][e], s[1][2 + e]));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            top[e] = fmaxf(m[e], x);
        }
        if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
            float corr[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                corr[e] = m[e] == -INFINITY ? 0.f : ex2(m[e] - top[e]);
                m[e] = top[e];
                l[e] *= corr[e];
            }
#pragma unroll
            for (int t = 0; t < 2 * NG; ++t) o[t][0] *= corr[0], o[t][1] *= corr[1], o[t][2] *= corr[0], o[t][3] *= corr[1];
        }
        const float base[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float p0 = ex2(s[b][2 * h] - base[0]), p1 = ex2(s[b][2 * h + 1] - base[1]);
                l[0] += p0, l[1] += p1;
                const uint32_t hi = pack_bf16(p0, p1);
                ph[b][h] = transpose8(hi);
                pl[b][h] = transpose8(pack_bf16(p0 - __uint_as_float(hi << 16), p1 - __uint_as_float(hi & 0xffff0000u)));
            }
    };
    // stage i has landed (false: the wait ran out); the stage that pair i - 2 was read from is refilled
    auto arrive = [&](int i) {
        // (every warp waits for its own copies, of which one pair of blocks is on its way here, also where another warp's wait has run out)
        const bool landed = mbar_try_wait(&full[st], parity) || mbar_wait(&full[st], parity);
        if (!__all_sync(0xffffffffu, landed)) {
            if (lane == 0) atomicExch(error_flag, 41), *(volatile int*)&s_failed = 1;
            return false;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");        // (every lane has finished reading that stage)
        __syncwarp();
        if (i + kDecStages - 2 < count) request(i + kDecStages - 2, kDecStages - 2);
        return true;
    };
    // The scores of pair i + 1 are computed beside the weighted sum of pair i: one is integer work and short of independent products,
    // the other fused multiply-adds.
    uint32_t ph[2][2], pl[2][2];
    unsigned char* stage = ring + st * stage_bytes<D>();
    if (count > 0) {
        float s[2][4];
        bool ok = arrive(0);
        if (ok) {
            scores(stage, begin + 2 * warp, present & 3u, s);
            present >>= 2;
            weigh(s, ph, pl);
        }
        for (int i = 1; i < count && ok; ++i) {
            const unsigned char* last = stage;
            if (++st == kDecStages) st = 0, parity ^= 1u;
            stage = ring + st * stage_bytes<D>();
            ok = arrive(i);
            if (!ok) break;
            scores(stage, begin + 2 * (i * kDecWarps + warp), present & 3u, s);
            present >>= 2;
            values(last, ph, pl);
            weigh(s, ph, pl);
        }
        if (ok) values(stage, ph, pl);
        if (++st == kDecStages) st = 0, parity ^= 1u;
    }
    __syncthreads();     // all rings have been read
    // ---- merge the warps: [warp][head][D] values, [warp][head] maxima and sums ----
    float* sm_o = reinterpret_cast<float*>(smem);
    float* sm_m = sm_o + kDecWarps * kDecHeads * D;
    float* sm_l = sm_m + kDecWarps * kDecHeads;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        float x = l[e];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        const int head = 2 * quad + e;
        if (row == 0) sm_m[warp * kDecHeads + head] = m[e], sm_l[warp * kDecHeads + head] = x;
        float4* dst = reinterpret_cast<float4*>(sm_o + (size_t)(warp * kDecHeads + head) * D) + row;
#pragma unroll
        for (int k = 0; k < NG; ++k) dst[k * 8] = make_float4(o[2 * k][e], o[2 * k][2 + e], o[2 * k + 1][e], o[2 * k + 1][2 + e]);
    }
    __syncthreads();
    float* sm_part = sm_l + kDecWarps * kDecHeads;                // a cluster's CTA: [head][D] values, [head][2] maximum and sum
    for (int i = threadIdx.x; i < nh * D; i += kDecWarps * 32) {
        const int h = i / D, x = i - h * D;
        float M = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
        for (int w = 0; w < kDecWarps; ++w) M = fmaxf(M, sm_m[w * kDecHeads + h]);
#pragma unroll
        for (int w = 0; w < kDecWarps; ++w) {
            const float f = sm_m[w * kDecHeads + h] == -INFINITY ? 0.f : ex2(sm_m[w * kDecHeads + h] - M);
            L += sm_l[w * kDecHeads + h] * f;
            O += sm_o[(size_t)(w * kDecHeads + h) * D + x] * f;
        }
        O *= 64.f;                              // (the operands were (code - zero) 2^-6)
        if (CLUSTER && gridDim.x > 1) {
            sm_part[i] = O;
            if (x == 0) sm_part[kDecHeads * D + h * 2] = M, sm_part[kDecHeads * D + h * 2 + 1] = L;
        } else if (alone) {
            out[(size_t)token * out_stride + (size_t)(head0 + h) * D + x] = __float2bfloat16_rn(L == 0.f ? 0.f : O / L);
        } else {
            const size_t place = ((size_t)blockIdx.x * 2 + (first_piece ? 0 : 1)) * kDecHeads + h;
            part_o[place * D + x] = O;
            if (x == 0) part_ml[place * 2] = M, part_ml[place * 2 + 1] = L;
        }
    }
    if (CLUSTER && gridDim.x > 1) {
        namespace cg = cooperative_groups;
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();                                           // every CTA's part is in its shared memory
        for (int i = (int)blockIdx.x * kDecWarps * 32 + threadIdx.x; i < nh * D; i += (int)gridDim.x * kDecWarps * 32) {
            const int h = i / D;
            float m[kDecCluster], M = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
            for (int c = 0; c < kDecCluster; ++c) {
                m[c] = c < (int)gridDim.x ? cluster.map_shared_rank(sm_part, c)[kDecHeads * D + h * 2] : -INFINITY;
                M = fmaxf(M, m[c]);
            }
#pragma unroll
            for (int c = 0; c < kDecCluster; ++c) {
                if (c >= (int)gridDim.x) break;
                const float* part = cluster.map_shared_rank(sm_part, c);
                const float f = m[c] == -INFINITY ? 0.f : ex2(m[c] - M);
                L += part[kDecHeads * D + h * 2 + 1] * f;
                O += part[i] * f;
            }
            out[(size_t)token * out_stride + (size_t)head0 * D + i] = __float2bfloat16_rn(L == 0.f ? 0.f : O / L);
        }
        cluster.sync();                                           // (a CTA's shared memory has been read before it leaves)
    }
    if (__syncthreads_or(*(volatile int*)&s_failed)) break;       // (the rings are filled again)
    }
}

// A CTA per (head, request), a thread per value: joins what several CTAs have of it.  The maxima and sums of up to D parts are fetched at once, a
// part a thread; the values then eight parts at a time (part after part, each a trip to the L2, took 13 us for 20 parts).
template <int D>
__global__ void __launch_bounds__(D)
attention_decode_merge_kernel(__nv_bfloat16* __restrict__ out, int out_stride, const int* __restrict__ query_start_loc, const int* __restrict__ seq_lens,
                              int num_requests, int nq, int nkv, int window, int unit, int parts, const float* __restrict__ part_o,
                              const float* __restrict__ part_ml) {
    __shared__ long long s_total[2];
    __shared__ float s_weight[D], s_warp[2][D / 32];
    const int head = blockIdx.x, r = blockIdx.y, x = threadIdx.x;
    const int g = nq / nkv, blocks_per_kv = (g + kDecHeads - 1) / kDecHeads, head_blocks = nkv * blocks_per_kv;
    if (threadIdx.x < 32) {
        long long total = 0, before = 0;
        for (int i = threadIdx.x; i < num_requests; i += 32) {
            const long long n = (long long)units_of(i, query_start_loc, seq_lens, window, unit) * head_blocks;
            total += n;
            before += i < r ? n : 0;
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            total += __shfl_xor_sync(0xffffffffu, total, d);
            before += __shfl_xor_sync(0xffffffffu, before, d);
        }
        if (threadIdx.x == 0) s_total[0] = total, s_total[1] = before;
    }
    __syncthreads();
    griddep_wait();
    griddep_launch();
    const int units = units_of(r, query_start_loc, seq_lens, window, unit);
    if (units == 0) return;
    const int kvh = head / g, in_kv = head - kvh * g, hblock = kvh * blocks_per_kv + in_kv / kDecHeads, h = in_kv % kDecHeads;
    const long long share = (s_total[0] + parts - 1) / parts, from = s_total[1] + (long long)hblock * units, to = from + units;
    const int c0 = (int)(from / share), c1 = (int)((to - 1) / share);
    if (c0 == c1) return;
    // the first CTA has it as its last piece, unless it is also its first; all others as their first
    auto place_of = [&](int c) { return ((size_t)c * 2 + (c == c0 && from != c0 * share ? 1 : 0)) * kDecHeads + h; };
    float M = -INFINITY, L = 0.f, O = 0.f;
    for (int first = c0; first <= c1; first += D) {
        const int count = min(D, c1 + 1 - first);
        float m = -INFINITY, l = 0.f;
        if (x < count) {
            const float2 ml = *reinterpret_cast<const float2*>(part_ml + place_of(first + x) * 2);
            m = ml.x, l = ml.y;
        }
        const float top = warp_max(m);
        if ((x & 31) == 0) s_warp[0][x >> 5] = top;
        __syncthreads();
        float here = M;
#pragma unroll
        for (int w = 0; w < D / 32; ++w) here = fmaxf(here, s_warp[0][w]);
        const float f = m == -INFINITY ? 0.f : ex2(m - here);
        s_weight[x] = f;
        const float sum = warp_sum(l * f);
        if ((x & 31) == 0) s_warp[1][x >> 5] = sum;
        __syncthreads();
        const float keep = M == -INFINITY ? 0.f : ex2(M - here);
        M = here, L *= keep, O *= keep;
#pragma unroll
        for (int w = 0; w < D / 32; ++w) L += s_warp[1][w];
#pragma unroll 8
        for (int c = 0; c < count; ++c) O += part_o[place_of(first + c) * D + x] * s_weight[c];
        __syncthreads();
    }
    out[(size_t)query_start_loc[r] * out_stride + (size_t)head * D + x] = __float2bfloat16_rn(L == 0.f ? 0.f : O / L);
}

}  // namespace kv4
}  // namespace cib

using namespace cib;

extern "C" int cib_attention_kv4_decode_supports(int d, int page_size) {
    return kv4::sizes_ok(d, page_size) && (d == 64 || d == 128 || d == 256);
}

// As many CTAs as an SM holds: shared memory for 4 at head size 128, registers below.
extern "C" int cib_attention_kv4_decode_ctas(int d) { return 148 * (d > 128 ? 2 : 4); }
extern "C" long long cib_attention_kv4_decode_scratch_floats(int d, int ctas) { return (long long)ctas * 2 * kv4::kDecHeads * (d + 2); }

// Computes the rows of the requests that bring one token; the others' are left as they are.  cluster > 0: so many CTAs (1, 2, 4 or 8) share the blocks of
// each (request, head block); ctas, unit and scratch mean nothing then.  Else ctas: how many CTAs share the work; unit: blocks
// of 16 keys that a CTA has at least.  scratch: cib_attention_kv4_decode_scratch_floats, or none where no request has more than `unit`
// blocks (no request is split then, whatever its length).
extern "C" int cib_attention_kv4_decode(const void* q, int q_stride, void* out, int out_stride, const void* cache, int num_pages, int page_size,
                                        const int* block_table, int table_stride, int table_cols, const int* query_start_loc, const int* seq_lens, int num_requests, int nq,
                                        int nkv, int d, float scale, int window, int cluster, int ctas, int unit, float* scratch, int* error_flag, int use_pdl,
                                        cudaStream_t stream) {
    CIB_REQUIRE(cib_attention_kv4_decode_supports(d, page_size), "attention_kv4_decode: head size %d (64, 128 or 256), page size %d (a multiple of 16) are not taken", d, page_size);
    CIB_REQUIRE(num_requests >= 0 && num_requests <= 65535 && nq > 0 && nkv > 0 && nq % nkv == 0, "attention_kv4_decode: bad sizes R=%d nq=%d nkv=%d", num_requests, nq, nkv);
    CIB_REQUIRE(cluster == 0 || cluster == 1 || cluster == 2 || cluster == 4 || cluster == kv4::kDecCluster, "attention_kv4_decode: clusters of 1, 2, 4 or 8, not %d", cluster);
    CIB_REQUIRE(cluster > 0 || (ctas >= 1 && (scratch == nullptr || (unit >= 1 && unit <= 1 << 20))), "attention_kv4_decode: bad launch shape %d, %d", ctas, unit);
    CIB_REQUIRE(num_pages > 0 && table_stride > 0 && table_cols > 0 && cache != nullptr && ((uintptr_t)cache % 16) == 0, "attention_kv4_decode: bad cache geometry");
    CIB_REQUIRE((long long)num_pages * nkv * (page_size / kv4::kBlock) < (1ll << 31), "attention_kv4_decode: more than 2^31 blocks");
    CIB_REQUIRE(q_stride % 8 == 0 && ((uintptr_t)q % 16) == 0, "attention_kv4_decode: query rows must be 16-byte aligned");
    CIB_REQUIRE(window >= 0 && error_flag != nullptr, "attention_kv4_decode: window must be >= 0, error flag given");
    if (num_requests == 0) return 0;
    const float scale_log2 = scale * 1.4426950408889634f;
    if (scratch == nullptr) unit = 1 << 27;          // a request is one unit, so no CTA has a part of it
    const long long pairs = (long long)num_requests * nkv * ((nq / nkv + kv4::kDecHeads - 1) / kv4::kDecHeads);
    CIB_REQUIRE(cluster == 0 || pairs <= 65535, "attention_kv4_decode: %lld (request, head block)s are too many for clusters", pairs);
    float* part_ml = scratch == nullptr ? nullptr : scratch + (size_t)ctas * 2 * kv4::kDecHeads * d;
#define CIB_KV4_DECODE(DV)                                                                                                                           \
    if (d == DV && cluster > 0) {                                                                                                                    \
        static SmemLimit limit;                                                                                                                      \
        if (int rc = raise_smem_limit(limit, kv4::attention_decode_kernel<DV, true>, kv4::ring_bytes<DV>(), "attention_kv4_decode")) return rc;      \
        const cudaError_t e = launch_pdl_cluster(kv4::attention_decode_kernel<DV, true>, dim3(cluster, (unsigned)pairs), dim3(kv4::kDecWarps * 32),  \
                                                 (size_t)kv4::ring_bytes<DV>(), stream, use_pdl != 0, cluster, (const __nv_bfloat16*)q, q_stride,    \
                                                 (__nv_bfloat16*)out, out_stride, (const unsigned char*)cache, num_pages, page_size, block_table,    \
                                                 table_stride, table_cols, query_start_loc, seq_lens, num_requests, nq, nkv, scale_log2, window, 1,  \
                                                 nullptr, nullptr, error_flag);                                                                      \
        CIB_REQUIRE(e == cudaSuccess, "attention_kv4_decode: launch failed: %s", cudaGetErrorString(e));                                             \
        return 0;                                                                                                                                    \
    }                                                                                                                                                \
    if (d == DV) {                                                                                                                                   \
        static SmemLimit limit;                                                                                                                      \
        if (int rc = raise_smem_limit(limit, kv4::attention_decode_kernel<DV, false>, kv4::ring_bytes<DV>(), "attention_kv4_decode")) return rc;     \
        cudaError_t e = launch_pdl(kv4::attention_decode_kernel<DV, false>, dim3(ctas), dim3(kv4::kDecWarps * 32), (size_t)kv4::ring_bytes<DV>(),    \
                                   stream, use_pdl != 0, (const __nv_bfloat16*)q, q_stride, (__nv_bfloat16*)out, out_stride,                         \
                                   (const unsigned char*)cache, num_pages, page_size, block_table, table_stride, table_cols, query_start_loc,       \
                                   seq_lens, num_requests, nq, nkv, scale_log2, window, unit, scratch, part_ml, error_flag);                        \
        if (e == cudaSuccess && scratch != nullptr)                                                                                                  \
            e = launch_pdl(kv4::attention_decode_merge_kernel<DV>, dim3(nq, num_requests), dim3(DV), 0, stream, use_pdl != 0, (__nv_bfloat16*)out,   \
                           out_stride, query_start_loc, seq_lens, num_requests, nq, nkv, window, unit, ctas, scratch, part_ml);                      \
        CIB_REQUIRE(e == cudaSuccess, "attention_kv4_decode: launch failed: %s", cudaGetErrorString(e));                                             \
        return 0;                                                                                                                                    \
    }
    CIB_KV4_DECODE(64)
    CIB_KV4_DECODE(128)
    CIB_KV4_DECODE(256)
#undef CIB_KV4_DECODE
    return -1;
}
