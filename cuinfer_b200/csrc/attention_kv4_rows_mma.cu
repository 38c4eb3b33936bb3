// Prompt attention over the cache that is held in 4 bits (kv4.cuh) by mma.sync: bfloat16 and any head size that is a multiple of 32 up to 256, for the
// sizes (and scales below zero) that the tcgen05 kernel does not take.
//
// A CTA has 64 rows (query token x query head of one kv head) of one request, four warps of 16, and walks tiles of 32 keys.  Its threads take a
// tile's keys and values apart once for all rows, from words that were asked for a tile ahead, into shared memory as bfloat16 numbers (step * (code - zero)
// is exact): keys as [key][column], values transposed, [column][key], because a word of value codes holds two neighbouring keys of a column and
// the second product sums over keys.  Scores stay in registers; in the layout in which m16n8k16 leaves them they are the first operand of the second
// product: p is rounded to bfloat16 once (2^-8 of it), the sum is of the weights before that.  32-bit running maximum and sum per row.
//
// Bound by the latency of a tile's steps (four warps, two CTAs an SM) and mma.sync's rate.  2 x 400 tokens behind 1 600, 8 heads of 256 over 2: 637 us by
// 32-bit multiply-adds, 158 so; 8 heads of 96 262 and 63.
//
// Where a launch would leave SMs without work, a cluster of up to eight CTAs shares the key tiles of 64 rows and joins its parts through
// distributed shared memory.  A value that is not a number must not reach rows that do not see its key (0 x NaN is NaN): it is taken as zero, and where a
// CTA has met one, its rows look through the words of the values that they see at the end.
#include "kv4.cuh"
#include "mma_utils.cuh"

#include <cooperative_groups.h>

namespace cib {
namespace kv4m {

using namespace kv4;

constexpr int kRows = 64, kKeys = 32, kWarps = 4, kCluster = 8;
constexpr int kVPitch = kKeys + 8;                               // (bfloat16; eight rows of 16 bytes meet in no bank)
constexpr uint32_t kMinus2p127 = 0xff00ff00u, k2p127 = 0x7f007f00u, k2p123 = 0x7d007d00u, k64 = 0x42804280u;

template <int NG>
struct Sizes {
    static constexpr int D = kGroup * NG, P = D + 8, F = D + 4;  // pitches of bfloat16 rows, and of a partial result's
    static constexpr int kTiles = ((kRows + kKeys) * P + D * kVPitch) * 2, kPart = (kRows * F + 2 * kRows) * 4;
    static constexpr int kBytes = kTiles > kPart ? kTiles : kPart;
};

__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) { return fma_bf16x2(a, b, 0x80008000u); }
// four 8 x 8 tiles of 16-bit numbers; lane l gives the address of row l % 8 of tile l / 8
__device__ __forceinline__ void load_tiles(uint32_t (&r)[4], const __nv_bfloat16* p) {
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(p);
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

template <int NG>
__global__ void __launch_bounds__(kWarps * 32, 2)
attention_rows_mma_kernel(const __nv_bfloat16* __restrict__ q, int q_stride, __nv_bfloat16* __restrict__ out, int out_stride, const unsigned char* __restrict__ cache,
                          int num_pages, int page_size, const int* __restrict__ block_table, int table_stride, int table_cols,
                          const int* __restrict__ query_start_loc, const int* __restrict__ seq_lens, int num_requests, int least_query, int nq, int nkv,
                          float scale_log2, int window) {
    constexpr int D = Sizes<NG>::D, P = Sizes<NG>::P, F = Sizes<NG>::F;
    extern __shared__ __align__(16) unsigned char smem_b[];
    __nv_bfloat16* sQ = reinterpret_cast<__nv_bfloat16*>(smem_b);
    __nv_bfloat16* sK = sQ + kRows * P;
    __nv_bfloat16* sV = sK + kKeys * P;                          // [column][key]
    float* part = reinterpret_cast<float*>(smem_b);              // at the end, of a cluster's CTA: [row][D], then [row][maximum, sum]
    float* part_ml = part + kRows * F;
    __shared__ int s_req, s_tile, s_named[2], s_odd;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int kvh = blockIdx.z, g = nq / nkv;
    if (warp == 0) {
        // which request and which of its row tiles, 32 requests at a time; later (longer) tiles first
        int t = gridDim.y - 1 - blockIdx.y, req = num_requests, tile = 0;
        for (int r0 = 0; r0 < num_requests; r0 += 32) {
            const int r = r0 + lane;
            int tiles = 0;
            if (r < num_requests) {
                const int n = query_start_loc[r + 1] - query_start_loc[r];
                tiles = n < least_query ? 0 : (n * g + kRows - 1) / kRows;
            }
            int upto = tiles;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int o = __shfl_up_sync(0xffffffffu, upto, d);
                if (lane >= d) upto += o;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, t < upto);
            if (hit) {
                const int first = __ffs(hit) - 1;
                req = r0 + first;
                tile = t - (__shfl_sync(0xffffffffu, upto, first) - __shfl_sync(0xffffffffu, tiles, first));
                break;
            }
            t -= __shfl_sync(0xffffffffu, upto, 31);
        }
        if (lane == 0) s_req = req, s_tile = tile, s_odd = 0;
    }
    __syncthreads();
    griddep_wait();          // queries and this step's keys and values come from the kernel before
    griddep_launch();
    const int r = s_req;
    if (r >= num_requests) return;                               // (the whole cluster)
    const int q0 = query_start_loc[r], n = query_start_loc[r + 1] - q0, seq_len = seq_lens[r];
    const int row0 = s_tile * kRows, rows_total = n * g;
    const int first_pos = seq_len - n + row0 / g, last_pos = seq_len - n + (min(row0 + kRows, rows_total) - 1) / g;
    int k0 = window > 0 ? max(0, max(0, first_pos) - window + 1) / kKeys * kKeys : 0;       // (a window may be 2^31 - 1)
    int tiles = last_pos >= k0 ? (last_pos - k0) / kKeys + 1 : 0;
    {
        const int share = (tiles + (int)gridDim.x - 1) / (int)gridDim.x, j0 = (int)blockIdx.x * share;
        k0 += j0 * kKeys;
        tiles = min(max(tiles - j0, 0), share);
    }

    // ---- this thread's words of a tile: (key, quarter) of the keys, (block, half, eighth, pair) of the values ----
    const int key_in = tid >> 2, quarter = tid & 3, pair = tid & 3, eighth = (tid >> 2) & 7, half = (tid >> 5) & 1, block = tid >> 6;
    const int per_page = page_size / kBlock;
    const int* table = block_table + (size_t)r * table_stride;
    auto lookup = [&](int j) {
        const int b = k0 / kBlock + 2 * j + block, index = b / per_page;
        if (j >= tiles || b * kBlock >= seq_len || index >= table_cols) return -1;
        const int page = table[index];
        return page >= 0 && page < num_pages ? (page * nkv + kvh) * per_page + (b - index * per_page) : -1;
    };
    uint32_t key_code[NG], key_word[NG], value_code[NG], value_word[NG];
    int id;
    auto fetch = [&](int number) {
        id = number;
        const unsigned char* from = cache + (size_t)max(number, 0) * block_bytes(D);       // (a block that is not there: any other, cleared below)
        const uint32_t* kc = reinterpret_cast<const uint32_t*>(from) + ((key_in & 15) * 4 + quarter) * NG;
        const uint16_t* kw = reinterpret_cast<const uint16_t*>(from + key_words_at(D)) + (key_in & 15) * NG;
        const uint32_t* vc = reinterpret_cast<const uint32_t*>(from + value_codes_at(D)) + (tid & 63) * NG;
        const uint32_t* vw = reinterpret_cast<const uint32_t*>(from + value_words_at(D)) + (half * 4 + pair) * NG;
#pragma unroll
        for (int k = 0; k < NG; ++k) key_code[k] = kc[k], key_word[k] = kw[k], value_code[k] = vc[k], value_word[k] = vw[k];
    };
    auto put = [&](int j) {
        if ((tid & 63) == 0) s_named[block] = id >= 0;
        const int token = 16 * block + 8 * half + 2 * pair, key = k0 + j * kKeys + token;
        const uint32_t keep = id < 0 ? 0u : (key < seq_len ? 0xffffu : 0u) | (key + 1 < seq_len ? 0xffff0000u : 0u);
#pragma unroll
        for (int k = 0; k < NG; ++k) {
            const uint32_t w = __byte_perm(key_word[k], 0, 0x1010), zero = mul_bf16x2(w & 0x000f000fu, kMinus2p127), step = mul_bf16x2(w & 0xfff0fff0u, k64);
            const uint32_t lo = key_code[k], hi = lo >> 8;
            uint4 v;
            v.x = mul_bf16x2(fma_bf16x2(lo & 0x000f000fu, k2p127, zero), step);
            v.y = mul_bf16x2(fma_bf16x2(lo & 0x00f000f0u, k2p123, zero), step);
            v.z = mul_bf16x2(fma_bf16x2(hi & 0x000f000fu, k2p127, zero), step);
            v.w = mul_bf16x2(fma_bf16x2(hi & 0x00f000f0u, k2p123, zero), step);
            *reinterpret_cast<uint4*>(sK + key_in * P + kGroup * k + 8 * quarter) = v;
        }
#pragma unroll
        for (int k = 0; k < NG; ++k) {
            uint32_t w = value_word[k] & keep;
            const uint32_t odd = ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u;          // a sign bit is set where a word is not a number
            if (odd) {
                s_odd = 1;
                w &= (odd & 0x8000u ? 0u : 0xffffu) | (odd & 0x80000000u ? 0u : 0xffff0000u);
            }
            const uint32_t zero = mul_bf16x2(w & 0x000f000fu, kMinus2p127), step = mul_bf16x2(w & 0xfff0fff0u, k64);
            const uint32_t lo = value_code[k], hi = lo >> 8;
            uint32_t* dst = reinterpret_cast<uint32_t*>(sV + (kGroup * k + 4 * eighth) * kVPitch + token);
            dst[0] = mul_bf16x2(fma_bf16x2(lo & 0x000f000fu, k2p127, zero), step);
            dst[kVPitch / 2] = mul_bf16x2(fma_bf16x2(lo & 0x00f000f0u, k2p123, zero), step);
            dst[kVPitch] = mul_bf16x2(fma_bf16x2(hi & 0x000f000fu, k2p127, zero), step);
            dst[kVPitch / 2 * 3] = mul_bf16x2(fma_bf16x2(hi & 0x00f000f0u, k2p123, zero), step);
        }
    };
    int id_next = lookup(0);
    if (tiles > 0) fetch(id_next);
    id_next = lookup(1);

    for (int i = tid; i < kRows * (D / 8); i += kWarps * 32) {
        const int row = i / (D / 8), x = (i - row * (D / 8)) * 8, grow = row0 + row;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (grow < rows_total) v = *reinterpret_cast<const uint4*>(q + (size_t)(q0 + grow / g) * q_stride + (size_t)(kvh * g + grow % g) * D + x);
        *reinterpret_cast<uint4*>(sQ + row * P + x) = v;
    }

    // ---- a lane's rows `lane / 4` and eight further of the warp's 16; of a tile's keys 8 t + 2 quad and the one after ----
    const int quad = lane & 3, row_a = 16 * warp + (lane >> 2);
    const bool live = row0 + 16 * warp < rows_total;
    int pos[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) pos[h] = row0 + row_a + 8 * h < rows_total ? seq_len - n + (row0 + row_a + 8 * h) / g : -1;
    const int warp_first = seq_len - n + (row0 + 16 * warp) / g, warp_last = seq_len - n + (min(row0 + 16 * warp + 16, rows_total) - 1) / g;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, acc[4 * NG][4];
#pragma unroll
    for (int i = 0; i < 4 * NG; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    const __nv_bfloat16* qa = sQ + (16 * warp + (lane & 15)) * P + (lane >> 4) * 8;
    const __nv_bfloat16* kb = sK + (lane & 7) * P + (lane >> 3) * 8;
    const __nv_bfloat16* vb = sV + (lane & 7) * kVPitch + (lane >> 3) * 8;

    for (int j = 0; j < tiles; ++j) {
        __syncthreads();                                         // the tile before has been read
        put(j);
        __syncthreads();
        if (j + 1 < tiles) {
            fetch(id_next);
            id_next = lookup(j + 2);
        }
        if (!live) continue;
        const int key0 = k0 + j * kKeys;
        float s[4][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
#pragma unroll
        for (int k = 0; k < NG; ++k) {
            uint32_t a0[4], a1[4];
            load_tiles(a0, qa + kGroup * k);
            load_tiles(a1, qa + kGroup * k + 16);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                uint32_t b[4];
                load_tiles(b, kb + 8 * t * P + kGroup * k);
                mma(s[t], a0, b[0], b[1]);
                mma(s[t], a1, b[2], b[3]);
            }
        }
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[t][e] *= scale_log2;
        const bool whole = s_named[0] && s_named[1] && key0 + kKeys - 1 <= warp_first && (window <= 0 || key0 > warp_last - window);
        if (!whole) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int key = key0 + 8 * t + 2 * quad + (e & 1), p = pos[e >> 1];
                    if (!(s_named[t >> 1] && key <= p && (window <= 0 || key > p - window))) s[t][e] = -INFINITY;
                }
        }
        float corr[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float x = -INFINITY;
#pragma unroll
            for (int t = 0; t < 4; ++t) x = fmaxf(x, fmaxf(s[t][2 * h], s[t][2 * h + 1]));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
            const float top = fmaxf(m[h], x), base = top == -INFINITY ? 0.f : top;
            corr[h] = top == m[h] ? 1.f : ex2(m[h] - base);
            m[h] = top;
            l[h] *= corr[h];
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    s[t][2 * h + e] = ex2(s[t][2 * h + e] - base);
                    l[h] += s[t][2 * h + e];
                }
        }
        if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
            for (int i = 0; i < 4 * NG; ++i) acc[i][0] *= corr[0], acc[i][1] *= corr[0], acc[i][2] *= corr[1], acc[i][3] *= corr[1];
        }
        uint32_t p[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            p[h][0] = pack_bf16(s[2 * h][0], s[2 * h][1]), p[h][1] = pack_bf16(s[2 * h][2], s[2 * h][3]);
            p[h][2] = pack_bf16(s[2 * h + 1][0], s[2 * h + 1][1]), p[h][3] = pack_bf16(s[2 * h + 1][2], s[2 * h + 1][3]);
        }
#pragma unroll
        for (int i = 0; i < 4 * NG; ++i) {
            uint32_t b[4];
            load_tiles(b, vb + 8 * i * kVPitch);
            mma(acc[i], p[0], b[0], b[1]);
            mma(acc[i], p[1], b[2], b[3]);
        }
    }
    __syncthreads();                                             // the last tile has been read, and `s_odd` written
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
    const bool alone = gridDim.x == 1;
    float f[2];
    unsigned bad[2] = {0, 0};                                    // groups whose sum holds a value that is not a number
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        f[h] = !alone ? 1.f : l[h] == 0.f ? 0.f : 1.f / l[h];
        if (s_odd) {
            for (int key = window > 0 ? max(0, pos[h] - window + 1) : 0; key <= pos[h] && key / page_size < table_cols; ++key) {
                const int page = table[key / page_size];
                if (page < 0 || page >= num_pages) continue;
                const unsigned char* at = cache + ((size_t)(page * nkv + kvh) * per_page + key % page_size / kBlock) * block_bytes(D);
                const uint16_t* words = reinterpret_cast<const uint16_t*>(at + value_words_at(D)) + ((key % kBlock) >> 1) * NG * 2 + (key & 1);
                for (int k = 0; k < NG; ++k)
                    if ((words[2 * k] & 0x7f80u) == 0x7f80u) bad[h] |= 1u << k;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4 * NG; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = row_a + 8 * h, grow = row0 + row, x = 8 * i + 2 * quad;
            const float ff = (bad[h] >> (i >> 2)) & 1u ? NAN : f[h];
            const float a = acc[i][2 * h] * ff, b = acc[i][2 * h + 1] * ff;
            if (!alone) part[row * F + x] = a, part[row * F + x + 1] = b;
            else if (grow < rows_total) {
                __nv_bfloat16* dst = out + (size_t)(q0 + grow / g) * out_stride + (size_t)(kvh * g + grow % g) * D + x;
                dst[0] = __float2bfloat16_rn(a), dst[1] = __float2bfloat16_rn(b);
            }
        }
    if (alone) return;
    if (quad == 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) part_ml[(row_a + 8 * h) * 2] = m[h], part_ml[(row_a + 8 * h) * 2 + 1] = l[h];
    }
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();                                              // every CTA's part is in its shared memory
    const int rows = min(kRows, rows_total - row0);
    for (int i = (int)blockIdx.x * kWarps * 32 + tid; i < rows * D; i += (int)gridDim.x * kWarps * 32) {
        const int row = i / D, x = i - row * D, grow = row0 + row;
        float top[kCluster], M = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
        for (int c = 0; c < kCluster; ++c) {
            top[c] = c < (int)gridDim.x ? cluster.map_shared_rank(part_ml, c)[row * 2] : -INFINITY;
            M = fmaxf(M, top[c]);
        }
#pragma unroll
        for (int c = 0; c < kCluster; ++c) {
            if (c >= (int)gridDim.x) break;
            const float w = top[c] == -INFINITY ? 0.f : ex2(top[c] - M);
            L += cluster.map_shared_rank(part_ml, c)[row * 2 + 1] * w;
            O += cluster.map_shared_rank(part, c)[row * F + x] * w;
        }
        out[(size_t)(q0 + grow / g) * out_stride + (size_t)(kvh * g + grow % g) * D + x] = __float2bfloat16_rn(L == 0.f ? 0.f : O / L);
    }
    cluster.sync();                                              // (a CTA's shared memory has been read before it leaves)
}

template <int NG>
static int launch(cudaStream_t stream, bool use_pdl, int cluster, int tiles, const __nv_bfloat16* q, int q_stride, __nv_bfloat16* out, int out_stride,
                  const unsigned char* cache, int num_pages, int page_size, const int* block_table, int table_stride, int table_cols, const int* query_start_loc,
                  const int* seq_lens, int num_requests, int least_query, int nq, int nkv, float scale, int window) {
    static SmemLimit limit;
    if (int rc = raise_smem_limit(limit, attention_rows_mma_kernel<NG>, Sizes<NG>::kBytes, "attention_kv4_rows_mma")) return rc;
    const cudaError_t e = launch_pdl_cluster(attention_rows_mma_kernel<NG>, dim3(cluster, tiles, nkv), dim3(kWarps * 32), (size_t)Sizes<NG>::kBytes, stream, use_pdl, cluster,
                                             q, q_stride, out, out_stride, cache, num_pages, page_size, block_table, table_stride, table_cols, query_start_loc,
                                             seq_lens, num_requests, least_query, nq, nkv, scale * 1.4426950408889634f, window);
    CIB_REQUIRE(e == cudaSuccess, "attention_kv4_rows_mma: launch failed: %s", cudaGetErrorString(e));
    return 0;
}

}  // namespace kv4m
}  // namespace cib

using namespace cib;

// num_tiles = sum over requests of ceil(tokens_r * (nq / nkv) / 64), or more: CTAs that find none leave.  cluster: so many CTAs (1, 2, 4 or 8) share
// the keys of a tile.  least_query: requests that bring fewer tokens are left as they are.
extern "C" int cib_attention_kv4_rows_mma(const void* q, int q_stride, void* out, int out_stride, const void* cache, int num_pages, int page_size,
                                          const int* block_table, int table_stride, int table_cols, const int* query_start_loc, const int* seq_lens,
                                          int num_requests, int num_tiles, int cluster, int least_query, int nq, int nkv, int d, float scale, int window, int use_pdl,
                                          cudaStream_t stream) {
    CIB_REQUIRE(kv4::sizes_ok(d, page_size), "attention_kv4_rows_mma: head size %d must be a multiple of 32 up to 256, page size %d a multiple of 16", d, page_size);
    CIB_REQUIRE(num_requests >= 0 && nq > 0 && nkv > 0 && nq % nkv == 0 && nkv <= 65535, "attention_kv4_rows_mma: bad sizes R=%d nq=%d nkv=%d", num_requests, nq, nkv);
    CIB_REQUIRE(num_tiles >= 0 && num_tiles <= 65535, "attention_kv4_rows_mma: %d row tiles are too many", num_tiles);
    CIB_REQUIRE(cluster == 1 || cluster == 2 || cluster == 4 || cluster == kv4m::kCluster, "attention_kv4_rows_mma: clusters of 1, 2, 4 or 8, not %d", cluster);
    CIB_REQUIRE(num_pages > 0 && table_stride > 0 && table_cols > 0 && cache != nullptr && ((uintptr_t)cache % 16) == 0, "attention_kv4_rows_mma: bad cache geometry");
    CIB_REQUIRE((long long)num_pages * nkv * (page_size / kv4::kBlock) < (1ll << 31), "attention_kv4_rows_mma: more than 2^31 blocks");
    CIB_REQUIRE(q_stride >= nq * d && out_stride >= nq * d, "attention_kv4_rows_mma: row strides %d and %d are too small", q_stride, out_stride);
    CIB_REQUIRE(q_stride % 8 == 0 && ((uintptr_t)q % 16) == 0, "attention_kv4_rows_mma: query rows must be 16-byte aligned");
    CIB_REQUIRE(window >= 0, "attention_kv4_rows_mma: window must be >= 0 (0 = all keys)");
    if (num_requests == 0 || num_tiles == 0) return 0;
#define CIB_KV4_ROWS(NGV)                                                                                                                                    \
    if (d == 32 * NGV)                                                                                                                                       \
        return kv4m::launch<NGV>(stream, use_pdl != 0, cluster, num_tiles, (const __nv_bfloat16*)q, q_stride, (__nv_bfloat16*)out, out_stride,                  \
                                 (const unsigned char*)cache, num_pages, page_size, block_table, table_stride, table_cols, query_start_loc, seq_lens,           \
                                 num_requests, least_query, nq, nkv, scale, window)
    CIB_KV4_ROWS(1);
    CIB_KV4_ROWS(2);
    CIB_KV4_ROWS(3);
    CIB_KV4_ROWS(4);
    CIB_KV4_ROWS(5);
    CIB_KV4_ROWS(6);
    CIB_KV4_ROWS(7);
    CIB_KV4_ROWS(8);
#undef CIB_KV4_ROWS
    return -1;
}
