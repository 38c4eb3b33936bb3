// Prompt attention over the cache that is held in 4 bits (kv4.cuh) without tensor cores: any head size that is a multiple of 32 up to 256, any head
// counts, 32-bit queries, and bfloat16 ones whose rows are not 16-byte aligned.
//
//   out = softmax(scale * q K^T over the keys position - window < j <= position) V,  32-bit multiply-adds throughout, the exact exponential
//
// A CTA has 64 rows (query token x query head of one kv head) of one request and walks tiles of 32 keys: half of its threads take the tile's keys
// apart and half its values, into shared memory as 32-bit numbers, from words that were asked for a tile ahead, so a code is taken apart once for
// 64 rows (a token at a time, four heads for a code, a prompt of 400 tokens, 16 heads over 8 of 128, took 263 us, 90 so).  A warp has eight rows: a lane
// computes the scores of four of them with two keys (32 multiply-adds, two to an instruction, for 6 loads of 16 bytes), the warp takes the exponentials of its own
// scores and passes them to itself as the weights of the sum of the values, of which a lane has every 32nd column: 8 D / 32 sums in registers.  Nothing
// but the tile is exchanged between warps.  Bound by latency: with 8 heads of 256 issue slots are 0.39 busy, the multiply-add pipe 0.25 and shared memory 0.39
// (two warps a scheduler; their registers hold the sums).
//
// Where a launch would leave SMs without work, a cluster of up to eight CTAs shares the key tiles of 64 rows; the partial results are joined through
// distributed shared memory.
//
// Keys whose page the block table does not name are left out; a row without keys is zero.  Values of keys that a row does not see are not
// multiplied at all (0 x NaN is NaN): which rows see a key is the same for all lanes, and only tiles that not every row sees whole ask.
#include "kv4.cuh"
#include "mma_utils.cuh"

#include <cooperative_groups.h>

namespace cib {
namespace kv4r {

using namespace kv4;

// two 32-bit multiply-adds at a time; {a, b} of two neighbouring registers
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 both(uint64_t a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

constexpr int kRows = 64, kKeys = 32, kWarps = 8, kCluster = 8;

template <int NG>
struct Sizes {
    static constexpr int D = kGroup * NG, P = D + 4;             // (rows of shared memory four numbers apart: no two of eight 16-byte accesses meet in a bank)
    static constexpr int kFloats = (kRows + 2 * kKeys) * P + kWarps * kKeys * 8 + 2 * kRows;
};

template <int NG>
__global__ void __launch_bounds__(kWarps * 32, NG <= 4 ? 2 : 1)
attention_rows_kernel(const void* __restrict__ q, int bf16, int q_stride, void* __restrict__ out, int out_stride, const unsigned char* __restrict__ cache, int num_pages,
                      int page_size, const int* __restrict__ block_table, int table_stride, int table_cols, const int* __restrict__ query_start_loc,
                      const int* __restrict__ seq_lens, int num_requests, int least_query, int nq, int nkv, float scale, int window) {
    constexpr int D = Sizes<NG>::D, P = Sizes<NG>::P;
    extern __shared__ __align__(16) float smem_f[];
    float* sQ = smem_f;                                          // [row][D], scaled; at the end a CTA's partial result
    float* sK = sQ + kRows * P;
    float* sV = sK + kKeys * P;
    float* sP = sV + kKeys * P;                                  // [warp][key][8 rows]
    float* sML = sP + kWarps * kKeys * 8;                        // [row][maximum, sum]
    __shared__ int s_req, s_tile, s_named[2];
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
        if (lane == 0) s_req = req, s_tile = tile;
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

    // ---- this thread's words of a tile ----
    const bool takes_keys = tid < 128;
    const int u = tid & 127;
    const int block = u >> 6;                                    // keys: (key, quarter); values: (half, eighth, pair) of a block
    const int key_in = u >> 2, quarter = u & 3;
    const int pair = u & 3, eighth = (u >> 2) & 7, half = (u >> 5) & 1;
    const int per_page = page_size / kBlock;
    const int* table = block_table + (size_t)r * table_stride;
    auto lookup = [&](int j) {
        const int b = k0 / kBlock + 2 * j + block, index = b / per_page;
        if (j >= tiles || b * kBlock >= seq_len || index >= table_cols) return -1;
        const int page = table[index];
        return page >= 0 && page < num_pages ? (page * nkv + kvh) * per_page + (b - index * per_page) : -1;
    };
    uint32_t code[NG], word[NG];
    int id;
    auto fetch = [&](int number) {
        id = number;
        const unsigned char* from = cache + (size_t)max(number, 0) * block_bytes(D);       // (a block that is not there: any other, cleared below)
        if (takes_keys) {
            const uint32_t* c = reinterpret_cast<const uint32_t*>(from) + ((key_in & 15) * 4 + quarter) * NG;
            const uint16_t* w = reinterpret_cast<const uint16_t*>(from + key_words_at(D)) + (key_in & 15) * NG;
#pragma unroll
            for (int k = 0; k < NG; ++k) code[k] = c[k], word[k] = w[k];
        } else {
            const uint32_t* c = reinterpret_cast<const uint32_t*>(from + value_codes_at(D)) + (u & 63) * NG;
            const uint32_t* w = reinterpret_cast<const uint32_t*>(from + value_words_at(D)) + (half * 4 + pair) * NG;
#pragma unroll
            for (int k = 0; k < NG; ++k) code[k] = c[k], word[k] = w[k];
        }
    };
    // step * (code - zero): the code under the exponent of 2^23, less 2^23 + zero, is exact
    auto number = [](uint32_t code4, float minus, float step) { return (__uint_as_float(0x4b000000u | code4) - minus) * step; };
    auto put = [&](int j) {
        if (takes_keys) {
            if ((u & 63) == 0) s_named[block] = id >= 0;
            float* dst = sK + key_in * P + 8 * quarter;
#pragma unroll
            for (int k = 0; k < NG; ++k) {
                const uint32_t c = code[k], w = id < 0 ? 0u : word[k];
                const float minus = 8388608.f + (float)(w & 15u), step = step_of(w);
                *reinterpret_cast<float4*>(dst + kGroup * k) = make_float4(number(c & 15u, minus, step), number((c >> 16) & 15u, minus, step),
                                                                           number((c >> 4) & 15u, minus, step), number((c >> 20) & 15u, minus, step));
                *reinterpret_cast<float4*>(dst + kGroup * k + 4) = make_float4(number((c >> 8) & 15u, minus, step), number((c >> 24) & 15u, minus, step),
                                                                               number((c >> 12) & 15u, minus, step), number(c >> 28, minus, step));
            }
        } else {
            const int token = 16 * block + 8 * half + 2 * pair, key = k0 + j * kKeys + token;
            const uint32_t keep = id < 0 ? 0u : (key < seq_len ? 0xffffu : 0u) | (key + 1 < seq_len ? 0xffff0000u : 0u);
            float* dst = sV + token * P + 4 * eighth;
#pragma unroll
            for (int k = 0; k < NG; ++k) {
                const uint32_t w = word[k] & keep;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const uint32_t c = code[k] >> (16 * t), wt = w >> (16 * t);
                    const float minus = 8388608.f + (float)(wt & 15u), step = step_of(wt);
                    *reinterpret_cast<float4*>(dst + t * P + kGroup * k) =
                        make_float4(number(c & 15u, minus, step), number((c >> 4) & 15u, minus, step), number((c >> 8) & 15u, minus, step), number((c >> 12) & 15u, minus, step));
                }
            }
        }
    };
    int id_next = lookup(0);
    if (tiles > 0) fetch(id_next);
    id_next = lookup(1);

    for (int i = tid; i < kRows * D; i += kWarps * 32) {
        const int row = i / D, x = i - row * D, grow = row0 + row;
        float v = 0.f;
        if (grow < rows_total) {
            const size_t at = (size_t)(q0 + grow / g) * q_stride + (size_t)(kvh * g + grow % g) * D + x;
            v = (bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(q)[at]) : reinterpret_cast<const float*>(q)[at]) * scale;
        }
        sQ[row * P + x] = v;
    }

    // ---- a lane's four rows and two keys of the scores ----
    const int rg = lane >> 4, ki = lane & 15;
    const bool live = row0 + 8 * warp < rows_total;
    int pos[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int grow = row0 + 8 * warp + 4 * rg + i;
        pos[i] = grow < rows_total ? seq_len - n + grow / g : -1;
    }
    const int warp_first = seq_len - n + (row0 + 8 * warp) / g, warp_last = row0 + 8 * warp + 7 < rows_total ? seq_len - n + (row0 + 8 * warp + 7) / g : 0x7fffffff;
    float m[4], l[4];
    uint64_t acc[4][NG];                                         // rows 2 i and 2 i + 1
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < NG; ++k) acc[i][k] = 0;
    const float* qr = sQ + (8 * warp + 4 * rg) * P;
    const float* kr = sK + ki * P;
    float* pw = sP + warp * kKeys * 8;

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
        uint64_t sums[4][2] = {};                                // of even and odd columns
#pragma unroll 4
        for (int c = 0; c < D; c += 4) {
            const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(kr + c), b = *reinterpret_cast<const ulonglong2*>(kr + 16 * P + c);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(qr + i * P + c);
                sums[i][0] = fma2(x.y, a.y, fma2(x.x, a.x, sums[i][0]));
                sums[i][1] = fma2(x.y, b.y, fma2(x.x, b.x, sums[i][1]));
            }
        }
        float s[4][2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 a = both(sums[i][0]), b = both(sums[i][1]);
            s[i][0] = a.x + a.y, s[i][1] = b.x + b.y;
        }
        const bool whole = s_named[0] && s_named[1] && key0 + kKeys - 1 <= warp_first && (window <= 0 || (warp_last != 0x7fffffff && key0 > warp_last - window));
        uint32_t seen = 0xffu;                                   // of key `lane`: which of the warp's eight rows see it
        if (!whole) {
            seen = 0;
            const bool named = s_named[lane >> 4] != 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int p = __shfl_sync(0xffffffffu, pos[i & 3], (i >> 2) * 16), key = key0 + lane;
                if (named && key <= p && (window <= 0 || key > p - window)) seen |= 1u << i;
            }
            const uint32_t first = __shfl_sync(0xffffffffu, seen, ki) >> (4 * rg), second = __shfl_sync(0xffffffffu, seen, ki + 16) >> (4 * rg);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (!((first >> i) & 1u)) s[i][0] = -INFINITY;
                if (!((second >> i) & 1u)) s[i][1] = -INFINITY;
            }
        }
        float corr[4];
        bool changes = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float x = fmaxf(s[i][0], s[i][1]);
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
            const float top = fmaxf(m[i], x), base = top == -INFINITY ? 0.f : top;
            corr[i] = top == m[i] ? 1.f : expf(m[i] - base);
            changes = changes || top != m[i];
            m[i] = top;
            s[i][0] = expf(s[i][0] - base), s[i][1] = expf(s[i][1] - base);
            l[i] = l[i] * corr[i] + s[i][0] + s[i][1];
        }
        if (__any_sync(0xffffffffu, changes)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int from = (i >> 1) * 16;
                const uint64_t f = pair_of(__shfl_sync(0xffffffffu, corr[2 * (i & 1)], from), __shfl_sync(0xffffffffu, corr[2 * (i & 1) + 1], from));
#pragma unroll
                for (int k = 0; k < NG; ++k) acc[i][k] = mul2(acc[i][k], f);
            }
        }
        *reinterpret_cast<float4*>(pw + ki * 8 + 4 * rg) = make_float4(s[0][0], s[1][0], s[2][0], s[3][0]);
        *reinterpret_cast<float4*>(pw + (ki + 16) * 8 + 4 * rg) = make_float4(s[0][1], s[1][1], s[2][1], s[3][1]);
        __syncwarp();
        if (whole) {
#pragma unroll 4
            for (int x = 0; x < kKeys; ++x) {
                const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(pw + x * 8), b = *reinterpret_cast<const ulonglong2*>(pw + x * 8 + 4);
#pragma unroll
                for (int k = 0; k < NG; ++k) {
                    const float v = sV[x * P + kGroup * k + lane];
                    const uint64_t vv = pair_of(v, v);
                    acc[0][k] = fma2(a.x, vv, acc[0][k]);
                    acc[1][k] = fma2(a.y, vv, acc[1][k]);
                    acc[2][k] = fma2(b.x, vv, acc[2][k]);
                    acc[3][k] = fma2(b.y, vv, acc[3][k]);
                }
            }
        } else {
            for (int x = 0; x < kKeys; ++x) {
                const uint32_t rows = __shfl_sync(0xffffffffu, seen, x);
                if (rows == 0) continue;
                const float4 a = *reinterpret_cast<const float4*>(pw + x * 8), b = *reinterpret_cast<const float4*>(pw + x * 8 + 4);
                const float p[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
                for (int k = 0; k < NG; ++k) {
                    const float v = sV[x * P + kGroup * k + lane];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 o = both(acc[i][k]);
                        acc[i][k] = pair_of((rows >> (2 * i)) & 1u ? fmaf(p[2 * i], v, o.x) : o.x, (rows >> (2 * i + 1)) & 1u ? fmaf(p[2 * i + 1], v, o.y) : o.y);
                    }
                }
            }
        }
        __syncwarp();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
    auto store = [&](int row, int x, float sum, float value) {
        const int grow = row0 + row;
        const size_t at = (size_t)(q0 + grow / g) * out_stride + (size_t)(kvh * g + grow % g) * D + x;
        // (a sum that is not a number stays one: only a row without keys is zero)
        const float o = sum == 0.f ? 0.f : value / sum;
        if (bf16) reinterpret_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(o);
        else reinterpret_cast<float*>(out)[at] = o;
    };
    if (gridDim.x == 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float sum = __shfl_sync(0xffffffffu, l[i & 3], (i >> 2) * 16);
            if (row0 + 8 * warp + i < rows_total) {
#pragma unroll
                for (int k = 0; k < NG; ++k) store(8 * warp + i, kGroup * k + lane, sum, i & 1 ? both(acc[i >> 1][k]).y : both(acc[i >> 1][k]).x);
            }
        }
        return;
    }
    __syncwarp();                                                // (a warp reads its own rows of the queries only: they may go)
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int k = 0; k < NG; ++k) sQ[(8 * warp + i) * P + kGroup * k + lane] = i & 1 ? both(acc[i >> 1][k]).y : both(acc[i >> 1][k]).x;
    if (ki == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sML[(8 * warp + 4 * rg + i) * 2] = m[i], sML[(8 * warp + 4 * rg + i) * 2 + 1] = l[i];
    }
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();                                              // every CTA's part is in its shared memory
    const int rows = min(kRows, rows_total - row0);
    for (int i = (int)blockIdx.x * kWarps * 32 + tid; i < rows * D; i += (int)gridDim.x * kWarps * 32) {
        const int row = i / D, x = i - row * D;
        float top[kCluster], M = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
        for (int c = 0; c < kCluster; ++c) {
            top[c] = c < (int)gridDim.x ? cluster.map_shared_rank(sML, c)[row * 2] : -INFINITY;
            M = fmaxf(M, top[c]);
        }
#pragma unroll
        for (int c = 0; c < kCluster; ++c) {
            if (c >= (int)gridDim.x) break;
            const float f = top[c] == -INFINITY ? 0.f : expf(top[c] - M);
            L += cluster.map_shared_rank(sML, c)[row * 2 + 1] * f;
            O += cluster.map_shared_rank(sQ, c)[row * P + x] * f;
        }
        store(row, x, L, O);
    }
    cluster.sync();                                              // (a CTA's shared memory has been read before it leaves)
}

template <int NG>
static int launch(cudaStream_t stream, bool use_pdl, int cluster, int tiles, const void* q, int bf16, int q_stride, void* out, int out_stride, const unsigned char* cache,
                  int num_pages, int page_size, const int* block_table, int table_stride, int table_cols, const int* query_start_loc, const int* seq_lens,
                  int num_requests, int least_query, int nq, int nkv, float scale, int window) {
    static SmemLimit limit;
    constexpr size_t bytes = Sizes<NG>::kFloats * sizeof(float);
    if (int rc = raise_smem_limit(limit, attention_rows_kernel<NG>, (int)bytes, "attention_kv4_rows")) return rc;
    const cudaError_t e = launch_pdl_cluster(attention_rows_kernel<NG>, dim3(cluster, tiles, nkv), dim3(kWarps * 32), bytes, stream, use_pdl, cluster, q, bf16, q_stride, out,
                                             out_stride, cache, num_pages, page_size, block_table, table_stride, table_cols, query_start_loc, seq_lens,
                                             num_requests, least_query, nq, nkv, scale, window);
    CIB_REQUIRE(e == cudaSuccess, "attention_kv4_rows: launch failed: %s", cudaGetErrorString(e));
    return 0;
}

}  // namespace kv4r
}  // namespace cib

using namespace cib;

// How many CTAs of the kernel an SM holds.
extern "C" int cib_attention_kv4_rows_ctas(int d) { return d <= 128 ? 2 : 1; }

// num_tiles = sum over requests of ceil(tokens_r * (nq / nkv) / 64), or more: CTAs that find none leave.  cluster: so many CTAs (1, 2, 4 or 8) share
// the keys of a tile.  least_query: requests that bring fewer tokens are left as they are.
extern "C" int cib_attention_kv4_rows(const void* q, int dtype, int q_stride, void* out, int out_stride, const void* cache, int num_pages, int page_size,
                                      const int* block_table, int table_stride, int table_cols, const int* query_start_loc, const int* seq_lens, int num_requests,
                                      int num_tiles, int cluster, int least_query, int nq, int nkv, int d, float scale, int window, int use_pdl, cudaStream_t stream) {
    CIB_REQUIRE(kv4::sizes_ok(d, page_size), "attention_kv4_rows: head size %d must be a multiple of 32 up to 256, page size %d a multiple of 16", d, page_size);
    CIB_REQUIRE(num_requests >= 0 && nq > 0 && nkv > 0 && nq % nkv == 0 && nkv <= 65535, "attention_kv4_rows: bad sizes R=%d nq=%d nkv=%d", num_requests, nq, nkv);
    CIB_REQUIRE(num_tiles >= 0 && num_tiles <= 65535, "attention_kv4_rows: %d row tiles are too many", num_tiles);
    CIB_REQUIRE(cluster == 1 || cluster == 2 || cluster == 4 || cluster == kv4r::kCluster, "attention_kv4_rows: clusters of 1, 2, 4 or 8, not %d", cluster);
    CIB_REQUIRE(num_pages > 0 && table_stride > 0 && table_cols > 0 && cache != nullptr && ((uintptr_t)cache % 16) == 0, "attention_kv4_rows: bad cache geometry");
    CIB_REQUIRE((long long)num_pages * nkv * (page_size / kv4::kBlock) < (1ll << 31), "attention_kv4_rows: more than 2^31 blocks");
    CIB_REQUIRE(q_stride >= nq * d && out_stride >= nq * d, "attention_kv4_rows: row strides %d and %d are too small", q_stride, out_stride);
    CIB_REQUIRE(window >= 0, "attention_kv4_rows: window must be >= 0 (0 = all keys)");
    CIB_REQUIRE(dtype == kF32 || dtype == kBF16, "attention_kv4_rows: unsupported dtype %d", dtype);
    if (num_requests == 0 || num_tiles == 0) return 0;
#define CIB_KV4_ROWS(NGV)                                                                                                                                    \
    if (d == 32 * NGV)                                                                                                                                       \
        return kv4r::launch<NGV>(stream, use_pdl != 0, cluster, num_tiles, q, dtype == kBF16 ? 1 : 0, q_stride, out, out_stride, (const unsigned char*)cache,      \
                                 num_pages, page_size, block_table, table_stride, table_cols, query_start_loc, seq_lens, num_requests, least_query, nq, nkv, scale, window)
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
