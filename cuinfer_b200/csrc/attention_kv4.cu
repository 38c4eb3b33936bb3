// Paged causal attention of single tokens over the cache that is held in 4 bits (kv4.cuh), the all-sizes kernel: any head size that is a
// multiple of 32 up to 256, any head counts, 32-bit or bfloat16 queries, an optional window.  (It takes several tokens of a request too, a token at a
// time; attention_kv4_rows.cu shares the keys among them.)
//
//   out = softmax(scale * q K^T over the keys position - window < j <= position) V
//
// The queries of a request are the last n positions of its sequence.  A CTA takes one token and up to four query heads of one kv
// head (a key is taken apart once for all four); its warps share the keys in chunks of 32, a key to a lane for the scores, a value
// column to a lane for the weighted sum, and merge their running maxima and sums in shared memory.  Where that leaves SMs without work, a
// cluster of up to eight CTAs shares the keys and joins its parts through distributed shared memory: one token of 4 000 keys, 16 heads over 8 of
// 128, takes 31 us (45 with conversions of integers and a value at a time, 270 without clusters), 64 of them 424, most of it taking every code apart for
// two heads.  32-bit throughout,
// the exact exponential; nothing is rounded before the end.  Keys whose page the block table does not name are left out; a row
// without keys is zero; rows that belong to no request are left as they are.
#include "kv4.cuh"
#include "mma_utils.cuh"

#include <cooperative_groups.h>

namespace cib {
namespace kv4 {

constexpr int kHeads = 4;
constexpr int kMaxWarps = 8;
constexpr int kMaxCluster = 8;

template <int N>
struct alignas(N * 4) Words {
    uint32_t w[N];
};
// code - zero (the lowest four bits of `x`): under the exponent of 2^23, less 2^23 + zero, it is exact
__device__ __forceinline__ float less(uint32_t x, float minus) { return __uint_as_float(0x4b000000u | (x & 15u)) - minus; }

template <typename T, int NG>
__global__ void __launch_bounds__(kMaxWarps * 32)
attention_generic_kernel(const T* __restrict__ q, int q_stride, T* __restrict__ out, int out_stride, unsigned char* __restrict__ cache, int num_pages,
                         int page_size, const int* __restrict__ block_table, int table_stride, int table_cols, const int* __restrict__ query_start_loc,
                         const int* __restrict__ seq_lens, int num_requests, int nq, int nkv, float scale, int window, int cluster) {
    constexpr int d = kGroup * NG;
    extern __shared__ __align__(16) float smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int t = blockIdx.x / cluster, rank = blockIdx.x - t * cluster, kvh = blockIdx.y;
    const int g = nq / nkv;
    const int head0 = kvh * g + blockIdx.z * kHeads;
    const int nh = min(kHeads, (kvh + 1) * g - head0);
    griddep_wait();
    griddep_launch();
    // the request of this row: the last one that starts at or before it
    int before = 0;
    for (int r0 = 0; r0 <= num_requests; r0 += 32) {
        const int r = r0 + lane;
        before += __popc(__ballot_sync(0xffffffffu, r <= num_requests && query_start_loc[min(r, num_requests)] <= t));
    }
    const int r = before - 1;
    if (r < 0 || r >= num_requests) return;
    const int q0 = query_start_loc[r], n = query_start_loc[r + 1] - q0;
    const int pos = seq_lens[r] - n + (t - q0);
    const int lo = window > 0 ? max(0, pos - window + 1) : 0;
    const int* table = block_table + (size_t)r * table_stride;

    float* qs = smem;                                      // [head][d], scaled
    for (int i = threadIdx.x; i < nh * d; i += blockDim.x) qs[i] = to_f32(q[(size_t)t * q_stride + (size_t)head0 * d + i]) * scale;
    __syncthreads();

    float acc[kHeads][NG];
    float m[kHeads], l[kHeads];
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
        m[h] = -INFINITY, l[h] = 0.f;
#pragma unroll
        for (int k = 0; k < NG; ++k) acc[h][k] = 0.f;
    }
    constexpr int V = NG % 4 == 0 ? 4 : NG % 2 == 0 ? 2 : 1;     // words of a load
    for (int c = lo / 32 * 32 + (rank * warps + warp) * 32; c <= pos; c += cluster * warps * 32) {
        const int j = c + lane;                            // lanes 0-15 have a block's keys, 16-31 the next one's
        const unsigned char* block = nullptr;
        if (c + (lane & 16) <= pos && (c + (lane & 16)) / page_size < table_cols) {
            const int page = table[(c + (lane & 16)) / page_size];
            if (page >= 0 && page < num_pages) block = block_of(cache, page * page_size + (c + (lane & 16)) % page_size, num_pages, page_size, nkv, kvh, d);
        }
        const bool seen = block != nullptr && j >= lo && j <= pos;
        float s[kHeads] = {0.f, 0.f, 0.f, 0.f};
        if (seen) {
            const Words<V>* codes = reinterpret_cast<const Words<V>*>(block) + (lane & 15) * 4 * (NG / V);
            const uint16_t* words = reinterpret_cast<const uint16_t*>(block + key_words_at(d)) + (lane & 15) * NG;
#pragma unroll
            for (int k0 = 0; k0 < NG; k0 += V) {
                Words<V> code[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) code[u] = codes[u * (NG / V) + k0 / V];
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const uint32_t w = words[k0 + k];
                    const float minus = 8388608.f + (float)(w & 15u), step = step_of(w);
                    float dot[kHeads] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const uint32_t x = code[u].w[k];
                        float v[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = less(x >> (4 * (e >> 1) + 16 * (e & 1)), minus);
#pragma unroll
                        for (int h = 0; h < kHeads; ++h) {
                            if (h < nh) {
                                const float4* qv = reinterpret_cast<const float4*>(qs + h * d + (k0 + k) * kGroup + u * 8);
                                const float4 a = qv[0], b = qv[1];
                                dot[h] = fmaf(a.x, v[0], fmaf(a.y, v[1], fmaf(a.z, v[2], fmaf(a.w, v[3], dot[h]))));
                                dot[h] = fmaf(b.x, v[4], fmaf(b.y, v[5], fmaf(b.z, v[6], fmaf(b.w, v[7], dot[h]))));
                            }
                        }
                    }
#pragma unroll
                    for (int h = 0; h < kHeads; ++h) s[h] = fmaf(step, dot[h], s[h]);
                }
            }
        }
        float p[kHeads];
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
            p[h] = 0.f;
            if (h >= nh) continue;
            const float top = fmaxf(m[h], warp_max(seen ? s[h] : -INFINITY));
            const float base = top == -INFINITY ? 0.f : top;
            if (seen) p[h] = expf(s[h] - base);
            const float corr = m[h] == -INFINITY ? 0.f : expf(m[h] - base);
            l[h] = l[h] * corr + warp_sum(p[h]);
            m[h] = top;
#pragma unroll
            for (int k = 0; k < NG; ++k) acc[h][k] *= corr;
        }
        // values: two tokens share a word; what is not seen counts as zero, whatever lies there
        const uint32_t mask = __ballot_sync(0xffffffffu, seen);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const unsigned char* from = reinterpret_cast<const unsigned char*>(__shfl_sync(0xffffffffu, (unsigned long long)block, 16 * b));
            if (((mask >> (16 * b)) & 0xffffu) == 0) continue;
            const uint32_t* words = reinterpret_cast<const uint32_t*>(from + value_words_at(d));
            const uint32_t* codes = reinterpret_cast<const uint32_t*>(from + value_codes_at(d)) + (lane >> 2) * 4 * NG;
#pragma unroll 4
            for (int i = 0; i < 8; ++i) {                  // tokens 2 i and 2 i + 1
                const uint32_t two = mask >> (16 * b + 2 * i), keep = (two & 1u ? 0xffffu : 0u) | (two & 2u ? 0xffff0000u : 0u);
                float p0[kHeads], p1[kHeads];
#pragma unroll
                for (int h = 0; h < kHeads; ++h) p0[h] = __shfl_sync(0xffffffffu, p[h], 16 * b + 2 * i), p1[h] = __shfl_sync(0xffffffffu, p[h], 16 * b + 2 * i + 1);
#pragma unroll
                for (int k = 0; k < NG; ++k) {
                    const uint32_t w = words[i * NG + k] & keep, x = codes[((i >> 2) * 32 + (i & 3)) * NG + k] >> (4 * (lane & 3));
                    const float x0 = less(x, 8388608.f + (float)(w & 15u)) * step_of(w), x1 = less(x >> 16, 8388608.f + (float)((w >> 16) & 15u)) * step_of(w >> 16);
#pragma unroll
                    for (int h = 0; h < kHeads; ++h) acc[h][k] = fmaf(p0[h], x0, fmaf(p1[h], x1, acc[h][k]));
                }
            }
        }
    }
    // merge: [warp][head][d + 2]
    float* part = smem + kHeads * d;
    float* share = part + (size_t)warps * kHeads * (d + 2);      // of a cluster's CTA: [head][d + 2]
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
        float* mine = part + (size_t)(warp * kHeads + h) * (d + 2);
#pragma unroll
        for (int k = 0; k < NG; ++k) mine[k * kGroup + lane] = acc[h][k];
        if (lane == 0) mine[d] = m[h], mine[d + 1] = l[h];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < nh * d; i += blockDim.x) {
        const int h = i / d, x = i - h * d;
        float top = -INFINITY, sum = 0.f, o = 0.f;
        for (int w = 0; w < warps; ++w) top = fmaxf(top, part[(size_t)(w * kHeads + h) * (d + 2) + d]);
        for (int w = 0; w < warps; ++w) {
            const float* from = part + (size_t)(w * kHeads + h) * (d + 2);
            const float f = from[d] == -INFINITY ? 0.f : expf(from[d] - top);
            sum += from[d + 1] * f;
            o += from[x] * f;
        }
        if (cluster > 1) {
            share[h * (d + 2) + x] = o;
            if (x == 0) share[h * (d + 2) + d] = top, share[h * (d + 2) + d + 1] = sum;
            continue;
        }
        // (a sum that is not a number stays one: only a row without keys is zero)
        out[(size_t)t * out_stride + (size_t)head0 * d + i] = from_f32<T>(sum == 0.f ? 0.f : o / sum);
    }
    if (cluster == 1) return;
    namespace cg = cooperative_groups;
    cg::cluster_group group = cg::this_cluster();
    group.sync();                                          // every CTA's part is in its shared memory
    for (int i = rank * blockDim.x + threadIdx.x; i < nh * d; i += cluster * blockDim.x) {
        const int h = i / d, x = i - h * d;
        float top = -INFINITY, sum = 0.f, o = 0.f;
        for (int c = 0; c < cluster; ++c) top = fmaxf(top, group.map_shared_rank(share, c)[h * (d + 2) + d]);
        for (int c = 0; c < cluster; ++c) {
            const float* from = group.map_shared_rank(share, c) + h * (d + 2);
            const float f = from[d] == -INFINITY ? 0.f : expf(from[d] - top);
            sum += from[d + 1] * f;
            o += from[x] * f;
        }
        out[(size_t)t * out_stride + (size_t)head0 * d + i] = from_f32<T>(sum == 0.f ? 0.f : o / sum);
    }
    group.sync();                                          // (a CTA's shared memory has been read before it leaves)
}

}  // namespace kv4
}  // namespace cib

using namespace cib;

// query_start_loc holds num_requests + 1 boundaries of the num_tokens rows.  longest: no request has more keys (it shapes the launch only).
extern "C" int cib_attention_kv4_generic(const void* q, int dtype, int q_stride, void* out, int out_stride, const void* cache, int num_pages, int page_size,
                                         const int* block_table, int table_stride, int table_cols, const int* query_start_loc, const int* seq_lens, int num_tokens,
                                         int num_requests, int longest, int nq, int nkv, int d, float scale, int window, int use_pdl,
                                         cudaStream_t stream) {
    CIB_REQUIRE(num_tokens >= 0 && nq > 0 && nkv > 0 && nq % nkv == 0, "attention_kv4: bad sizes T=%d nq=%d nkv=%d", num_tokens, nq, nkv);
    CIB_REQUIRE(kv4::sizes_ok(d, page_size), "attention_kv4: head size %d must be a multiple of 32 up to 256, page size %d a multiple of 16", d, page_size);
    CIB_REQUIRE(num_requests > 0 || num_tokens == 0, "attention_kv4: tokens without requests");
    CIB_REQUIRE(num_pages > 0 && table_stride > 0 && table_cols > 0 && cache != nullptr && ((uintptr_t)cache % 16) == 0, "attention_kv4: bad cache geometry");
    CIB_REQUIRE((long long)num_pages * page_size < (1ll << 31), "attention_kv4: %d pages of %d slots do not fit 32-bit slot numbers", num_pages, page_size);
    CIB_REQUIRE(q_stride >= nq * d && out_stride >= nq * d, "attention_kv4: row strides %d and %d are too small", q_stride, out_stride);
    CIB_REQUIRE(window >= 0, "attention_kv4: window must be >= 0 (0 = all keys)");
    CIB_REQUIRE(dtype == kF32 || dtype == kBF16, "attention_kv4: unsupported dtype %d", dtype);
    const int g = nq / nkv;
    CIB_REQUIRE(nkv <= 65535 && (g + kv4::kHeads - 1) / kv4::kHeads <= 65535, "attention_kv4: too many heads");
    if (num_tokens == 0) return 0;
    // a warp for every two chunks of 32 keys, so that a short context's merge stays small
    const int keys = window > 0 && window < longest ? window : longest;
    const int warps = keys <= 64 ? 1 : keys <= 128 ? 2 : keys <= 512 ? 4 : kv4::kMaxWarps;
    // (a CTA's warps have 256 keys on their way; up to four CTAs an SM)
    const long long ctas = (long long)num_tokens * nkv * ((g + kv4::kHeads - 1) / kv4::kHeads);
    int cluster = 1;
    while (cluster < kv4::kMaxCluster && ctas * cluster * 2 <= 148 * 4 && keys > cluster * 256) cluster *= 2;
    const size_t smem = (size_t)(kv4::kHeads * d + (warps + (cluster > 1 ? 1 : 0)) * kv4::kHeads * (d + 2)) * sizeof(float);
    CIB_REQUIRE((long long)num_tokens * cluster < (1ll << 31), "attention_kv4: too many rows");
    const dim3 grid(num_tokens * cluster, nkv, (g + kv4::kHeads - 1) / kv4::kHeads);
    cudaError_t e = cudaErrorInvalidValue;
#define CIB_KV4_SINGLE(NGV)                                                                                                                                \
    if (d == 32 * NGV && dtype == kF32)                                                                                                                    \
        e = launch_pdl_cluster(kv4::attention_generic_kernel<float, NGV>, grid, dim3(warps * 32), smem, stream, use_pdl != 0, cluster, (const float*)q, q_stride, \
                               (float*)out, out_stride, (unsigned char*)cache, num_pages, page_size, block_table, table_stride, table_cols, query_start_loc,    \
                               seq_lens, num_requests, nq, nkv, scale, window, cluster);                                                         \
    if (d == 32 * NGV && dtype == kBF16)                                                                                                                   \
        e = launch_pdl_cluster(kv4::attention_generic_kernel<__nv_bfloat16, NGV>, grid, dim3(warps * 32), smem, stream, use_pdl != 0, cluster,                 \
                               (const __nv_bfloat16*)q, q_stride, (__nv_bfloat16*)out, out_stride, (unsigned char*)cache, num_pages, page_size, block_table,    \
                               table_stride, table_cols, query_start_loc, seq_lens, num_requests, nq, nkv, scale, window, cluster)
    CIB_KV4_SINGLE(1);
    CIB_KV4_SINGLE(2);
    CIB_KV4_SINGLE(3);
    CIB_KV4_SINGLE(4);
    CIB_KV4_SINGLE(5);
    CIB_KV4_SINGLE(6);
    CIB_KV4_SINGLE(7);
    CIB_KV4_SINGLE(8);
#undef CIB_KV4_SINGLE
    CIB_REQUIRE(e == cudaSuccess, "attention_kv4: launch failed: %s", cudaGetErrorString(e));
    return 0;
}
