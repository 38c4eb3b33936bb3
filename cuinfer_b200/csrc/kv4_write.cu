// Appending a step's keys and values to the cache that is held in 4 bits (kv4.cuh says how), with the per-head norm and the
// rotation of the position applied on the way, and reading slots back.
//
//   q' = rot(norm(q)),  k' = rot(norm(k)) rounded once to 32 bits and quantised,  v quantised
//   norm(x) = x / sqrt(mean(x^2) + eps) * gain (optional);  rot: pairs (i, i + rotary / 2), table rows of (cos, sin) (optional)
//
// The queries are computed in 32 bits, as where the cache is not quantised.  The keys' norm and rotation are computed in 64 bits: a value next
// to the border between two codes would else fall to either side by the order of a sum, a difference of a whole step.
#include "kv4.cuh"
#include "mma_utils.cuh"

namespace cib {
namespace kv4 {

constexpr int kWarps = 4;

// Any head size that is a multiple of 32: a warp per (token, head); lane l holds value l of every group.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
write_kernel(const T* qkv, int row_stride, T* q_out, int q_stride, const int* __restrict__ positions,
             const int* __restrict__ slots, AnyVec q_gain, AnyVec k_gain, int has_norm, float eps, const float* __restrict__ rope_table,
             int rotary, int max_positions, unsigned char* __restrict__ cache, int num_pages, int page_size, int nq, int nkv, int d) {
    __shared__ float s_x[kWarps][kMaxHeadDim];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = blockIdx.x;
    const int head = blockIdx.y * kWarps + warp;
    griddep_wait();
    griddep_launch();        // (behind the wait: what follows may count on everything in front of this kernel being done)
    if (head >= nq + 2 * nkv) return;
    const int kind = head < nq ? 0 : (head < nq + nkv ? 1 : 2);              // query, key, value
    const int kvh = kind == 0 ? 0 : (head - nq) % nkv;
    unsigned char* block = nullptr;
    int token = 0;
    if (kind != 0) {
        const int slot = slots[t];
        block = block_of(cache, slot, num_pages, page_size, nkv, kvh, d);
        if (block == nullptr) return;
        token = slot % page_size % kBlock;
    }
    float* x = s_x[warp];
    const T* src = qkv + (size_t)t * row_stride + (size_t)head * d;
    for (int i = lane; i < d; i += 32) x[i] = to_f32(src[i]);
    __syncwarp();
    const int half = rotary >> 1;
    const float* table = nullptr;
    if (half > 0 && kind != 2) {
        int pos = positions[t];
        pos = pos < 0 ? 0 : (pos >= max_positions ? max_positions - 1 : pos);
        table = rope_table + (size_t)pos * rotary;
    }
    if (kind == 0) {
        float factor = 1.f;
        if (has_norm) {
            float ss = 0.f;
            for (int i = lane; i < d; i += 32) ss += x[i] * x[i];
            factor = rsqrtf(warp_sum(ss) / (float)d + eps);
        }
        T* dst = q_out + (size_t)t * q_stride + (size_t)head * d;
        auto normed = [&](int i) { return has_norm ? x[i] * factor * q_gain[i] : x[i]; };
        for (int i = lane; i < d; i += 32) {
            float y = normed(i);
            if (i < rotary) {
                const int p = i < half ? i : i - half;
                const float c = table[2 * p], s = table[2 * p + 1];
                y = i < half ? y * c - normed(i + half) * s : y * c + normed(i - half) * s;
            }
            dst[i] = from_f32<T>(y);
        }
        return;
    }
    double factor = 1.0;
    if (kind == 1 && has_norm) {
        double ss = 0.0;
        for (int i = lane; i < d; i += 32) ss += (double)x[i] * (double)x[i];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        factor = 1.0 / sqrt(ss / (double)d + (double)eps);
    }
    auto normed = [&](int i) { return has_norm ? (double)x[i] * factor * (double)k_gain[i] : (double)x[i]; };
    const int groups = d / kGroup;
    for (int g = 0; g < groups; ++g) {
        const int i = g * kGroup + lane;
        float y = x[i];
        if (kind == 1) {
            double z = normed(i);
            if (i < rotary) {
                const int p = i < half ? i : i - half;
                const double c = table[2 * p], s = table[2 * p + 1];
                z = i < half ? z * c - normed(i + half) * s : z * c + normed(i - half) * s;
            }
            y = (float)z;
        }
        const bool bad = __any_sync(0xffffffffu, !holds(y));
        const float hi = warp_max(fmaxf(y, 0.f)), lo = -warp_max(fmaxf(-y, 0.f));
        const Scale s = scale_of(lo, hi, bad);
        uint32_t code = code_of(y, s, bad);
        if (kind == 1) {
            const int e = lane & 7;
            code <<= 4 * (e >> 1) + 16 * (e & 1);
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) code |= __shfl_xor_sync(0xffffffffu, code, o);
            if (e == 0) reinterpret_cast<uint32_t*>(block)[(token * 4 + (lane >> 3)) * groups + g] = code;
            if (lane == 0) reinterpret_cast<uint16_t*>(block + key_words_at(d))[token * groups + g] = (uint16_t)s.word;
        } else {
            const int e = lane & 3;
            code <<= 4 * e;
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) code |= __shfl_xor_sync(0xffffffffu, code, o);
            const int word = (((token >> 3) * 8 + (lane >> 2)) * 4 + ((token & 7) >> 1)) * groups + g;
            if (e == 0) reinterpret_cast<uint16_t*>(block + value_codes_at(d))[word * 2 + (token & 1)] = (uint16_t)code;
            if (lane == 0) reinterpret_cast<uint16_t*>(block + value_words_at(d))[((token >> 1) * groups + g) * 2 + (token & 1)] = (uint16_t)s.word;
        }
    }
}

// A warp per (slot, kv head): rows of slots that are none are left as they are.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
read_kernel(unsigned char* __restrict__ cache, int num_pages, int page_size, const int* __restrict__ slots, T* __restrict__ keys, int key_stride,
            T* __restrict__ values, int value_stride, int nkv, int d) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = blockIdx.x;
    const int kvh = blockIdx.y * kWarps + warp;
    griddep_wait();
    griddep_launch();
    if (kvh >= nkv) return;
    const int slot = slots[t];
    const unsigned char* block = block_of(cache, slot, num_pages, page_size, nkv, kvh, d);
    if (block == nullptr) return;
    const int token = slot % page_size % kBlock;
    const int groups = d / kGroup;
    for (int g = 0; g < groups; ++g) {
        const uint32_t kw = reinterpret_cast<const uint16_t*>(block + key_words_at(d))[token * groups + g];
        const uint32_t vw = reinterpret_cast<const uint16_t*>(block + value_words_at(d))[((token >> 1) * groups + g) * 2 + (token & 1)];
        const uint32_t kc = reinterpret_cast<const uint32_t*>(block)[(token * 4 + (lane >> 3)) * groups + g];
        const int word = (((token >> 3) * 8 + (lane >> 2)) * 4 + ((token & 7) >> 1)) * groups + g;
        const uint32_t vc = reinterpret_cast<const uint16_t*>(block + value_codes_at(d))[word * 2 + (token & 1)];
        const int e = lane & 7;
        const int k = (int)((kc >> (4 * (e >> 1) + 16 * (e & 1))) & 15u) - (int)(kw & 15u);
        const int v = (int)((vc >> (4 * (lane & 3))) & 15u) - (int)(vw & 15u);
        const int i = kvh * d + g * kGroup + lane;
        keys[(size_t)t * key_stride + i] = from_f32<T>(step_of(kw) * (float)k);
        values[(size_t)t * value_stride + i] = from_f32<T>(step_of(vw) * (float)v);
    }
}

}  // namespace kv4
}  // namespace cib

using namespace cib;

extern "C" int cib_qk_norm_rope_kv4_write(const void* qkv, int dtype, int row_stride, void* q_out, int q_stride, const int* positions,
                                          const int* slots, const void* q_gain, const void* k_gain, int gain_dtype, int has_norm, float eps,
                                          const float* rope_table, int rotary, int max_positions, void* cache, int num_pages, int page_size,
                                          int num_tokens, int nq, int nkv, int d, int use_pdl, cudaStream_t stream) {
    CIB_REQUIRE(num_tokens >= 0 && nq > 0 && nkv > 0, "qk_norm_rope_kv4_write: bad sizes T=%d nq=%d nkv=%d", num_tokens, nq, nkv);
    CIB_REQUIRE(kv4::sizes_ok(d, page_size), "qk_norm_rope_kv4_write: head size %d must be a multiple of 32 up to 256, page size %d a multiple of 16", d, page_size);
    CIB_REQUIRE(rotary >= 0 && rotary <= d && rotary % 2 == 0, "qk_norm_rope_kv4_write: rotary size %d must be even and at most the head size %d", rotary, d);
    CIB_REQUIRE(rotary == 0 || (rope_table != nullptr && max_positions > 0), "qk_norm_rope_kv4_write: rotary table missing");
    CIB_REQUIRE(!has_norm || (q_gain && k_gain), "qk_norm_rope_kv4_write: norm gains missing");
    CIB_REQUIRE(row_stride >= (nq + 2 * nkv) * d && q_stride >= nq * d, "qk_norm_rope_kv4_write: row strides %d and %d are too small", row_stride, q_stride);
    CIB_REQUIRE(cache != nullptr && num_pages > 0 && ((uintptr_t)cache % 16) == 0, "qk_norm_rope_kv4_write: cache missing or not 16-byte aligned");
    CIB_REQUIRE(dtype == kF32 || dtype == kBF16, "qk_norm_rope_kv4_write: unsupported dtype %d", dtype);
    if (num_tokens == 0) return 0;
    const AnyVec qg{q_gain, gain_dtype == kBF16}, kg{k_gain, gain_dtype == kBF16};
    const int heads = nq + 2 * nkv;
    CIB_REQUIRE((heads + kv4::kWarps - 1) / kv4::kWarps <= 65535, "qk_norm_rope_kv4_write: %d heads are too many", heads);
    const dim3 grid(num_tokens, (heads + kv4::kWarps - 1) / kv4::kWarps);
    cudaError_t e;
    if (dtype == kF32)
        e = launch_pdl(kv4::write_kernel<float>, grid, dim3(kv4::kWarps * 32), 0, stream, use_pdl != 0, (const float*)qkv, row_stride, (float*)q_out, q_stride,
                       positions, slots, qg, kg, has_norm, eps, rope_table, rotary, max_positions, (unsigned char*)cache, num_pages, page_size, nq, nkv, d);
    else
        e = launch_pdl(kv4::write_kernel<__nv_bfloat16>, grid, dim3(kv4::kWarps * 32), 0, stream, use_pdl != 0, (const __nv_bfloat16*)qkv, row_stride,
                       (__nv_bfloat16*)q_out, q_stride, positions, slots, qg, kg, has_norm, eps, rope_table, rotary, max_positions, (unsigned char*)cache, num_pages,
                       page_size, nq, nkv, d);
    CIB_REQUIRE(e == cudaSuccess, "qk_norm_rope_kv4_write: launch failed: %s", cudaGetErrorString(e));
    return 0;
}

extern "C" int cib_kv4_read(const void* cache, int num_pages, int page_size, const int* slots, void* keys, int key_stride, void* values, int value_stride,
                            int dtype, int num_slots, int nkv, int d, int use_pdl, cudaStream_t stream) {
    CIB_REQUIRE(num_slots >= 0 && nkv > 0 && nkv <= 4 * 65535, "kv4_read: bad sizes");
    CIB_REQUIRE(kv4::sizes_ok(d, page_size), "kv4_read: head size %d must be a multiple of 32 up to 256, page size %d a multiple of 16", d, page_size);
    CIB_REQUIRE(key_stride >= nkv * d && value_stride >= nkv * d, "kv4_read: row strides %d and %d are too small", key_stride, value_stride);
    CIB_REQUIRE(cache != nullptr && num_pages > 0 && ((uintptr_t)cache % 16) == 0, "kv4_read: cache missing or not 16-byte aligned");
    CIB_REQUIRE(dtype == kF32 || dtype == kBF16, "kv4_read: unsupported dtype %d", dtype);
    if (num_slots == 0) return 0;
    const dim3 grid(num_slots, (nkv + kv4::kWarps - 1) / kv4::kWarps);
    cudaError_t e;
    if (dtype == kF32)
        e = launch_pdl(kv4::read_kernel<float>, grid, dim3(kv4::kWarps * 32), 0, stream, use_pdl != 0, (unsigned char*)cache, num_pages, page_size, slots,
                       (float*)keys, key_stride, (float*)values, value_stride, nkv, d);
    else
        e = launch_pdl(kv4::read_kernel<__nv_bfloat16>, grid, dim3(kv4::kWarps * 32), 0, stream, use_pdl != 0, (unsigned char*)cache, num_pages, page_size, slots,
                       (__nv_bfloat16*)keys, key_stride, (__nv_bfloat16*)values, value_stride, nkv, d);
    CIB_REQUIRE(e == cudaSuccess, "kv4_read: launch failed: %s", cudaGetErrorString(e));
    return 0;
}
