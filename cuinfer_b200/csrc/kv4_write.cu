// Appending a step's keys and values to the cache that is held in 4 bits (kv4.cuh says how), with the per-head norm and the
// rotation of the position applied on the way, and reading slots back.
//
//   q' = rot(norm(q)),  k' = rot(norm(k)) rounded once to 32 bits and quantised,  v quantised
//   norm(x) = x / sqrt(mean(x^2) + eps) * gain (optional);  rot: pairs (i, i + rotary / 2), table rows of (cos, sin) (optional)
//
// The queries are computed in 32 bits, as where the cache is not quantised.  The keys' norm and rotation are computed in 64 bits: a value next
// to the border between two codes would else fall to either side by the order of a sum, a difference of a whole step.
#include <algorithm>

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

template <typename T, int E>
struct alignas(sizeof(T) * E > 16 ? 16 : sizeof(T) * E) Lane {
    T v[E];
};

// Prompts: head sizes 64, 128 and 256, a rotation of the whole head or none.  A head lies in L = D / 16 lanes; a lane has eight values of its first
// half and their rotation partners of the second, so nothing is exchanged but the sums; eight values are a whole word of key codes and two half
// words of value codes.  A warp takes PASSES x 32 / L heads of one token, with all loads on their way at once.
//
// Keys are computed in 32 bits here too, together with a bound of their error, and only a warp that has a value (or a step) within
// that bound of a border between two codes does it again in 64 bits: the codes are those of the 64-bit computation, which alone took
// two thirds of the time.  The bound, in units of 2^-24 of |a cos| + |b sin| (of the value where nothing is rotated): the sum of squares is 8 + 1 + 4
// additions deep at most and eps one more, which the root halves, 7; the reciprocal root is good to two units in the last place, 4; two products, 2;
// the rotation's products and sum, 2; and the 64-bit result is rounded to 32 itself, 1.  16, and two more for the products of these errors
// and what the bound is computed with.  Without a norm 3, of which 4 are made.
constexpr int kRowWarps = 8, kRowCtas = 2;          // CTAs an SM (three, which leave 80 registers, spill: 100 us for 8 001 tokens of 48 heads instead of 70)

template <typename T>
struct alignas(sizeof(T) * 8 > 16 ? 16 : sizeof(T) * 8) Eight {
    T v[8];
};

// Sixteen values of a lane (eight of either half; a group is four lanes of a half) as they are stored: the lane's codes and the groups' words.
// `key`: in the order of key codes, else of value codes.  `worst`: how far values of the group may be off; returns whether a code, a zero point or
// a step could be another one then.  Codes are small whole numbers: four of them are summed up by weight and converted at once.
__device__ __forceinline__ bool quantise_lane(const float (&x)[16], bool key, float worst, int lane, uint32_t (&word)[2], uint32_t (&step)[2]) {
    bool near = false;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float lo = 0.f, hi = 0.f, odd = 0.f;                         // odd: 0, or not a number where a value is not finite
#pragma unroll
        for (int e = 0; e < 8; ++e) lo = fminf(lo, x[8 * h + e]), hi = fmaxf(hi, x[8 * h + e]), odd = fmaf(x[8 * h + e], 0.f, odd);
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        const bool bad = ((__ballot_sync(0xffffffffu, !(odd == 0.f) || !holds(hi) || !holds(lo)) >> (lane & 28)) & 15u) != 0;
        const Scale s = scale_of(lo, hi, bad);
        float c[8], off = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float f = quotient(x[8 * h + e], s.step, s.inverse), k = rintf(f);
            off = fmaxf(off, fabsf(f - k));
            c[e] = fminf(fmaxf(k + s.zero, 0.f), 15.f);
        }
        float low, high;                                             // the halves of the lane's word
        if (key) {
            low = fmaf(fmaf(fmaf(c[6], 16.f, c[4]), 16.f, c[2]), 16.f, c[0]);
            high = fmaf(fmaf(fmaf(c[7], 16.f, c[5]), 16.f, c[3]), 16.f, c[1]);
        } else {
            low = fmaf(fmaf(fmaf(c[3], 16.f, c[2]), 16.f, c[1]), 16.f, c[0]);
            high = fmaf(fmaf(fmaf(c[7], 16.f, c[6]), 16.f, c[5]), 16.f, c[4]);
        }
        // (whole numbers below 2^16: adding 2^23 leaves them in the lowest bits)
        word[h] = bad ? 0u : __byte_perm(__float_as_uint(low + 8388608.f), __float_as_uint(high + 8388608.f), 0x5410);
        step[h] = s.word;
        const float margin = 0.5f - (worst * s.inverse + 1.9073486e-06f);          // (2^-19: the quotients themselves)
        const float z = quotient(-lo, s.step, s.inverse), range = hi - lo, slack = 2.f * worst + range * 4.7683716e-07f;       // (2^-21)
        const uint32_t below = __float_as_uint(fmaxf((range - slack) * (1.f / 15.f), 0.f)) + 0xfffffu, above = __float_as_uint((range + slack) * (1.f / 15.f)) + 0xfffffu;
        near = near || !(fmaxf(off, fabsf(z - rintf(z))) <= margin) || ((below ^ above) & ~0xfffffu) != 0 || !(fmaxf(hi, -lo) < 8.507059e37f) || !(odd == 0.f);     // 2^126
    }
    return near;
}
// ... and where they go: `li` is the lane within its head.
template <int D>
__device__ __forceinline__ void store_lane(unsigned char* block, bool key, int token, int li, const uint32_t (&word)[2], const uint32_t (&step)[2]) {
    constexpr int NG = D / kGroup;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int g = (li >> 2) + h * (NG / 2), quarter = li & 3;
        if (key) {
            reinterpret_cast<uint32_t*>(block)[(token * 4 + quarter) * NG + g] = word[h];
            if (quarter == 0) reinterpret_cast<uint16_t*>(block + key_words_at(D))[token * NG + g] = (uint16_t)step[h];
        } else {
            uint16_t* codes = reinterpret_cast<uint16_t*>(block + value_codes_at(D)) +
                              ((((token >> 3) * 8 + 2 * quarter) * 4 + ((token & 7) >> 1)) * NG + g) * 2 + (token & 1);
            codes[0] = (uint16_t)word[h];
            codes[8 * NG] = (uint16_t)(word[h] >> 16);
            if (quarter == 0) reinterpret_cast<uint16_t*>(block + value_words_at(D))[((token >> 1) * NG + g) * 2 + (token & 1)] = (uint16_t)step[h];
        }
    }
}
// The key heads of a pass in 64 bits (a call of its own: few warps need it, and its registers would cost all of them).
template <typename T, int L>
__device__ __noinline__ void write_keys_exactly(const T* src, bool mine, const float* gain, int has_norm, float eps, const float* table, int has_rope,
                                                unsigned char* block, int token, int li) {
    constexpr int D = 16 * L;
    const Eight<T> first = *reinterpret_cast<const Eight<T>*>(src), second = *reinterpret_cast<const Eight<T>*>(src + D / 2);
    double factor = 1.0;
    if (has_norm) {
        double ss = 0.0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const double a = to_f32(first.v[e]), b = to_f32(second.v[e]);
            ss += a * a + b * b;
        }
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        factor = 1.0 / sqrt(ss / (double)D + (double)eps);
    }
    float x[16];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        double a = to_f32(first.v[e]), b = to_f32(second.v[e]);
        if (has_norm) a = a * factor * (double)gain[8 * li + e], b = b * factor * (double)gain[D / 2 + 8 * li + e];
        if (has_rope) {
            const double c = table[16 * li + 2 * e], s = table[16 * li + 2 * e + 1];
            x[e] = (float)(a * c - b * s);
            x[8 + e] = (float)(b * c + a * s);
        } else {
            x[e] = (float)a, x[8 + e] = (float)b;
        }
    }
    uint32_t word[2], step[2];
    quantise_lane(x, true, 0.f, threadIdx.x & 31, word, step);
    if (mine) store_lane<D>(block, true, token, li, word, step);
}

template <typename T, int L, int PASSES>
__global__ void __launch_bounds__(kRowWarps * 32, kRowCtas)
write_rows_kernel(const T* qkv, int row_stride, T* q_out, int q_stride, const int* __restrict__ positions, const int* __restrict__ slots, AnyVec q_gain,
                  AnyVec k_gain, int has_norm, float eps, const float* __restrict__ rope_table, int has_rope, int max_positions,
                  unsigned char* __restrict__ cache, int num_pages, int page_size, int nq, int nkv, int num_tokens) {
    constexpr int D = 16 * L, NG = D / kGroup, HPP = 32 / L;         // heads a pass
    __shared__ __align__(16) float s_gain[2][D];
    if (has_norm)
        for (int i = threadIdx.x; i < 2 * D; i += blockDim.x) s_gain[i / D][i % D] = i < D ? q_gain[i] : k_gain[i - D];
    const int lane = threadIdx.x & 31, sub = lane / L, li = lane % L;
    const int heads = nq + 2 * nkv, chunks = (heads + HPP * PASSES - 1) / (HPP * PASSES);
    const size_t head_bytes = (size_t)(page_size / kBlock) * block_bytes(D);
    griddep_wait();
    griddep_launch();
    __syncthreads();
    // the launch has as many CTAs as the GPU holds: a warp goes on with the next piece of work instead of leaving and another starting
    const long long pieces = (long long)num_tokens * chunks;
    for (long long w = (long long)blockIdx.x * kRowWarps + (threadIdx.x >> 5); w < pieces; w += (long long)gridDim.x * kRowWarps) {
    const int t = (int)(w / chunks), base = (int)(w - (long long)t * chunks) * HPP * PASSES;
    float cs[16];
    unsigned again = 0;                                              // passes with a key near a border
    const float* rope_row = rope_table;
    const int slot = slots[t];
    if (has_rope) {
        int pos = positions[t];
        pos = pos < 0 ? 0 : (pos >= max_positions ? max_positions - 1 : pos);
        rope_row = rope_table + (size_t)pos * D;
        const float4* tp = reinterpret_cast<const float4*>(rope_row + 16 * li);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float4 v = tp[e];
            cs[4 * e] = v.x, cs[4 * e + 1] = v.y, cs[4 * e + 2] = v.z, cs[4 * e + 3] = v.w;
        }
    }
    const T* src = qkv + (size_t)t * row_stride + 8 * li;
    Eight<T> first[PASSES], second[PASSES];
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
        const int head = base + p * HPP + sub;
        if (head < heads) {
            first[p] = *reinterpret_cast<const Eight<T>*>(src + (size_t)head * D);
            second[p] = *reinterpret_cast<const Eight<T>*>(src + (size_t)head * D + D / 2);
        }
    }
    unsigned char* block0 = block_of(cache, slot, num_pages, page_size, nkv, 0, D);
    const int token = block0 == nullptr ? 0 : slot % page_size % kBlock;
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
        const int head = base + p * HPP + sub;
        const int kind = head < nq ? 0 : (head < nq + nkv ? 1 : 2);          // (a head behind the last one: a value that is not stored)
        const bool stored = head < heads;
        if (base + p * HPP >= heads) break;
        float x[16];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = stored ? to_f32(first[p].v[e]) : 0.f, x[8 + e] = stored ? to_f32(second[p].v[e]) : 0.f;
        float error = 0.f;                                           // of the values as they are computed below, at most
        bool rough = false;                                          // the mean square has left the range in which 32 bits hold it
        if (__any_sync(0xffffffffu, kind != 2)) {
            if (has_norm) {
                float s0 = 0.f, s1 = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) s0 = fmaf(x[e], x[e], s0), s1 = fmaf(x[8 + e], x[8 + e], s1);
                float ss = s0 + s1;
#pragma unroll
                for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                const float mean = ss / (float)D + eps, factor = kind == 2 ? 1.f : rsqrtf(mean);
                rough = !(mean > 1e-30f && ss < 3e38f);
                const float* gain = s_gain[kind == 0 ? 0 : 1] + 8 * li;
#pragma unroll
                for (int e = 0; e < 8; e += 4) {
                    const float4 a = *reinterpret_cast<const float4*>(gain + e), b = *reinterpret_cast<const float4*>(gain + D / 2 + e);
                    if (kind != 2) {
                        x[e] = x[e] * factor * a.x, x[e + 1] = x[e + 1] * factor * a.y, x[e + 2] = x[e + 2] * factor * a.z, x[e + 3] = x[e + 3] * factor * a.w;
                        x[8 + e] = x[8 + e] * factor * b.x, x[9 + e] = x[9 + e] * factor * b.y, x[10 + e] = x[10 + e] * factor * b.z, x[11 + e] = x[11 + e] * factor * b.w;
                    }
                }
            }
            if (kind != 2) {
                if (has_rope) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float c = cs[2 * e], s = cs[2 * e + 1], a = x[e], b = x[8 + e];
                        const float ac = a * c, bs = b * s, bc = b * c, as = a * s;
                        x[e] = ac - bs;
                        x[8 + e] = bc + as;
                        if (kind == 1) error = fmaxf(error, fmaxf(fabsf(ac) + fabsf(bs), fabsf(bc) + fabsf(as)));
                    }
                } else if (kind == 1 && has_norm) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) error = fmaxf(error, fabsf(x[e]));
                }
                error *= has_norm ? 1.0728836e-06f : 2.3841858e-07f;       // 18 and 4 times 2^-24
                if (kind == 1 && rough) error = INFINITY;
            }
        }
        if (kind == 0 && stored) {
            Eight<T> a, b;
#pragma unroll
            for (int e = 0; e < 8; ++e) a.v[e] = from_f32<T>(x[e]), b.v[e] = from_f32<T>(x[8 + e]);
            T* dst = q_out + (size_t)t * q_stride + (size_t)head * D + 8 * li;
            *reinterpret_cast<Eight<T>*>(dst) = a;
            *reinterpret_cast<Eight<T>*>(dst + D / 2) = b;
        }
        if (block0 == nullptr || !__any_sync(0xffffffffu, kind != 0)) continue;
        uint32_t word[2], step[2];
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) error = fmaxf(error, __shfl_xor_sync(0xffffffffu, error, o));
        const bool near = quantise_lane(x, kind == 1, error, lane, word, step);
        if (__any_sync(0xffffffffu, near && kind == 1 && error != 0.f)) again |= 1u << p;
        if (kind != 0 && stored) store_lane<D>(block0 + (head - nq - (kind == 2 ? nkv : 0)) * head_bytes, kind == 1, token, li, word, step);
    }
    // keys near a border: the pass's key heads again (a lane stores to where it stored before)
    while (again != 0) {
        const int p = __ffs(again) - 1;
        again &= again - 1;
        const int head = base + p * HPP + sub;
        const bool mine = head >= nq && head < nq + nkv;
        write_keys_exactly<T, L>(src + (size_t)(mine ? head : nq) * D, mine, s_gain[1], has_norm, eps, rope_row, has_rope,
                                 block0 + (mine ? head - nq : 0) * head_bytes, token, li);
    }
    }
}

// The same head sizes with few tokens, or a rotation of a part of the head whose halves are whole lanes.  A lane has E = D / 32 neighbouring values of a
// head, 32 / E lanes a group; a warp takes HB heads of one token: all their loads are issued at once, and what depends on the token only
// (slot, position, table row, gains) is fetched once and before the wait for the kernel in front.  The rotation's partner
// lies `rotary / 2 / E` lanes away; it is exchanged as it came, so that the exchange is exact, and normed again where it arrives.
// Bound by the memory's latency.
template <typename T, int E, int HB>
__global__ void __launch_bounds__(kWarps * 32)
write_lanes_kernel(const T* qkv, int row_stride, T* q_out, int q_stride, const int* __restrict__ positions, const int* __restrict__ slots, AnyVec q_gain,
                   AnyVec k_gain, int has_norm, float eps, const float* __restrict__ rope_table, int rotary, int max_positions,
                   unsigned char* __restrict__ cache, int num_pages, int page_size, int nq, int nkv, int num_tokens) {
    constexpr int D = 32 * E, NG = E, kLanes = 32 / E;               // lanes of a group
    const int lane = threadIdx.x & 31;
    const int heads = nq + 2 * nkv, chunks = (heads + HB - 1) / HB;
    const int w = blockIdx.x * kWarps + (threadIdx.x >> 5);
    const int t = w / chunks, base = (w - t * chunks) * HB;
    const bool live = t < num_tokens;
    const int i0 = lane * E;
    const int reach = rotary / (2 * E);                              // lanes of half a rotation
    const bool rotates = lane < 2 * reach;
    const int partner = !rotates ? lane : lane < reach ? lane + reach : lane - reach;
    int slot = -1;
    float cs[2 * E], gain_q[E], gain_k[E], gain_p[E];                // cosines and sines; gains of this lane and, for keys, of its partner
    if (live) {
        slot = slots[t];
        if (rotates) {
            int pos = positions[t];
            pos = pos < 0 ? 0 : (pos >= max_positions ? max_positions - 1 : pos);
            const float* tp = rope_table + (size_t)pos * rotary + 2 * ((lane < reach ? lane : lane - reach) * E);
#pragma unroll
            for (int e = 0; e < 2 * E; e += 4) {
                const float4 v = *reinterpret_cast<const float4*>(tp + e);
                cs[e] = v.x, cs[e + 1] = v.y, cs[e + 2] = v.z, cs[e + 3] = v.w;
            }
        }
        if (has_norm) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (base < nq) gain_q[e] = q_gain[i0 + e];
                if (base + HB > nq) gain_k[e] = k_gain[i0 + e], gain_p[e] = k_gain[partner * E + e];
            }
        }
    }
    griddep_wait();
    griddep_launch();
    if (!live) return;
    const T* src = qkv + (size_t)t * row_stride + (size_t)base * D + i0;
    Lane<T, E> raw[HB];
#pragma unroll
    for (int h = 0; h < HB; ++h)
        if (base + h < heads) raw[h] = *reinterpret_cast<const Lane<T, E>*>(src + h * D);
    unsigned char* block0 = block_of(cache, slot, num_pages, page_size, nkv, 0, D);
    const size_t head_bytes = (size_t)(page_size / kBlock) * block_bytes(D);
    const int token = block0 == nullptr ? 0 : slot % page_size % kBlock;
#pragma unroll
    for (int h = 0; h < HB; ++h) {
        const int head = base + h;
        if (head >= heads) break;
        const int kind = head < nq ? 0 : (head < nq + nkv ? 1 : 2);
        float x[E];
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = to_f32(raw[h].v[e]);
        if (kind == 0) {
            if (has_norm) {
                float ss = 0.f;
#pragma unroll
                for (int e = 0; e < E; ++e) ss += x[e] * x[e];
                const float factor = rsqrtf(warp_sum(ss) / (float)D + eps);
#pragma unroll
                for (int e = 0; e < E; ++e) x[e] = x[e] * factor * gain_q[e];
            }
            if (reach > 0) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float other = __shfl_sync(0xffffffffu, x[e], partner);
                    if (rotates) x[e] = lane < reach ? x[e] * cs[2 * e] - other * cs[2 * e + 1] : x[e] * cs[2 * e] + other * cs[2 * e + 1];
                }
            }
            Lane<T, E> o;
#pragma unroll
            for (int e = 0; e < E; ++e) o.v[e] = from_f32<T>(x[e]);
            *reinterpret_cast<Lane<T, E>*>(q_out + (size_t)t * q_stride + (size_t)head * D + i0) = o;
            continue;
        }
        if (block0 == nullptr) continue;
        unsigned char* block = block0 + (head - nq - (kind == 2 ? nkv : 0)) * head_bytes;
        if (kind == 1 && (has_norm || reach > 0)) {
            double factor = 1.0;
            if (has_norm) {
                double ss = 0.0;
#pragma unroll
                for (int e = 0; e < E; ++e) ss += (double)x[e] * (double)x[e];
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                factor = 1.0 / sqrt(ss / (double)D + (double)eps);
            }
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float other = __shfl_sync(0xffffffffu, x[e], partner);
                double a = has_norm ? (double)x[e] * factor * (double)gain_k[e] : (double)x[e];
                if (rotates) {
                    const double b = has_norm ? (double)other * factor * (double)gain_p[e] : (double)other;
                    const double c = cs[2 * e], s = cs[2 * e + 1];
                    a = lane < reach ? a * c - b * s : a * c + b * s;
                }
                // (the exchange of value e is over before x[e] changes: all lanes are here)
                x[e] = (float)a;
            }
        }
        float lo = 0.f, hi = 0.f;
        bool bad = false;
#pragma unroll
        for (int e = 0; e < E; ++e) lo = fminf(lo, x[e]), hi = fmaxf(hi, x[e]), bad = bad || !holds(x[e]);
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        const uint32_t group_lanes = (kLanes == 32 ? 0xffffffffu : ((1u << kLanes) - 1u) << (lane / kLanes * kLanes));
        bad = (__ballot_sync(0xffffffffu, bad) & group_lanes) != 0;
        const Scale s = scale_of(lo, hi, bad);
        uint32_t code[E];
#pragma unroll
        for (int e = 0; e < E; ++e) code[e] = code_of(x[e], s, bad);
        const int g = lane / kLanes, in = (lane & (kLanes - 1)) * E;   // this lane's first value within its group
        if (kind == 1) {
            // eight values a word, value e of them in bits 4 (e / 2) + 16 (e % 2)
            uint32_t word = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int at = (in + e) & 7;
                word |= code[e] << (4 * (at >> 1) + 16 * (at & 1));
            }
#pragma unroll
            for (int o = 1; o < 8 / E; o <<= 1) word |= __shfl_xor_sync(0xffffffffu, word, o);
            if ((in & 7) == 0) reinterpret_cast<uint32_t*>(block)[(token * 4 + (in >> 3)) * NG + g] = word;
            if (in == 0) reinterpret_cast<uint16_t*>(block + key_words_at(D))[token * NG + g] = (uint16_t)s.word;
        } else {
            // four values a half word
            constexpr int kHalves = E > 4 ? E / 4 : 1;
            uint16_t* codes = reinterpret_cast<uint16_t*>(block + value_codes_at(D));
#pragma unroll
            for (int u = 0; u < kHalves; ++u) {
                uint32_t half = 0;
#pragma unroll
                for (int e = 0; e < (E > 4 ? 4 : E); ++e) half |= code[4 * u + e] << (4 * ((in + e) & 3));
                if (E == 2) half |= __shfl_xor_sync(0xffffffffu, half, 1);
                const int word = (((token >> 3) * 8 + (in >> 2) + u) * 4 + ((token & 7) >> 1)) * NG + g;
                if (E >= 4 || (in & 3) == 0) codes[word * 2 + (token & 1)] = (uint16_t)half;
            }
            if (in == 0) reinterpret_cast<uint16_t*>(block + value_words_at(D))[((token >> 1) * NG + g) * 2 + (token & 1)] = (uint16_t)s.word;
        }
    }
}

// A warp per (slot, HB kv heads), a lane E = D / 32 neighbouring values: head sizes 64, 128 and 256.
template <typename T, int E, int HB>
__global__ void __launch_bounds__(kWarps * 32)
read_lanes_kernel(unsigned char* __restrict__ cache, int num_pages, int page_size, const int* __restrict__ slots, T* __restrict__ keys, int key_stride,
                  T* __restrict__ values, int value_stride, int nkv, int num_slots) {
    constexpr int D = 32 * E, NG = E, kLanes = 32 / E;
    const int lane = threadIdx.x & 31;
    const int chunks = (nkv + HB - 1) / HB;
    const int w = blockIdx.x * kWarps + (threadIdx.x >> 5);
    const int t = w / chunks, base = (w - t * chunks) * HB;
    griddep_wait();
    griddep_launch();
    if (t >= num_slots) return;
    const int slot = slots[t];
    const unsigned char* block0 = block_of(cache, slot, num_pages, page_size, nkv, base, D);
    if (block0 == nullptr) return;
    const size_t head_bytes = (size_t)(page_size / kBlock) * block_bytes(D);
    const int token = slot % page_size % kBlock;
    const int g = lane / kLanes, in = (lane & (kLanes - 1)) * E;
    uint32_t kc[HB], kw[HB], vw[HB], vc[HB];
#pragma unroll
    for (int h = 0; h < HB; ++h) {
        if (base + h >= nkv) break;
        const unsigned char* block = block0 + h * head_bytes;
        kc[h] = reinterpret_cast<const uint32_t*>(block)[(token * 4 + (in >> 3)) * NG + g];
        kw[h] = reinterpret_cast<const uint16_t*>(block + key_words_at(D))[token * NG + g];
        vw[h] = reinterpret_cast<const uint16_t*>(block + value_words_at(D))[((token >> 1) * NG + g) * 2 + (token & 1)];
        const uint16_t* codes = reinterpret_cast<const uint16_t*>(block + value_codes_at(D));
        const int word = (((token >> 3) * 8 + (in >> 2)) * 4 + ((token & 7) >> 1)) * NG + g;
        vc[h] = codes[word * 2 + (token & 1)];
        if (E == 8) vc[h] |= (uint32_t)codes[(word + 4 * NG) * 2 + (token & 1)] << 16;
    }
#pragma unroll
    for (int h = 0; h < HB; ++h) {
        if (base + h >= nkv) break;
        Lane<T, E> k, v;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int at = (in + e) & 7;
            k.v[e] = from_f32<T>(step_of(kw[h]) * (float)((int)((kc[h] >> (4 * (at >> 1) + 16 * (at & 1))) & 15u) - (int)(kw[h] & 15u)));
            v.v[e] = from_f32<T>(step_of(vw[h]) * (float)((int)((vc[h] >> (4 * (E == 2 ? (in + e) & 3 : e))) & 15u) - (int)(vw[h] & 15u)));
        }
        *reinterpret_cast<Lane<T, E>*>(keys + (size_t)t * key_stride + (size_t)(base + h) * D + lane * E) = k;
        *reinterpret_cast<Lane<T, E>*>(values + (size_t)t * value_stride + (size_t)(base + h) * D + lane * E) = v;
    }
}

// From so many warps of a head each on, a warp takes four heads: the GPU is full either way.
constexpr long long kManyHeads = 148 * 64;

template <typename T>
static cudaError_t launch_write(int d, cudaStream_t stream, bool use_pdl, const T* qkv, int row_stride, T* q_out, int q_stride, const int* positions, const int* slots,
                                AnyVec qg, AnyVec kg, int has_norm, float eps, const float* rope_table, int rotary, int max_positions, unsigned char* cache,
                                int num_pages, int page_size, int nq, int nkv, int num_tokens) {
    const int heads = nq + 2 * nkv;
    const bool many = (long long)num_tokens * heads >= kManyHeads;
    if (many && (rotary == 0 || rotary == d) && (uintptr_t)qkv % 16 == 0 && (uintptr_t)q_out % 16 == 0 && (size_t)row_stride * sizeof(T) % 16 == 0 &&
        (size_t)q_stride * sizeof(T) % 16 == 0) {
        constexpr int P = sizeof(T) == 2 ? 2 : 1;
        const int per_warp = 512 / d * P;                            // heads a warp takes
        const long long row_warps = (long long)num_tokens * ((heads + per_warp - 1) / per_warp);
        const dim3 rows((unsigned)std::min<long long>((row_warps + kRowWarps - 1) / kRowWarps, 148 * kRowCtas));
#define CIB_KV4_ROWS(LV)                                                                                                                           \
    return launch_pdl(write_rows_kernel<T, LV, P>, rows, dim3(kRowWarps * 32), 0, stream, use_pdl, qkv, row_stride, q_out, q_stride, positions, slots, qg, kg,  \
                      has_norm, eps, rope_table, rotary > 0 ? 1 : 0, max_positions, cache, num_pages, page_size, nq, nkv, num_tokens)
        if (d == 64) CIB_KV4_ROWS(4);
        if (d == 128) CIB_KV4_ROWS(8);
        CIB_KV4_ROWS(16);
#undef CIB_KV4_ROWS
    }
    const long long warps = (long long)num_tokens * ((heads + (many ? 3 : 0)) / (many ? 4 : 1));
    const dim3 grid((unsigned)((warps + kWarps - 1) / kWarps));
#define CIB_KV4_WRITE(EV, HB)                                                                                                                      \
    return launch_pdl(write_lanes_kernel<T, EV, HB>, grid, dim3(kWarps * 32), 0, stream, use_pdl, qkv, row_stride, q_out, q_stride, positions, slots, qg, \
                      kg, has_norm, eps, rope_table, rotary, max_positions, cache, num_pages, page_size, nq, nkv, num_tokens)
    if (d == 64) { if (many) CIB_KV4_WRITE(2, 4); else CIB_KV4_WRITE(2, 1); }
    if (d == 128) { if (many) CIB_KV4_WRITE(4, 4); else CIB_KV4_WRITE(4, 1); }
    if (many) CIB_KV4_WRITE(8, 4); else CIB_KV4_WRITE(8, 1);
#undef CIB_KV4_WRITE
}

template <typename T>
static cudaError_t launch_read(int d, cudaStream_t stream, bool use_pdl, unsigned char* cache, int num_pages, int page_size, const int* slots, T* keys,
                               int key_stride, T* values, int value_stride, int nkv, int num_slots) {
    const bool many = (long long)num_slots * nkv >= kManyHeads;
    const long long warps = (long long)num_slots * ((nkv + (many ? 3 : 0)) / (many ? 4 : 1));
    const dim3 grid((unsigned)((warps + kWarps - 1) / kWarps));
#define CIB_KV4_READ(EV, HB)                                                                                                                      \
    return launch_pdl(read_lanes_kernel<T, EV, HB>, grid, dim3(kWarps * 32), 0, stream, use_pdl, cache, num_pages, page_size, slots, keys, key_stride,  \
                      values, value_stride, nkv, num_slots)
    if (d == 64) { if (many) CIB_KV4_READ(2, 4); else CIB_KV4_READ(2, 1); }
    if (d == 128) { if (many) CIB_KV4_READ(4, 4); else CIB_KV4_READ(4, 1); }
    if (many) CIB_KV4_READ(8, 4); else CIB_KV4_READ(8, 1);
#undef CIB_KV4_READ
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
    const int width = dtype == kF32 ? 4 : 2, lane_bytes = d / 32 * width < 16 ? d / 32 * width : 16;
    const bool lanes = (d == 64 || d == 128 || d == 256) && rotary % (d / 16) == 0 && (uintptr_t)rope_table % 16 == 0 && (uintptr_t)qkv % lane_bytes == 0 &&
                       (uintptr_t)q_out % lane_bytes == 0 && (size_t)row_stride * width % lane_bytes == 0 && (size_t)q_stride * width % lane_bytes == 0 &&
                       (long long)num_tokens * heads < (1ll << 31);
    if (lanes && dtype == kF32)
        e = kv4::launch_write<float>(d, stream, use_pdl != 0, (const float*)qkv, row_stride, (float*)q_out, q_stride, positions, slots, qg, kg, has_norm, eps, rope_table,
                                     rotary, max_positions, (unsigned char*)cache, num_pages, page_size, nq, nkv, num_tokens);
    else if (lanes)
        e = kv4::launch_write<__nv_bfloat16>(d, stream, use_pdl != 0, (const __nv_bfloat16*)qkv, row_stride, (__nv_bfloat16*)q_out, q_stride, positions, slots, qg, kg,
                                             has_norm, eps, rope_table, rotary, max_positions, (unsigned char*)cache, num_pages, page_size, nq, nkv, num_tokens);
    else if (dtype == kF32)
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
    const int width = dtype == kF32 ? 4 : 2, lane_bytes = d / 32 * width < 16 ? d / 32 * width : 16;
    const bool lanes = (d == 64 || d == 128 || d == 256) && (uintptr_t)keys % lane_bytes == 0 && (uintptr_t)values % lane_bytes == 0 &&
                       (size_t)key_stride * width % lane_bytes == 0 && (size_t)value_stride * width % lane_bytes == 0 && (long long)num_slots * nkv < (1ll << 31);
    if (lanes && dtype == kF32)
        e = kv4::launch_read<float>(d, stream, use_pdl != 0, (unsigned char*)cache, num_pages, page_size, slots, (float*)keys, key_stride, (float*)values, value_stride,
                                    nkv, num_slots);
    else if (lanes)
        e = kv4::launch_read<__nv_bfloat16>(d, stream, use_pdl != 0, (unsigned char*)cache, num_pages, page_size, slots, (__nv_bfloat16*)keys, key_stride,
                                            (__nv_bfloat16*)values, value_stride, nkv, num_slots);
    else if (dtype == kF32)
        e = launch_pdl(kv4::read_kernel<float>, grid, dim3(kv4::kWarps * 32), 0, stream, use_pdl != 0, (unsigned char*)cache, num_pages, page_size, slots,
                       (float*)keys, key_stride, (float*)values, value_stride, nkv, d);
    else
        e = launch_pdl(kv4::read_kernel<__nv_bfloat16>, grid, dim3(kv4::kWarps * 32), 0, stream, use_pdl != 0, (unsigned char*)cache, num_pages, page_size, slots,
                       (__nv_bfloat16*)keys, key_stride, (__nv_bfloat16*)values, value_stride, nkv, d);
    CIB_REQUIRE(e == cudaSuccess, "kv4_read: launch failed: %s", cudaGetErrorString(e));
    return 0;
}
