// RMSNorm of every query and key head with the position rotation in the same
// pass, and with the append of the rotated K and of V to the paged cache.
//
// Mathematics, per head row x[0 .. D): n_e = x_e r w_e, r = 1 / sqrt(mean x^2 +
// eps); each rotated pair (a, b) of n becomes (a c - b s, a s + b c), (s, c) =
// sin, cos of position * inv_freqs[i].  Everything is f32 from the load to the
// one rounding of the store; the angle is the exact product (f64), reduced by
// multiples of pi/2 there, so positions of 10^5 lose nothing.
//
// Bound by bytes: each row is read once and written once.  A lane holds two
// 16-byte chunks of a head that contain both members of its pairs, so neither
// the rotation nor the store exchanges anything between lanes and the mean
// takes log2(lanes per head) exchanges.  A workgroup first requests its first
// chunks, then builds the (cos, sin) table of its rows in LDS while they are on
// their way: D / 2 angles per row serve all heads.
#include "common.hpp"
#include "kv_slot.hpp"

#include <algorithm>
#include <initializer_list>

namespace fellm {
namespace {

// sin and cos of pos * f.  pi/2 in two f64 parts (the first exact in 53 bits);
// the polynomials are least-maximum fits on |r| <= pi/4 (sin r = r + r^3 P(r^2),
// cos r = 1 - r^2 / 2 + r^4 Q(r^2)), off by at most 4.3e-8 and 7.3e-8 in f32.
__device__ __forceinline__ void angle_sincos(uint32_t pos, float f, float &s, float &c) {
    const double t = (double)pos * (double)f;
    const double k = rint(t * 0.63661977236758134308);
    double r = fma(-k, 1.57079632679489661923, t);
    r = fma(-k, 6.123233995736766e-17, r);
    const uint32_t quad = (uint32_t)(int64_t)k & 3;
    const float x = (float)r, z = x * x;
    float p = fmaf(2.71831163445313e-06f, z, -0.0001983933470910415f);
    p = fmaf(p, z, 0.008333329111337662f);
    p = fmaf(p, z, -0.1666666716337204f);
    const float sn = fmaf(x * z, p, x);
    float q = fmaf(2.443845005473122e-05f, z, -0.001388736767694354f);
    q = fmaf(q, z, 0.04166664555668831f);
    const float cs = fmaf(z * z, q, fmaf(-0.5f, z, 1.0f));
    const float a = quad & 1 ? cs : sn, b = quad & 1 ? sn : cs;
    s = quad & 2 ? -a : a;
    c = (quad + 1) & 2 ? -b : b;
}

struct NormArgs {
    const void *q, *k, *v;
    void *q_out, *k_out;
    uint32_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride;  // elements per row
    uint32_t n_q, n_k, rows, head_dim, rope_dim, pairing;
    const float *q_weight, *k_weight, *inv_freqs;
    const uint32_t *positions;  // null: position0 + row
    uint32_t position0;
    float eps;
    // cache append (kv.arena null: none)
    KvDev kv;
    const uint32_t *kv_positions;
    const uint32_t *sequences;  // block table row of each row; null: the row itself
    uint32_t *err_flag;
    uint32_t head_split;
};

// The K row of the cache slot of `row`, or ~0 (and the error flag) outside the cache.
__device__ __forceinline__ uint64_t row_slot(const NormArgs &a, uint32_t row, bool report) {
    const uint64_t off = kv_slot_offset(a.kv, a.sequences ? a.sequences[row] : row, a.kv_positions[row]);
    if (off == ~0ull && report && a.err_flag) *a.err_flag = 1;
    return off;
}
__device__ __forceinline__ uint32_t row_position(const NormArgs &a, uint32_t row) {
    return a.positions ? a.positions[row] : a.position0 + row;
}

constexpr uint32_t kNormThreads = 256;
constexpr uint64_t kMaxGroups = 0xffffffffull / kNormThreads;  // a launch has fewer than 2^32 threads

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
// V outputs, rounded by the hardware's conversion and stored in one access.
template <typename A, bool STREAM, int V>
__device__ __forceinline__ void put_row(typename A::T *p, const float (&v)[V]) {
    Pack<typename A::T, V> pk;
#pragma unroll
    for (int i = 0; i < V; ++i) pk.v[i] = HwStore<A>::type::store(v[i]);
    if constexpr (STREAM) __builtin_nontemporal_store(__builtin_bit_cast(u32x4_t, pk), reinterpret_cast<u32x4_t *>(p));
    else store_f32<A, V>(p, v);
}

// A: activations, C: cache elements, L: lanes per head, R: rows per workgroup,
// STREAM: non-temporal rows.
// Measured, kernel alone (32/4 heads of 128): 16384 bf16 rows out of one
// projection 70 -> 55 us (5.5 TB/s) with the norm weights in LDS rather than in
// registers, one head in flight per lane group and streamed rows; f32 rows gain
// from two heads in flight, with the weights in registers (half as many as 16-bit
// chunks need): 4000 rows 27.4 against 34.8 us; streaming gains them only what
// the cache cannot hold (16000 rows 121 -> 114 us, 4000 rows 27.4 -> 31.9).
template <typename A, typename C, int L, int R, bool STREAM, bool WRITE>
__global__ __launch_bounds__(kNormThreads) void qk_norm_kernel(NormArgs a) {
    using T = typename A::T;
    constexpr int V = 16 / sizeof(T);
    constexpr bool REG = sizeof(T) == 4;  // norm weights in registers
    constexpr int U = REG ? 2 : 1;        // heads that a lane group has in flight
    constexpr uint32_t GROUPS = kNormThreads / L;
    extern __shared__ __align__(16) float table[];  // per row: rope_dim / 2 cos, then as many sin
    const uint32_t half = a.rope_dim / 2;
    const uint32_t row0 = blockIdx.x / a.head_split * R, part = blockIdx.x % a.head_split;
    const uint32_t nrows = min((uint32_t)R, a.rows - row0);
    // this workgroup's heads of each row: q, k and (append) v heads in one numbering
    const uint32_t all = a.n_q + a.n_k + (WRITE ? a.n_k : 0);
    const uint32_t per = (all + a.head_split - 1) / a.head_split;
    const uint32_t h0 = part * per, heads = min(per, all - min(all, h0));
    const uint32_t total = nrows * heads;

    // this lane's chunks of a head, and the index of its first pair (~0: not rotated)
    const uint32_t l = threadIdx.x % L, slot0 = threadIdx.x / L;
    const bool active = l * 2 * V < a.head_dim;
    uint32_t ca, cb, pair = ~0u;
    if (a.pairing == 1) {
        if (l * V < half) ca = l * V, cb = half + l * V, pair = l * V;
        else ca = a.rope_dim + (l * V - half) * 2, cb = ca + V;
    } else {
        const uint32_t off = a.pairing == 2 ? a.head_dim - a.rope_dim : 0;
        ca = l * 2 * V, cb = ca + V;
        if (ca >= off && ca - off < a.rope_dim) pair = (ca - off) / 2;
    }

    if (!active) ca = cb = 0;

    using P = Pack<T, V>;
    P xa[U], xb[U];
    uint32_t rr[U], hh[U];
    auto fetch = [&](uint32_t slot) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t s = slot + u * GROUPS;
            rr[u] = R == 1 ? 0 : s / heads;
            hh[u] = h0 + (R == 1 ? s : s % heads);
            if (s < total && active) {
                const uint32_t h = hh[u];
                const size_t row = row0 + rr[u];
                const T *src = h < a.n_q ? static_cast<const T *>(a.q) + row * a.q_stride + h * a.head_dim
                               : h < a.n_q + a.n_k
                                   ? static_cast<const T *>(a.k) + row * a.k_stride + (h - a.n_q) * a.head_dim
                                   : static_cast<const T *>(a.v) + row * a.v_stride + (h - a.n_q - a.n_k) * a.head_dim;
                if constexpr (STREAM) {
                    xa[u] = __builtin_bit_cast(P, __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(src + ca)));
                    xb[u] = __builtin_bit_cast(P, __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(src + cb)));
                } else {
                    xa[u] = *reinterpret_cast<const P *>(src + ca);
                    xb[u] = *reinterpret_cast<const P *>(src + cb);
                }
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) xa[u].v[e] = xb[u].v[e] = T{};
            }
        }
    };
    fetch(slot0);
    [[maybe_unused]] float qwa[V], qwb[V], kwa[V], kwb[V];
    [[maybe_unused]] float *weights = table + R * a.rope_dim;  // of q, then of k
    if constexpr (REG) {
        load_f32<F32, V>(a.q_weight + ca, qwa);
        load_f32<F32, V>(a.q_weight + cb, qwb);
        load_f32<F32, V>(a.k_weight + ca, kwa);
        load_f32<F32, V>(a.k_weight + cb, kwb);
    } else {
        for (uint32_t i = threadIdx.x; i < 2 * a.head_dim; i += kNormThreads)
            weights[i] = i < a.head_dim ? a.q_weight[i] : a.k_weight[i - a.head_dim];
    }
    for (uint32_t i = threadIdx.x; i < nrows * half; i += kNormThreads) {
        const uint32_t r = R == 1 ? 0 : i / half, e = R == 1 ? i : i % half;
        float s, c;
        angle_sincos(row_position(a, row0 + r), a.inv_freqs[e], s, c);
        table[r * a.rope_dim + e] = c;
        table[r * a.rope_dim + half + e] = s;
    }
    __syncthreads();
    const float inv_d = 1.0f / (float)a.head_dim;
    for (uint32_t slot = slot0; slot < total; slot += U * GROUPS) {
        float ya[U][V], yb[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < V; ++e) ya[u][e] = A::load(xa[u].v[e]), yb[u][e] = A::load(xb[u].v[e]);
        uint32_t srr[U], shh[U];
#pragma unroll
        for (int u = 0; u < U; ++u) srr[u] = rr[u], shh[u] = hh[u];
        if (slot + U * GROUPS < total) fetch(slot + U * GROUPS);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t h = shh[u], row = row0 + srr[u];
            const bool here = slot + u * GROUPS < total && active;
            const bool is_q = h < a.n_q, is_v = WRITE && h >= a.n_q + a.n_k;
            if (!is_v) {
                float ss = 0.0f;
#pragma unroll
                for (int e = 0; e < V; ++e) ss = fmaf(ya[u][e], ya[u][e], fmaf(yb[u][e], yb[u][e], ss));
#pragma unroll
                for (int o = L / 2; o; o >>= 1) ss += __shfl_xor(ss, o);
                const float r = __builtin_amdgcn_rsqf(fmaf(ss, inv_d, a.eps));
                float wa[V], wb[V];
                if constexpr (REG) {
#pragma unroll
                    for (int e = 0; e < V; ++e) wa[e] = is_q ? qwa[e] : kwa[e], wb[e] = is_q ? qwb[e] : kwb[e];
                } else {
                    const float *w = weights + (is_q ? 0 : a.head_dim);
                    load_f32<F32, V>(w + ca, wa);
                    load_f32<F32, V>(w + cb, wb);
                }
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    ya[u][e] = ya[u][e] * r * wa[e];
                    yb[u][e] = yb[u][e] * r * wb[e];
                }
                if (pair != ~0u && here) {
                    float c[V], s[V];
                    const float *t = table + srr[u] * a.rope_dim + pair;
                    load_f32<F32, V>(t, c);
                    load_f32<F32, V>(t + half, s);
                    if (a.pairing == 1) {
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            const float x = ya[u][e], y = yb[u][e];
                            ya[u][e] = fmaf(x, c[e], -(y * s[e]));
                            yb[u][e] = fmaf(x, s[e], y * c[e]);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < V; e += 2) {
                            const float x = ya[u][e], y = ya[u][e + 1], x2 = yb[u][e], y2 = yb[u][e + 1];
                            ya[u][e] = fmaf(x, c[e / 2], -(y * s[e / 2]));
                            ya[u][e + 1] = fmaf(x, s[e / 2], y * c[e / 2]);
                            yb[u][e] = fmaf(x2, c[(e + V) / 2], -(y2 * s[(e + V) / 2]));
                            yb[u][e + 1] = fmaf(x2, s[(e + V) / 2], y2 * c[(e + V) / 2]);
                        }
                    }
                }
            }
            if (!here) continue;
            if (is_q) {
                T *dst = static_cast<T *>(a.q_out) + (size_t)row * a.q_out_stride + h * a.head_dim;
                put_row<A, STREAM>(dst + ca, ya[u]);
                put_row<A, STREAM>(dst + cb, yb[u]);
                continue;
            }
            const uint32_t kh = h - a.n_q - (is_v ? a.n_k : 0);
            if (!is_v && a.k_out) {
                T *dst = static_cast<T *>(a.k_out) + (size_t)row * a.k_out_stride + kh * a.head_dim;
                put_row<A, STREAM>(dst + ca, ya[u]);
                put_row<A, STREAM>(dst + cb, yb[u]);
            }
            if constexpr (WRITE) {
                const uint64_t off = row_slot(a, row, true);
                if (off != ~0ull) {
                    typename C::T *dst = reinterpret_cast<typename C::T *>(a.kv.arena + off) +
                                         (is_v ? (size_t)a.kv.block_size * a.kv.stride : 0) + kh * a.head_dim;
                    store_f32<C, V>(dst + ca, ya[u]);
                    store_f32<C, V>(dst + cb, yb[u]);
                }
            }
        }
    }
}

// Any head size and alignment: one wavefront per (row, head), a pair (or an
// unrotated element) per lane and step.  Both members of a pair are read and
// written by the same lane, and every read of the sum comes before any write.
template <typename A, typename C, bool WRITE>
__global__ __launch_bounds__(kNormThreads) void qk_norm_any_kernel(NormArgs a) {
    using T = typename A::T;
    const uint32_t lane = threadIdx.x % kWave;
    const uint32_t all = a.n_q + a.n_k + (WRITE ? a.n_k : 0);
    const uint64_t id = (uint64_t)blockIdx.x * (kNormThreads / kWave) + threadIdx.x / kWave;
    if (id >= (uint64_t)a.rows * all) return;
    const uint32_t row = (uint32_t)(id / all), h = (uint32_t)(id % all);
    const bool is_q = h < a.n_q, is_v = h >= a.n_q + a.n_k;
    const uint32_t kh = is_q ? 0 : h - a.n_q - (is_v ? a.n_k : 0);
    const T *src = is_q ? static_cast<const T *>(a.q) + (size_t)row * a.q_stride + (size_t)h * a.head_dim
                        : is_v ? static_cast<const T *>(a.v) + (size_t)row * a.v_stride + (size_t)kh * a.head_dim
                               : static_cast<const T *>(a.k) + (size_t)row * a.k_stride + (size_t)kh * a.head_dim;
    const float *w = is_q ? a.q_weight : a.k_weight;
    T *dst = nullptr;
    if (is_q) dst = static_cast<T *>(a.q_out) + (size_t)row * a.q_out_stride + (size_t)h * a.head_dim;
    else if (!is_v && a.k_out) dst = static_cast<T *>(a.k_out) + (size_t)row * a.k_out_stride + (size_t)kh * a.head_dim;
    typename C::T *slot = nullptr;
    if (WRITE && !is_q) {
        const uint64_t off = row_slot(a, row, lane == 0);
        if (off != ~0ull)
            slot = reinterpret_cast<typename C::T *>(a.kv.arena + off) + (is_v ? (size_t)a.kv.block_size * a.kv.stride : 0) +
                   (size_t)kh * a.head_dim;
    }
    auto put = [&](uint32_t e, float v) {
        if (dst) dst[e] = A::store(v);
        if (slot) slot[e] = C::store(v);
    };
    if (is_v) {
        for (uint32_t e = lane; e < a.head_dim; e += kWave) put(e, A::load(src[e]));
        return;
    }
    float ss = 0.0f;
    for (uint32_t e = lane; e < a.head_dim; e += kWave) {
        const float x = A::load(src[e]);
        ss = fmaf(x, x, ss);
    }
    const float r = __builtin_amdgcn_rsqf(fmaf(wave_sum(ss), 1.0f / (float)a.head_dim, a.eps));
    const uint32_t half = a.rope_dim / 2, lo = a.pairing == 2 ? a.head_dim - a.rope_dim : 0;
    const uint32_t pos = row_position(a, row);
    for (uint32_t i = lane; i < half; i += kWave) {
        const uint32_t ea = a.pairing == 1 ? i : lo + 2 * i, eb = a.pairing == 1 ? i + half : ea + 1;
        float s, c;
        angle_sincos(pos, a.inv_freqs[i], s, c);
        const float x = A::load(src[ea]) * r * w[ea], y = A::load(src[eb]) * r * w[eb];
        put(ea, fmaf(x, c, -(y * s)));
        put(eb, fmaf(x, s, y * c));
    }
    for (uint32_t i = lane; i < a.head_dim - a.rope_dim; i += kWave) {
        const uint32_t e = i + (a.pairing == 2 ? 0 : a.rope_dim);
        put(e, A::load(src[e]) * r * w[e]);
    }
}

template <typename A, typename C, bool WRITE>
int launch_norm(NormArgs a, hipStream_t st) {
    constexpr uint32_t V = 16 / sizeof(typename A::T);
    const uint32_t all = a.n_q + a.n_k + (WRITE ? a.n_k : 0);
    bool vec = a.head_dim % (2 * V) == 0 && a.rope_dim % (2 * V) == 0 && a.head_dim <= kWave / 2 * 2 * V;
    for (const void *p : {a.q, a.k, a.v, (const void *)a.q_out, (const void *)a.k_out, (const void *)a.q_weight,
                          (const void *)a.k_weight, (const void *)a.kv.arena})
        vec = vec && aligned_to(p, 16);
    for (uint32_t s : {a.q_stride, a.k_stride, a.v_stride, a.q_out_stride, a.k_out_stride}) vec = vec && s % V == 0;
    if (WRITE) vec = vec && a.kv.block_bytes % 16 == 0;
    if (!vec) {
        const uint64_t grid = ((uint64_t)a.rows * all + kNormThreads / kWave - 1) / (kNormThreads / kWave);
        if (grid > kMaxGroups) return FELLM_ERR_SHAPE;
        FELLM_LAUNCH((qk_norm_any_kernel<A, C, WRITE>), dim3((uint32_t)grid), dim3(kNormThreads), 0, st, a);
        return launch_status();
    }
    auto go = [&]<int L, int R, bool STREAM>() {
        const uint32_t groups = (a.rows + R - 1) / R;
        // few rows: a row's heads over several workgroups
        const uint32_t most = std::max(1u, all / (kNormThreads / L));
        a.head_split = groups >= 256 ? 1 : std::min(most, std::max(1u, 512 / groups));
        if ((uint64_t)groups * a.head_split > kMaxGroups) return (int)FELLM_ERR_SHAPE;
        FELLM_LAUNCH((qk_norm_kernel<A, C, L, R, STREAM, WRITE>), dim3(groups * a.head_split), dim3(kNormThreads),
                     ((size_t)R * a.rope_dim + (V == 4 ? 0 : 2 * a.head_dim)) * sizeof(float), st, a);
        return launch_status();
    };
    auto rows = [&]<int L>() {
        // (rows and their outputs; 256 MB is what the last-level cache holds)
        const bool stream = V == 8 || (uint64_t)a.rows * 2 * all * a.head_dim * 4 > (256u << 20);
        if (a.rows < 2048) return go.template operator()<L, 1, V == 8>();
        return stream ? go.template operator()<L, 4, true>() : go.template operator()<L, 4, V == 8>();
    };
    const uint32_t lanes = a.head_dim / (2 * V);
    if (lanes <= 4) return rows.template operator()<4>();
    if (lanes <= 8) return rows.template operator()<8>();
    if (lanes <= 16) return rows.template operator()<16>();
    return rows.template operator()<32>();
}

int check_norm(const NormArgs &a) {
    if (int rc = check_rope_shape(a.head_dim, a.rope_dim, a.pairing)) return rc;
    if (!a.n_q || !a.n_k) return FELLM_ERR_SHAPE;
    const uint64_t qw = (uint64_t)a.n_q * a.head_dim, kw = (uint64_t)a.n_k * a.head_dim;
    if (qw > 0x7fffffffull || kw > 0x7fffffffull) return FELLM_ERR_SHAPE;
    if (a.q_stride < qw || a.q_out_stride < qw || a.k_stride < kw || (a.k_out && a.k_out_stride < kw)) return FELLM_ERR_SHAPE;
    if (a.kv.arena && (a.v_stride < kw || a.kv.stride != kw)) return FELLM_ERR_SHAPE;
    // in place only element for element
    if (a.q_out == a.q && a.q_out_stride != a.q_stride) return FELLM_ERR_SHAPE;
    if (a.k_out == a.k && a.k_out_stride != a.k_stride) return FELLM_ERR_SHAPE;
    return FELLM_OK;
}

}  // namespace
}  // namespace fellm

extern "C" int fellm_rocm_qk_norm_rope(const void *q, uint32_t q_stride, void *q_out, uint32_t q_out_stride,
                                       uint32_t n_q_heads, const void *k, uint32_t k_stride, void *k_out,
                                       uint32_t k_out_stride, uint32_t n_kv_heads, uint32_t act_dtype, uint32_t rows,
                                       uint32_t head_dim, uint32_t rope_dim, uint32_t pairing, const float *q_weight,
                                       const float *k_weight, float eps, const float *inv_freqs,
                                       const uint32_t *positions, uint32_t position0, void *stream) {
    using namespace fellm;
    if (rows == 0) return FELLM_OK;
    if (!q || !q_out || !k || !k_out || !q_weight || !k_weight || (rope_dim && !inv_freqs)) return FELLM_ERR_ARITY;
    NormArgs a{};
    a.q = q, a.k = k, a.q_out = q_out, a.k_out = k_out;
    a.q_stride = q_stride, a.k_stride = k_stride, a.q_out_stride = q_out_stride, a.k_out_stride = k_out_stride;
    a.n_q = n_q_heads, a.n_k = n_kv_heads, a.rows = rows;
    a.head_dim = head_dim, a.rope_dim = rope_dim, a.pairing = pairing;
    a.q_weight = q_weight, a.k_weight = k_weight, a.eps = eps, a.inv_freqs = inv_freqs;
    a.positions = positions, a.position0 = position0;
    if (int rc = check_norm(a)) return rc;
    return dispatch_act(act_dtype, [&]<typename A>() -> int { return launch_norm<A, F16, false>(a, as_stream(stream)); });
}

extern "C" int fellm_rocm_qk_norm_rope_kv_write(const void *q, uint32_t q_stride, void *q_out, uint32_t q_out_stride,
                                                uint32_t n_q_heads, const void *k, uint32_t k_stride, void *k_out,
                                                const void *v, uint32_t v_stride, uint32_t n_kv_heads,
                                                uint32_t act_dtype, uint32_t rows, uint32_t head_dim, uint32_t rope_dim,
                                                uint32_t pairing, const float *q_weight, const float *k_weight,
                                                float eps, const float *inv_freqs, const uint32_t *rope_positions,
                                                const uint32_t *kv_positions, const uint32_t *sequences,
                                                const FellmRocmPagedKv *kvp, uint32_t *err_flag, void *stream) {
    using namespace fellm;
    if (rows == 0) return FELLM_OK;
    if (!q || !q_out || !k || !v || !q_weight || !k_weight || !kv_positions || !kvp || (rope_dim && !inv_freqs))
        return FELLM_ERR_ARITY;
    NormArgs a{};
    a.q = q, a.k = k, a.v = v, a.q_out = q_out, a.k_out = k_out;
    a.q_stride = q_stride, a.k_stride = k_stride, a.v_stride = v_stride, a.q_out_stride = q_out_stride;
    a.n_q = n_q_heads, a.n_k = n_kv_heads, a.rows = rows;
    a.k_out_stride = n_kv_heads * head_dim;
    a.head_dim = head_dim, a.rope_dim = rope_dim, a.pairing = pairing;
    a.q_weight = q_weight, a.k_weight = k_weight, a.eps = eps, a.inv_freqs = inv_freqs;
    a.positions = rope_positions ? rope_positions : kv_positions;
    a.kv_positions = kv_positions, a.sequences = sequences, a.err_flag = err_flag;
    if (!make_kv(kvp, a.kv)) return FELLM_ERR_SHAPE;
    if (int rc = check_norm(a)) return rc;
    return dispatch_act(act_dtype, [&]<typename A>() -> int {
        return dispatch_cache(kvp->kv_dtype, [&]<typename C>() -> int { return launch_norm<A, C, true>(a, as_stream(stream)); });
    });
}
