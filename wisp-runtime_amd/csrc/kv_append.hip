// Head norms, rotation and storing of new tokens in a paged K/V cache (paged.hpp), one launch for packed prompts and
// single decode tokens alike.
//
// For a head vector x of length D of a token at position p:
//     y = x * rsqrt(mean(x^2) + eps) * w                        (y = x without norm weights)
//     out[e] = y[e] cos[p][e] + s(e) y[e'] sin[p][e]   e < R     (e' the partner, s(e) -1 for a pair's first element)
//     out[e] = y[e]                                    e >= R
// in binary32, rounded once to the cache's type. Pairs are (i, i + R/2), or (2i, 2i + 1) interleaved. q heads go to qo,
// k heads to their page, v heads are copied. Positions follow from the lengths on the device: token j of sequence b,
// which brings n of its kv_len[b] positions, is at kv_len[b] - n + j.
//
// HBM-bound: each element is read once and written once. A lane holds 16 bytes (8 elements) of a head, so D/8 lanes
// share a head and a wave takes 512/D heads at a time; the sum of squares and the partner's values move between those
// lanes by DPP. A wave walks its token's head groups, the next group's load ahead of this one's stores. What hides the
// latencies is the number of waves: cos, sin and the norm weights stay packed, so that the kernel fits 64 registers and
// 8 waves a SIMD (with 85: 43 us for 6,976 tokens of 40 heads of 128, where 61 take 34.6 and, a wave a token, 31.3:
// 4.7 TB/s).
#include "paged.hpp"
#include "wisp_device.hpp"
#include "wisp_internal.hpp"

namespace wisp {

struct AppendArgs {
    const uint16_t *q, *k, *v;
    int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;  // token and head strides, elements
    const uint16_t *qw, *kw;                      // norm weights [D], both or neither
    float eps;
    const void *cos, *sin;  // [cs_rows][rot]
    int64_t cs_rows;
    int rot;
    const int *cu, *kv_len, *table;
    int width, B, T, hq, hk, per_wave, waves;  // head groups a wave takes, waves of a token
    PagedKV kv;
    uint16_t* qo;  // [T][hq][D]
};

template <bool F16>
__device__ __forceinline__ void widen8(const uint4 u, float* f) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = F16 ? half_lo_f(w[i]) : bf16_lo(w[i]);
        f[2 * i + 1] = F16 ? half_hi_f(w[i]) : bf16_hi(w[i]);
    }
}
template <bool F16>
__device__ __forceinline__ uint32_t round2(float lo, float hi) {
    if constexpr (F16) {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, h2{(_Float16)lo, (_Float16)hi});
    } else {
        return pack_bf16x2(lo, hi);
    }
}

// Sum over the lanes of a head (D/8 of them, consecutive), in every one of them.
template <int D>
__device__ __forceinline__ float head_sum(float v) {
    v += dpp_f<0xB1>(v);   // xor 1
    v += dpp_f<0x4E>(v);   // xor 2
    v += dpp_f<0x141>(v);  // row_half_mirror: the other four of eight
    if constexpr (D >= 128) v += dpp_f<0x140>(v);  // row_mirror: the other eight of a row
    if constexpr (D == 256) v = add_xor16(v);
    return v;
}
// The value of the lane that holds the other half of the head's pairs, rot/2 elements away (the whole head rotated).
template <int D>
__device__ __forceinline__ uint32_t other_half(uint32_t v) {
    if constexpr (D == 64) {  // xor 4: row_half_mirror, then each quad reversed
        const int m = __builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, true);
        return (uint32_t)__builtin_amdgcn_update_dpp(0, m, 0x1B, 0xF, 0xF, true);
    } else if constexpr (D == 128) {  // xor 8: row_ror:8
        return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xF, 0xF, true);
    } else {  // xor 16: the swap leaves the partner's value in one of its two results
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return (threadIdx.x & 16) ? r[0] : r[1];
    }
}

// ROT: 0 half pairs of a part of the head, 1 half pairs of the whole head, 2 interleaved
template <bool F16, int D, int ROT, bool CS32>
__global__ __launch_bounds__(256) void k_kv_append(const AppendArgs a) {
    constexpr bool INTER = ROT == 2;
    constexpr int LPH = D / 8, HPW = 64 / LPH;  // lanes per head, heads per wave
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hl = lane & (LPH - 1), hw = lane / LPH, e0 = 8 * hl;
    const int heads = a.hq + 2 * a.hk, groups = (heads + HPW - 1) / HPW;
    const uint32_t id = (blockIdx.y * gridDim.x + blockIdx.x) * 4u + wv;
    const int tok = (int)(id / (uint32_t)a.waves), g0 = (int)(id - (uint32_t)tok * a.waves) * a.per_wave;
    if (tok >= a.T) return;

    auto load = [&](int g) {
        const int h = min(g * HPW + hw, heads - 1);
        const uint16_t* x = h < a.hq          ? a.q + tok * a.q_ts + h * a.q_hs
                            : h < a.hq + a.hk ? a.k + tok * a.k_ts + (h - a.hq) * a.k_hs
                                              : a.v + tok * a.v_ts + (h - a.hq - a.hk) * a.v_hs;
        return *reinterpret_cast<const uint4*>(x + e0);
    };
    uint4 next = load(g0);  // (before it is known whether the row belongs to a sequence: the rows of q, k and v are all there)

    // the token's sequence: the one whose range ends past it first; 64 ends are looked at together
    int b = 0, t1 = 0, len = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const int i = min(b0 + lane, a.B - 1), e = a.cu[i + 1], n = a.kv_len[i];
        const uint64_t past = __ballot(b0 + lane < a.B && e > tok);
        if (past) {
            const int w = __builtin_ctzll(past);
            b = b0 + w;
            t1 = min(__builtin_amdgcn_readlane(e, w), a.T);
            len = __builtin_amdgcn_readlane(n, w);
            break;
        }
    }
    if (t1 == 0 || scalar_at(a.cu, 0) > tok) return;  // a row that belongs to no sequence
    const int pos = len - (t1 - tok);
    bool bad = pos < 0 || pos >= a.cs_rows;
    const int64_t at = page_offset(a.kv, a.table + (int64_t)b * a.width, a.width, bad ? 0 : pos, bad);

    const bool rotated = ROT == 1 || e0 < a.rot;  // rot is a multiple of 16: a lane's eight elements are rotated or not together
    const int half = a.rot >> 1;
    const bool first = e0 < half;
    const int partner = rotated && !INTER ? (first ? hl + half / 8 : hl - half / 8) : hl;
    // the lane's cos and sin, as they are stored (pairs of the type, or binary32)
    constexpr int CN = CS32 ? 2 : 1;
    uint4 cs[CN], sn[CN];
    {
        const int64_t r = bad ? 0 : (int64_t)pos * a.rot + (rotated ? e0 : 0);
#pragma unroll
        for (int i = 0; i < CN; ++i) {
            cs[i] = *(reinterpret_cast<const uint4*>((const uint8_t*)a.cos + r * (CS32 ? 4 : 2)) + i);
            sn[i] = *(reinterpret_cast<const uint4*>((const uint8_t*)a.sin + r * (CS32 ? 4 : 2)) + i);
        }
    }
    const float sign = first ? -1.f : 1.f;  // of the partner's term
    const bool norm = a.qw != nullptr;
    uint4 w[2] = {};  // the lane's norm weights, of q and of k
    if (norm) {
        w[0] = *reinterpret_cast<const uint4*>(a.qw + e0);
        w[1] = *reinterpret_cast<const uint4*>(a.kw + e0);
    }
    const float nan = __int_as_float(0x7FC00000);
    const int g1 = min(g0 + a.per_wave, groups);
    for (int g = g0; g < g1; ++g) {
        const int h = g * HPW + hw;
        const bool is_q = h < a.hq, is_k = !is_q && h < a.hq + a.hk;
        const bool have = h < heads;
        uint4 res = next;
        if (g + 1 < g1) next = load(g + 1);  // ahead of this group's stores
        if (g * HPW < a.hq + a.hk) {  // (values are copied)
            float x[8];
            widen8<F16>(res, x);
            if (norm) {
                float ss = 0.f, f[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(x[i], x[i], ss);
                const float rs = rsqrtf(head_sum<D>(ss) * (1.f / D) + a.eps);
                widen8<F16>(is_q ? w[0] : w[1], f);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = x[i] * rs * f[i];
            }
            float y[8];
            float c[8], sv[8];
            if constexpr (CS32) {
                const uint32_t cw[8] = {cs[0].x, cs[0].y, cs[0].z, cs[0].w, cs[1].x, cs[1].y, cs[1].z, cs[1].w};
                const uint32_t sw[8] = {sn[0].x, sn[0].y, sn[0].z, sn[0].w, sn[1].x, sn[1].y, sn[1].z, sn[1].w};
#pragma unroll
                for (int i = 0; i < 8; ++i) c[i] = __uint_as_float(cw[i]), sv[i] = __uint_as_float(sw[i]);
            } else {
                widen8<F16>(cs[0], c);
                widen8<F16>(sn[0], sv);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float t;
                if constexpr (INTER) t = i & 1 ? x[i ^ 1] : -x[i ^ 1];
                else if constexpr (ROT == 1) t = sign * __uint_as_float(other_half<D>(__float_as_uint(x[i])));
                else t = sign * __shfl(x[i], hw * LPH + partner, 64);
                // unrotated elements: y = x exactly, whatever the partner holds
                y[i] = rotated ? __builtin_fmaf(x[i], c[i], t * sv[i]) : x[i];
            }
            if (is_q || is_k) {
                res = make_uint4(round2<F16>(y[0], y[1]), round2<F16>(y[2], y[3]), round2<F16>(y[4], y[5]),
                                 round2<F16>(y[6], y[7]));
                if (bad) {
                    const uint32_t n2 = round2<F16>(nan, nan);
                    res = make_uint4(n2, n2, n2, n2);
                }
            }
        }
        if (is_q) {
            *reinterpret_cast<uint4*>(a.qo + ((int64_t)tok * a.hq + h) * D + e0) = res;
        } else if (have && !bad) {
            uint8_t* base = is_k ? a.kv.kc + (h - a.hq) * a.kv.hs : a.kv.vc + (h - a.hq - a.hk) * a.kv.hs;
            *reinterpret_cast<uint4*>(base + at + 2 * e0) = res;
        }
    }
}

template <bool F16, int D>
static void launch_append(const AppendArgs& a, int rot, bool cs32, dim3 grid, hipStream_t st) {
#define WISP_APPEND(R, C) \
    if (rot == R && cs32 == C) hipLaunchKernelGGL((k_kv_append<F16, D, R, C>), grid, dim3(256), 0, st, a);
    WISP_APPEND(0, false)
    WISP_APPEND(0, true)
    WISP_APPEND(1, false)
    WISP_APPEND(1, true)
    WISP_APPEND(2, false)
    WISP_APPEND(2, true)
#undef WISP_APPEND
}

}  // namespace wisp

using namespace wisp;

extern "C" int wisp_kv_append(const void* q, int64_t q_ts, int64_t q_hs, const void* k, int64_t k_ts, int64_t k_hs,
                              const void* v, int64_t v_ts, int64_t v_hs, const void* q_norm_w, const void* k_norm_w,
                              float eps, const void* cos, const void* sin, int64_t cs_rows, int rot, int cs_dtype,
                              int interleaved, const int32_t* cu, const int32_t* kv_len, const int32_t* table, int width,
                              int B, int64_t T, int hq, int hk, int d, int dtype, void* kc, void* vc, int64_t pages,
                              int page, int64_t page_stride, int64_t head_stride, int64_t row_stride, void* qo,
                              void* stream) {
    clear_error();
    if (int rc = check_paged(kc, vc, pages, page, page_stride, head_stride, row_stride, width, B, hq, hk, d, dtype)) return rc;
    if (T < 0 || T > (1 << 30)) return fail_inval("T must be in [0, 2^30]");
    if (rot < 16 || rot > d || rot % 16) return fail_inval("rot must be a multiple of 16 in [16, d]");
    if (cs_rows < 1) return fail_inval("cos and sin need at least one row");
    if (cs_dtype != dtype && cs_dtype != WISP_DT_F32) return fail_inval("cos and sin must be float32 or of q's type");
    if (!q_norm_w != !k_norm_w) return fail_inval("norm weights: both or neither");
    if (T == 0) return WISP_OK;
    if (!q || !k || !v || !cos || !sin || !cu || !kv_len || !table || !qo) return fail_inval("null pointer");
    for (const void* p : {q, k, v, cos, sin, q_norm_w, k_norm_w, (const void*)qo})
        if (!aligned(p, 16)) {
            set_error("q, k, v, the norm weights, cos, sin and qo must be 16-byte aligned");
            return WISP_EALIGN;
        }
    for (int64_t s : {q_ts, q_hs, k_ts, k_hs, v_ts, v_hs})
        if (s % 8) {
            set_error("the token and head strides of q, k and v must be multiples of 8 elements");
            return WISP_EALIGN;
        }
    const int hpw = 512 / d, groups = (hq + 2 * hk + hpw - 1) / hpw;
    // Few tokens: a wave per head group, so that the call has as many requests in flight as it can. Enough for a wave each
    // to fill most of the 8,192 that the card holds: a wave walks all its token's groups and finds cos, sin and the page
    // once. Between them, two to three times the card's waves. Groups a wave 1, 2, 4 and all, inputs not in the cache: 10 groups
    // a token (40 heads of 128, 80 of 64 or 20 of 256 alike) 500 tokens 5.7, 6.0, 7.3, 10.9 us, 1,500 12.7, 11.5, 12.4, 17.9,
    // 4,500 29.6, 25.0, 26.2, 26.1, 6,143 38.3, 32.1, 34.0, 31.7, 20,000 116, 91, 91, 92; 3 groups (12 heads of 128) 4,500 12.1,
    // 12.1, -, 11.1, 8,000 17.7, 17.1, -, 16.0; 20 groups (80 heads of 128) 8,000 92, 74, 73, 80: so wide, four would be better.
    int per_wave = 1;
    if (T >= 6144) per_wave = groups;
    while (per_wave < groups && T * ((groups + 2 * per_wave - 1) / (2 * per_wave)) >= 16384) per_wave *= 2;
    const int waves = (groups + per_wave - 1) / per_wave;
    AppendArgs a{(const uint16_t*)q, (const uint16_t*)k, (const uint16_t*)v, q_ts, q_hs, k_ts, k_hs, v_ts, v_hs,
                 (const uint16_t*)q_norm_w, (const uint16_t*)k_norm_w, eps, cos, sin, cs_rows, rot, cu, kv_len, table,
                 width, B, (int)T, hq, hk, per_wave, waves, paged_kv(kc, vc, pages, page, page_stride, head_stride, row_stride),
                 (uint16_t*)qo};
    // in two dimensions: one holds fewer than 2^32 threads, 2^24 of these workgroups (what is past them is cut off unseen)
    const int64_t blocks = (T * waves + 3) / 4, row = 1 << 23;
    const dim3 grid((unsigned)(blocks < row ? blocks : row), (unsigned)((blocks + row - 1) / row));
    hipStream_t st = (hipStream_t)stream;
    const bool cs32 = cs_dtype == WISP_DT_F32;
    const int in = interleaved ? 2 : rot == d ? 1 : 0;
    if (dtype == WISP_DT_F16) {
        if (d == 64) launch_append<true, 64>(a, in, cs32, grid, st);
        else if (d == 128) launch_append<true, 128>(a, in, cs32, grid, st);
        else launch_append<true, 256>(a, in, cs32, grid, st);
    } else {
        if (d == 64) launch_append<false, 64>(a, in, cs32, grid, st);
        else if (d == 128) launch_append<false, 128>(a, in, cs32, grid, st);
        else launch_append<false, 256>(a, in, cs32, grid, st);
    }
    return check_launch("k_kv_append");
}
