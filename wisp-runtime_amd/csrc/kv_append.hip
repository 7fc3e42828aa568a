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
// lanes. A wave walks some of its token's head groups with the token's cos and sin in registers.
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
    int width, B, T, hq, hk, per_wave;  // per_wave: head groups a wave takes
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

template <bool F16, int D, bool INTER, bool CS32>
__global__ __launch_bounds__(256) void k_kv_append(const AppendArgs a) {
    constexpr int LPH = D / 8, HPW = 64 / LPH;  // lanes per head, heads per wave
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hl = lane & (LPH - 1), hw = lane / LPH, e0 = 8 * hl;
    const int heads = a.hq + 2 * a.hk, groups = (heads + HPW - 1) / HPW;
    const int waves = (groups + a.per_wave - 1) / a.per_wave;  // per token
    const int64_t id = (int64_t)blockIdx.x * 4 + wv;
    const int tok = (int)(id / waves), g0 = (int)(id - (int64_t)tok * waves) * a.per_wave;
    if (tok >= a.T) return;

    // the token's sequence: the last b whose range begins at or before it
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.cu[mid] <= tok) lo = mid;
        else hi = mid;
    }
    int t0, t1;
    token_range(a.cu, lo, a.T, t0, t1);
    if (tok < t0 || tok >= t1) return;  // a row that belongs to no sequence
    const int pos = a.kv_len[lo] - (t1 - tok);
    bool bad = pos < 0 || pos >= a.cs_rows;
    const int64_t at = page_offset(a.kv, a.table + (int64_t)lo * a.width, a.width, bad ? 0 : pos, bad);

    const bool rotated = e0 < a.rot;  // rot is a multiple of 16: a lane's eight elements are rotated or not together
    const int half = a.rot >> 1;
    const bool first = e0 < half;
    const int partner = rotated && !INTER ? (first ? hl + half / 8 : hl - half / 8) : hl;
    float cs[8], sn[8];
    {
        const int64_t r = bad ? 0 : (int64_t)pos * a.rot + (rotated ? e0 : 0);
        if constexpr (CS32) {
            const float *c = (const float*)a.cos + r, *s = (const float*)a.sin + r;
#pragma unroll
            for (int i = 0; i < 8; ++i) cs[i] = c[i], sn[i] = s[i];
        } else {
            widen8<F16>(*reinterpret_cast<const uint4*>((const uint16_t*)a.cos + r), cs);
            widen8<F16>(*reinterpret_cast<const uint4*>((const uint16_t*)a.sin + r), sn);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (INTER ? (i & 1) == 0 : first) sn[i] = -sn[i];
            if (!rotated) cs[i] = 1.f, sn[i] = 0.f;
        }
    }
    const float nan = __int_as_float(0x7FC00000);
    const int g1 = min(g0 + a.per_wave, groups);
    for (int g = g0; g < g1; ++g) {
        const int h = g * HPW + hw;
        const bool is_q = h < a.hq, is_k = !is_q && h < a.hq + a.hk;
        const bool have = h < heads;
        uint4 raw = make_uint4(0, 0, 0, 0);
        if (have) {
            const uint16_t* x = is_q   ? a.q + tok * a.q_ts + h * a.q_hs
                                : is_k ? a.k + tok * a.k_ts + (h - a.hq) * a.k_hs
                                       : a.v + tok * a.v_ts + (h - a.hq - a.hk) * a.v_hs;
            raw = *reinterpret_cast<const uint4*>(x + e0);
        }
        uint4 res = raw;
        float x[8], xp[8];
        widen8<F16>(raw, x);
        float rs = 1.f;
        if (a.qw) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(x[i], x[i], ss);
#pragma unroll
            for (int o = 1; o < LPH; o <<= 1) ss += __shfl_xor(ss, o, 64);
            rs = rsqrtf(ss * (1.f / D) + a.eps);
        }
        uint4 other = raw;
        if constexpr (!INTER) {
            const int src = hw * LPH + partner;
            other.x = __shfl((int)raw.x, src, 64);
            other.y = __shfl((int)raw.y, src, 64);
            other.z = __shfl((int)raw.z, src, 64);
            other.w = __shfl((int)raw.w, src, 64);
        }
        widen8<F16>(other, xp);
        if (is_q || is_k) {
            if (a.qw) {
                const uint16_t* w = is_q ? a.qw : a.kw;
                float wv8[8], wp[8];
                widen8<F16>(*reinterpret_cast<const uint4*>(w + e0), wv8);
                widen8<F16>(*reinterpret_cast<const uint4*>(w + 8 * partner), wp);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = x[i] * rs * wv8[i], xp[i] = xp[i] * rs * wp[i];
            }
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                // unrotated elements: y = x exactly, whatever the partner holds
                const float t = INTER ? x[i ^ 1] : xp[i];
                y[i] = rotated ? __builtin_fmaf(x[i], cs[i], t * sn[i]) : x[i];
                if (bad) y[i] = nan;
            }
            res = make_uint4(round2<F16>(y[0], y[1]), round2<F16>(y[2], y[3]), round2<F16>(y[4], y[5]),
                             round2<F16>(y[6], y[7]));
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
static void launch_append(const AppendArgs& a, bool inter, bool cs32, dim3 grid, hipStream_t st) {
#define WISP_APPEND(I, C) \
    if (inter == I && cs32 == C) hipLaunchKernelGGL((k_kv_append<F16, D, I, C>), grid, dim3(256), 0, st, a);
    WISP_APPEND(false, false)
    WISP_APPEND(false, true)
    WISP_APPEND(true, false)
    WISP_APPEND(true, true)
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
    // Few tokens: a wave per head group, so that the call has as many requests in flight as it can; many: a wave walks
    // more of its token's groups and loads cos, sin and the page id less often.
    int per_wave = 1;
    while (per_wave < groups && T * ((groups + 2 * per_wave - 1) / (2 * per_wave)) >= 16384) per_wave *= 2;
    const int waves = (groups + per_wave - 1) / per_wave;
    AppendArgs a{(const uint16_t*)q, (const uint16_t*)k, (const uint16_t*)v, q_ts, q_hs, k_ts, k_hs, v_ts, v_hs,
                 (const uint16_t*)q_norm_w, (const uint16_t*)k_norm_w, eps, cos, sin, cs_rows, rot, cu, kv_len, table,
                 width, B, (int)T, hq, hk, per_wave, paged_kv(kc, vc, pages, page, page_stride, head_stride, row_stride),
                 (uint16_t*)qo};
    const int64_t blocks = (T * waves + 3) / 4;
    if (blocks > 0x7FFFFFFF) return fail_inval("too many tokens for one call");
    const dim3 grid((unsigned)blocks);
    hipStream_t st = (hipStream_t)stream;
    const bool cs32 = cs_dtype == WISP_DT_F32, in = interleaved != 0;
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
