// Attention over the paged K/V cache (paged.hpp): packed prompts, one token of each of many sequences, and one token of
// each of many sequences behind a prefix that they share.
//
//     o_i = sum_{j <= lim_i} softmax_j(scale q_i . k_j) v_j
//
// with G = Hq/Hk query heads per K/V head, q . k and all sums in binary32 from the stored 16-bit values, o rounded once.
// The weights are rounded, too, as the matrix cores take 16-bit operands: k_attn_rows gives each as one value of the type,
// which moves o by half a step of it times sum |p v| / l at most; k_attn_flat, bound by HBM, as two, whose sum is the weight
// to 2^-17 (bfloat16). Against 64 bits (relative, of all outputs): prompts in bfloat16 0.0020, where the rounding of o alone
// gives 0.0016, and 0.0023 to 0.0017 behind a shared prefix (float16 0.00029 to 0.00021); two terms there would give the
// smaller figures, for 2,519 us instead of 1,839 at 16,384 tokens, 316 to 241 in a pack of seven prompts and 48.8 to 43.2 for
// 64 sequences behind 16,000 positions. l is the sum of the unrounded weights: that of the rounded ones changes those errors
// by 1 % and, at heads of 64, costs 4 % of the time.
// A row that may attend nothing (lim_i < 0) gives zeros. One pass over the positions with a running reference m: with
// p_j = 2^(c (s_j - m)), c = scale log2(e), the sums l = sum p_j and O = sum p_j v_j are kept, and multiplied by
// 2^(c (m_old - m_new)) when m moves. m need not be the maximum, only near it: it follows when the maximum has passed it
// by 2^kLazy, so that most tiles leave O alone; the result O / l is the same. Pieces of the positions give records
// (m, l, O) that k_attn_join adds up in the same way.
//
// Both kernels compute S^T = K Q^T and O^T = V^T P^T on the matrix cores: a lane then owns one query row (a column), its
// maximum and sum are a few steps in the lane, and the lane's S^T registers are the B operand of the second product as
// they stand, provided that V^T's positions are taken in the same order, which the LDS reads do that transpose 16-bit
// 4 x 16 blocks. K and V reach LDS by direct loads (no registers held while in flight); their rows are stored with their
// 16-byte chunks permuted so that both kinds of read touch all banks.
//
//  k_attn_rows  many query rows per K/V head (prompts, shared prefix): NW waves of 32 rows, a row being (token, head of
//               the group), so grouped heads share every K/V tile; all waves walk the same tiles of 64 positions.
//  k_attn_flat  one query token per sequence: a wave takes the G rows of one K/V head (16 at most), and the four waves
//               of a workgroup, each with a slot of its own, every fourth 32 positions. HBM-bound.
#include <float.h>
#include <math.h>

#include "paged.hpp"
#include "wisp_device.hpp"
#include "wisp_internal.hpp"

namespace wisp {
namespace {

typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef float f2_t __attribute__((ext_vector_type(2)));
typedef short s4_t __attribute__((ext_vector_type(4)));
typedef float f4_t __attribute__((ext_vector_type(4)));
typedef float f16_t __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) s4_t lds_s4_t;

constexpr int kTile = 64;          // positions per tile of k_attn_rows
constexpr int kSub = 32;           // positions per slot of k_attn_flat
constexpr int kStep = 4 * kSub;    // positions of a workgroup's four slots: the grain of its pieces
constexpr float kLazy = 6.f;       // m follows the maximum past 2^kLazy
constexpr int kSlotsY = 32768;     // grid.y of k_attn_rows
constexpr int kMaxParts = 64;       // parts of a shared prefix

// The step of the maximum past m, in scores, that m follows. (Finite: -inf, where m begins, plus an infinite step is NaN.)
__device__ __forceinline__ float follow(float c) { return fminf(kLazy / c, FLT_MAX); }

// float16 weights p: times 2^8, so that small ones keep their bits (the grain 2^-24 is then 2^-32 of the largest) and
// 2^(8 + kLazy) stays below the type's 65,504. bfloat16 has binary32's range.
template <bool F16>
constexpr float kBiasP = F16 ? 8.f : 0.f;

// D = A B + C, 32 x 32 x 16: lane l holds A[row l%32][8 (l/32) ..+7], B[8 (l/32) ..+7][col l%32] and, in register i,
// D[row 8 (i/4) + 4 (l/32) + i%4][col l%32]; 16 x 16 x 32: A[row l%16][8 (l/16) ..+7], B alike, D[row 4 (l/16) + i][col l%16]
template <bool F16>
__device__ __forceinline__ f16_t mfma32(uint4 a, uint4 b, f16_t c) {
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0, 0);
}
template <bool F16>
__device__ __forceinline__ f4_t mfma16(uint4 a, uint4 b, f4_t c) {
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0, 0);
}
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (F16)
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2_t{lo, hi}), h2_t));
    else
        return pack_bf16x2(lo, hi);
}
template <bool F16>
__device__ __forceinline__ float lo_of(uint32_t u) { return F16 ? half_lo_f(u) : bf16_lo(u); }
template <bool F16>
__device__ __forceinline__ float hi_of(uint32_t u) { return F16 ? half_hi_f(u) : bf16_hi(u); }

// 4 x 16 block of 16-bit values, transposed: of each 16 lanes, lane 4r + c gives the address of row r's values 4c .. 4c+3
// and receives column t = its number among the 16, rows 0 .. 3.
__device__ __forceinline__ uint2 read_tr(const uint8_t* p) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t*)p));
}

__device__ __forceinline__ uint32_t lds_addr(const void* p) { return (uint32_t)(uintptr_t)p; }
// 64 lanes x 16 bytes from base + each lane's 32-bit offset to LDS [lds, lds + 1024). The compiler neither emits nor counts
// these loads: the waits for them are wait_vm<n>, n = the loads issued after the awaited ones. M0 is written here only
// (a reserved register: the clobber is advisory), which tests/test_paged.py checks.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma16(uint32_t lds, const uint8_t* base, uint32_t off) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lds), "v"(off), "s"(base) : "memory", "m0");
}
#pragma clang diagnostic pop
template <int N>
__device__ __forceinline__ void wait_vm() {
    static_assert(N >= 0 && N < 64, "vmcnt is 6 bits");
    __builtin_amdgcn_s_waitcnt((N & 15) | 0x70 | 0xF00 | ((N >> 4) << 14));
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void wait_lds() {
    __builtin_amdgcn_s_waitcnt(0xC07F);
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void barrier() {
    __builtin_amdgcn_sched_barrier(0);  // arithmetic stays on its side, too
    wait_lds();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
__device__ __forceinline__ const uint8_t* uniform(const uint8_t* p) {
    const uint64_t v = (uint64_t)(uintptr_t)p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return (const uint8_t*)(uintptr_t)(((uint64_t)hi << 32) | lo);
}

// Where chunk c (16 bytes) of row r is stored in its row. K is read as 16 bytes of 16 or 32 consecutive rows at one chunk:
// rows that would share banks differ in r (two 128-byte rows cover the banks at D = 64). V is read by the transposing
// loads, 32 lanes at a time: 4 rows x 64 bytes in k_attn_rows, 8 rows x 32 bytes in k_attn_flat.
template <int D>
__device__ __forceinline__ int swz_k(int r, int c) { return c ^ (D == 64 ? (r >> 1) & 7 : r & 15); }
template <int D, bool FLAT>
__device__ __forceinline__ int swz_v(int r, int c) {
    if constexpr (FLAT) return c ^ (D == 64 ? ((r >> 1) & 3) << 1 : (r & 7) << 1);
    return c ^ (D == 64 ? ((r >> 1) & 1) << 2 : (r & 3) << 2);
}

// Where a pair holds a non-finite value (exponent bits all set): the sign bits of its halves.
template <bool F16>
__device__ __forceinline__ uint32_t nonfinite2(uint32_t u) {
    constexpr uint32_t M = F16 ? 0x7C007C00u : 0x7F807F80u, ONE = F16 ? 0x04000400u : 0x00800080u;
    return ((u & M) + ONE) & 0x80008000u;
}
// The values of a pair that are finite, others as 0.
template <bool F16>
__device__ __forceinline__ uint32_t finite2(uint32_t u) {
    const uint32_t n = nonfinite2<F16>(u);
    return (n & 0x8000u ? 0u : u & 0xFFFFu) | (n >> 31 ? 0u : u & 0xFFFF0000u);
}

// What four stored values hold besides finite ones, added to a: an infinity or NaN as it is, 0 for a finite one.
template <bool F16>
__device__ __forceinline__ void add_odd(uint2 u, f4_t& a) {
    a[0] += lo_of<F16>(u.x) - lo_of<F16>(finite2<F16>(u.x));
    a[1] += hi_of<F16>(u.x) - hi_of<F16>(finite2<F16>(u.x));
    a[2] += lo_of<F16>(u.y) - lo_of<F16>(finite2<F16>(u.y));
    a[3] += hi_of<F16>(u.y) - hi_of<F16>(finite2<F16>(u.y));
}
// A sum over attended values that has come out NaN (its statistics l are not): a weight that the type, or its second term,
// rounds to 0, or a negative second term, has met an infinite value. Then the sum is that of the values that are not finite.
__device__ __forceinline__ bool spoiled(float l, f4_t o) {
    const float z = (fabsf(o[0]) + fabsf(o[1])) + (fabsf(o[2]) + fabsf(o[3]));
    return fabsf(l) < INFINITY && z != z;
}
// Those values of four dims, added up over n rows of V: the lane's dims are the 8 bytes at own of row(i), all lanes' are the
// 16 VECS bytes at first. 64 rows are looked at together.
template <bool F16, int VECS, typename Row>
__device__ __forceinline__ f4_t odd_sum(int n, int lane, int first, int own, Row row) {
    f4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int i0 = 0; i0 < n; i0 += 64) {
        const uint4* r = reinterpret_cast<const uint4*>(row(min(i0 + lane, n - 1)) + first);
        uint32_t odd = 0;
#pragma unroll
        for (int v = 0; v < VECS; ++v)
            odd |= nonfinite2<F16>(r[v].x) | nonfinite2<F16>(r[v].y) | nonfinite2<F16>(r[v].z) | nonfinite2<F16>(r[v].w);
#pragma unroll 1
        for (uint64_t m = __ballot(i0 + lane < n && odd); m; m &= m - 1) {
            add_odd<F16>(*reinterpret_cast<const uint2*>(row(i0 + __builtin_ctzll(m)) + own), sum);
            if (!__any(sum[0] == sum[0] || sum[1] == sum[1] || sum[2] == sum[2] || sum[3] == sum[3])) return sum;  // NaN all
        }
    }
    return sum;
}
__device__ __forceinline__ void mend(float l, f4_t& o, f4_t odd) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (fabsf(l) < INFINITY && o[i] != o[i] && odd[i] != 0.f) o[i] = odd[i];
}

// The order of a turn's LDS reads and matrix instructions: NV operands of V (two reads each), then NK of K (one read), each
// read kAhead instructions before its use. (Left to itself the compiler reads two at a time and waits for them.)
constexpr int kAhead = 4;
template <int NV, int NK, int I>
__device__ __forceinline__ void order_step() {
    if constexpr (I >= kAhead) __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
    if constexpr (I < NV) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    else if constexpr (I < NV + NK) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    if constexpr (I + 1 < NV + NK + kAhead) order_step<NV, NK, I + 1>();
}
template <int NV, int NK>
__device__ __forceinline__ void order_turn() { order_step<NV, NK, 0>(); }

struct RowsArgs {
    const uint16_t* q;
    int64_t q_ts, q_hs;  // elements
    PagedKV kv;
    const int *cu, *kv_len, *table;  // cu null: one sequence of B rows, none of which is masked (a shared prefix)
    int width, B, T, hq, hk, G;
    float per_group;  // 1 / G
    float c;          // scale * log2(e)
    int nsplit;     // parts that the grid has for each row tile
    int part_min;   // tiles that a part is worth
    float *ml, *po;  // records of split row tiles: [(token * hq + head) * nsplit + part][2] and [..][D]
    uint16_t* out;   // [T][hq][D]; null: every tile leaves records
};

struct RowTile {
    int b, rows, off, end;      // sequence, its rows, position of its token 0, positions that the tile's rows attend
    int first, tok0, rem, left; // q row of the sequence's token 0; the tile's first row is head rem of the group of token
                                // tok0, and left rows of the sequence begin with it
    bool bad;                   // the sequence is longer than its table
};
// Parts that a row tile's positions are cut into: no more than nsplit, and part_min tiles each.
__device__ __forceinline__ int parts_of(int tiles, int nsplit, int part_min) {
    return max(1, min(nsplit, tiles / part_min));
}
// Of a tile whose rows are those from head rem of token tok0 on: token of its row x (x + rem < 2^11).
__device__ __forceinline__ int token_of(int tok0, int rem, int x, float per_group) {
    return tok0 + (int)(((float)(rem + x) + 0.5f) * per_group);
}

// Row tile number s of the pack (tiles of BM rows, sequence after sequence), or false.
template <int BM>
__device__ __forceinline__ bool find_tile(const RowsArgs& a, int s, int lane, RowTile& t) {
    const int G = a.G;
    t.bad = false;
    if (s < 0) return false;
    int r0;
    if (!a.cu) {
        t.b = 0, t.first = 0, t.rows = a.B * G, r0 = s * BM;
        if (r0 >= t.rows) return false;
    } else {
        int before = 0;
        bool found = false;
        for (int b0 = 0; b0 < a.B && !found; b0 += 64) {
            int lo = 0, hi = 0;
            if (b0 + lane < a.B) token_range(a.cu, b0 + lane, a.T, lo, hi);
            const int n = ((hi - lo) * G + BM - 1) / BM;
            const int sum = before + wave_scan(n);
            const uint64_t mine = __ballot(s < sum);
            if (mine) {
                const int w = __builtin_ctzll(mine);
                t.b = b0 + w;
                t.first = __builtin_amdgcn_readlane(lo, w);
                t.rows = (__builtin_amdgcn_readlane(hi, w) - t.first) * G;
                r0 = (s - (__builtin_amdgcn_readlane(sum, w) - __builtin_amdgcn_readlane(n, w))) * BM;
                found = true;
            } else {
                before = __builtin_amdgcn_readlane(sum, 63);
            }
        }
        if (!found) return false;
    }
    const int len = held(scalar_at(a.kv_len, t.b), a.width, a.kv.shift, t.bad);
    t.tok0 = (int)((uint32_t)r0 / (uint32_t)G);
    t.rem = r0 - t.tok0 * G;
    t.left = t.rows - r0;
    t.off = 0;
    t.end = len;
    if (a.cu) {
        t.off = len - (int)((uint32_t)t.rows / (uint32_t)G);
        const int last = __builtin_amdgcn_readfirstlane(token_of(t.tok0, t.rem, min(BM, t.left) - 1, a.per_group));
        t.end = max(0, t.off + last + 1);
    }
    return true;
}

// Grid: x = part * hk + head, so that a head's workgroups mostly share an XCD's L2 (hk a divisor or multiple of 8); y and z:
// the slot, counting down, since a prompt's last rows have the most positions.
//
// A tile costs a wave D / 4 matrix instructions of 32 cycles each (S and O, 1,024 cycles at D = 128) and about as many
// VALU cycles (32 weights per lane), and the LDS reads of its operands are as long. With eight waves, two to a SIMD, the
// two halves of the workgroup take turns: while waves 0-3 run a tile's matrix products, waves 4-7 weigh their tile, and
// a barrier swaps the parts. A turn M(j) is O += V(j) P(j), then S(j + 1) = K(j + 1) Q^T; a turn W(j) turns S(j) into
// P(j). K and V of four tiles are in LDS or on their way.
// Measured (32 query, 4 K/V heads of 128, bfloat16): 16,384 tokens 1,840 us, 1.20 PFLOP/s with the matrix cores 67 % and the
// VALU 58 % busy at the clock that the power limit leaves; one tile at a time without turns 2,305. 64 query, 8 K/V heads of
// 64, 1,018 tokens behind 24,000: 407 us, matrix cores 41 %, VALU 62 %, 28 % of the waves' time in waits: neither is full, the
// halves wait for each other. 16 query, 8 K/V heads of 256, 16,000 tokens: 2,230 us, 0.94 PFLOP/s, matrix cores 40 % (one wave
// a SIMD: weights and products by turns).
template <bool F16, int D, int NW>
__global__ __launch_bounds__(64 * NW, D == 64 && NW == 4 ? 3 : 1) void k_attn_rows(const RowsArgs a, int slots) {
    constexpr int BM = 32 * NW, KD = D / 16, ND = D / 32, RB = 2 * D;  // RB: bytes of a row
    constexpr int RPI = 1024 / RB;                                      // rows per load instruction
    constexpr int LPW = kTile / RPI / NW;                               // K (and V) load instructions per wave and tile
    constexpr int TB = kTile * RB;
    constexpr bool TURNS = NW == 8;
    constexpr int NST = TURNS ? 4 : 2;  // tiles in LDS
    static_assert(kTile % (RPI * NW) == 0, "tile rows per wave");
    __shared__ __align__(1024) uint8_t buf[NST][2][TB];  // [stage][K, V]
    __shared__ int bad_l, odd_l;  // a page that does not exist; an infinite or NaN value taken out of V
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, hf = lane >> 5;
    const int G = a.G;
    const int part = a.nsplit > 1 ? blockIdx.x / a.hk : 0, head = blockIdx.x - part * a.hk;
    const int slot = slots - 1 - (int)(blockIdx.y + kSlotsY * blockIdx.z);
    RowTile t;
    if (!find_tile<BM>(a, slot, lane, t)) return;
    const int tiles = (t.end + kTile - 1) / kTile;
    const int parts = a.out ? parts_of(tiles, a.nsplit, a.part_min) : a.nsplit;
    if (part >= parts) return;
    const int j0 = parts > 1 ? (int)((uint64_t)tiles * part / parts) : 0, j1 = parts > 1 ? (int)((uint64_t)tiles * (part + 1) / parts) : tiles;
    if (threadIdx.x == 0) bad_l = odd_l = 0;

    const int* trow = a.table + (int64_t)t.b * a.width;
    const uint8_t* kbase = a.kv.kc + head * a.kv.hs;
    const uint8_t* vbase = a.kv.vc + head * a.kv.hs;
    // instruction i of this wave fills rows PW wv + RPI i .. of the tile, all of one page; lane: row lane / (RB/16), stored
    // chunk lane % (RB/16)
    constexpr int PW = kTile / NW;
    const int dr = lane / (RB / 16), dc = lane % (RB / 16);
    uint32_t ko[LPW], vo[LPW];
#pragma unroll
    for (int i = 0; i < LPW; ++i) {
        const int r = PW * wv + RPI * i + dr;
        ko[i] = (uint32_t)(dr * (int)a.kv.rs + 16 * swz_k<D>(r, dc));
        vo[i] = (uint32_t)(dr * (int)a.kv.rs + 16 * swz_v<D, false>(r, dc));
    }
    bool bad = t.bad;
    const int last_row = max(0, t.end - 1) & ~(RPI - 1);
    // Tile j's page id, read a turn before its loads are issued (rows past the end repeat the last ones: their page exists).
    int page;
    auto find_pages = [&](int j) {
        const int at = min(j * kTile + PW * wv, last_row) >> a.kv.shift;
        page = scalar_at(trow, min(at, a.width - 1));
        if (at >= a.width) page = -1;
    };
    auto issue = [&](int j) {
        const uint32_t st = lds_addr(&buf[j & (NST - 1)][0][0]) + PW * wv * RB;
        const bool ok = (unsigned)page < (unsigned)a.kv.pages;
        bad = bad || !ok;
        const int64_t off = (ok ? (int64_t)page : 0) * a.kv.ps;
#pragma unroll
        for (int i = 0; i < LPW; ++i) {
            const int row = min(j * kTile + PW * wv + RPI * i, last_row) & ((1 << a.kv.shift) - 1);
            const int64_t at = off + (int64_t)row * a.kv.rs;
            dma16(st + i * 1024, uniform(kbase + at), ko[i]);
            dma16(st + TB + i * 1024, uniform(vbase + at), vo[i]);
        }
    };
    const bool late = TURNS && wv >= NW / 2;
    const int lead = late ? 3 : TURNS ? 2 : 1;  // tiles requested before the first is used
    for (int j = j0; j < min(j1, j0 + lead); ++j) {
        find_pages(j);
        issue(j);
    }
    find_pages(j0 + lead);

    // this lane's query row: (token, head of the group); rows past the sequence's repeat its last and are not stored
    const int x = 32 * wv + n, xx = min(x, t.left - 1);
    const int tok = token_of(t.tok0, t.rem, xx, a.per_group), g = t.rem + xx - (tok - t.tok0) * G;
    const int lim = a.cu ? t.off + tok : t.end - 1;
    const bool active = 32 * wv < t.left;
    // limits of the workgroup's first row, and of the wave's first and last
    const int lim_wg = a.cu ? t.off + t.tok0 : t.end - 1;
    const int lim_lo = __builtin_amdgcn_readfirstlane(lim), lim_hi = __builtin_amdgcn_readlane(lim, 31);
    uint4 qb[KD];
    {
        const uint16_t* qr = a.q + (int64_t)(t.first + tok) * a.q_ts + (int64_t)(head * G + g) * a.q_hs + 8 * hf;
#pragma unroll
        for (int s = 0; s < KD; ++s) qb[s] = *reinterpret_cast<const uint4*>(qr + 16 * s);
    }
    // q arrives here: awaited where it is first used, inside the loop, it would have the compiler wait there for every load
    // in flight, each time round
#pragma unroll
    for (int k = 0; k < KD; ++k) asm volatile("" : "+v"(qb[k].x), "+v"(qb[k].y), "+v"(qb[k].z), "+v"(qb[k].w));

    // The lane's places in a tile. K: row n (a block of 32 rows further on the same chunk: swz_k sees r % 16, or r % 16 / 2),
    // chunk 2k + hf. V: rows 4 hf + (lane % 16) / 4 (swz_v sees r % 4), dims 32 d + 16 (lane / 16 % 2) + 4 (lane % 4).
    int kl[KD], vl[ND];
#pragma unroll
    for (int k = 0; k < KD; ++k) kl[k] = n * RB + 16 * swz_k<D>(n, 2 * k + hf);
    {
        const int r = 4 * hf + ((lane & 15) >> 2);
#pragma unroll
        for (int d = 0; d < ND; ++d)
            vl[d] = r * RB + 16 * swz_v<D, false>(r, 4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) + 8 * (lane & 1);
    }

    f16_t o[ND], s[2];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
    float m = -INFINITY, mb = 0.f, l = 0.f;  // reference, c * m - bias (0 while m is -inf), this lane's share of the sum
    const float c = a.c, th = follow(a.c);
    uint4 pb[4];  // B operand of positions 16 ks ..: slot 8 hf + e is position 16 ks + 8 (e/4) + 4 hf + e%4

    auto scores = [&](int j) {  // S(j)
        const uint8_t* kt = &buf[j & (NST - 1)][0][0];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[u][i] = 0.f;
#pragma unroll
        for (int k = 0; k < KD; ++k)
#pragma unroll
            for (int u = 0; u < 2; ++u)
                s[u] = mfma32<F16>(*reinterpret_cast<const uint4*>(kt + kl[k] + 32 * u * RB), qb[k], s[u]);
    };
    auto weigh = [&](int j) {  // P(j), m, l
        const int p0 = j * kTile;
        if (lim_lo < p0 + kTile - 1) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (32 * u + 8 * (i >> 2) + (i & 3) > lim - p0 - 4 * hf) s[u][i] = -INFINITY;
        }
        float mx = s[0][0];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[u][i]);
        mx = max_xor32(mx);
        if (__any(mx > m + th)) {
            const float mn = fmaxf(m, mx);
            const float nb = mn == -INFINITY ? 0.f : mn * c - kBiasP<F16>;
            const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mb - nb);
            l *= f;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= f;
            m = mn;
            mb = nb;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float p[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][i], c, -mb));
                l += p[i];
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
                pb[2 * u + h] = make_uint4(pack2<F16>(p[8 * h], p[8 * h + 1]), pack2<F16>(p[8 * h + 2], p[8 * h + 3]),
                                           pack2<F16>(p[8 * h + 4], p[8 * h + 5]), pack2<F16>(p[8 * h + 6], p[8 * h + 7]));
        }
        // the weights are formed here, in this turn: the compiler would move them to where they are used, past the barrier
#pragma unroll
        for (int k = 0; k < 4; ++k) asm volatile("" : "+v"(pb[k].x), "+v"(pb[k].y), "+v"(pb[k].z), "+v"(pb[k].w));
    };
    auto collect = [&](int j) {  // O += V(j) P(j)
        const uint8_t* vt = &buf[j & (NST - 1)][1][0];
        auto v_operand = [&](int d, int ks) {
            const uint2 x = read_tr(vt + vl[d] + 16 * ks * RB), y = read_tr(vt + vl[d] + (16 * ks + 8) * RB);
            return make_uint4(x.x, x.y, y.x, y.y);
        };
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d] = mfma32<F16>(v_operand(d, ks), pb[ks], o[d]);
    };
    // Where a tile has positions that not all rows attend, V must hold nothing that weight 0 would not erase: rows past the
    // end, which may hold anything, are cleared, and an infinite or NaN value is taken out and added at the end to those
    // rows that attend it. By the threads first, first + many, ..
    auto unsafe = [&](int j) { return (j + 1) * kTile - 1 > lim_wg; };
    auto make_safe = [&](int j, int first, int many) {
        uint8_t* vt = &buf[j & (NST - 1)][1][0];
        const int tail = (t.end - j * kTile) * (RB / 16);
        for (int e = first; e < kTile * (RB / 16); e += many) {
            uint4 u = e < tail ? *reinterpret_cast<const uint4*>(vt + 16 * e) : make_uint4(0, 0, 0, 0);
            const bool odd = nonfinite2<F16>(u.x) | nonfinite2<F16>(u.y) | nonfinite2<F16>(u.z) | nonfinite2<F16>(u.w);
            if (odd) {
                u = make_uint4(finite2<F16>(u.x), finite2<F16>(u.y), finite2<F16>(u.z), finite2<F16>(u.w));
                odd_l = 1;
            }
            if (odd || e >= tail) *reinterpret_cast<uint4*>(vt + 16 * e) = u;
        }
    };

    // (one or two tiles are requested already, and are sooner done without turns)
    const bool turns = TURNS && j1 - j0 > 2;
    if (TURNS && turns) {
        // Interval 2j is W(j) of waves 0-3 and M(j - 1) of waves 4-7, interval 2j + 1 the other way round. In W(j) waves 0-3
        // request their part of tile j + 2 and waves 4-7 theirs of tile j + 3, whose stages' tiles j - 2 and j - 1 nobody
        // reads any more. All await tile j + 1 before interval 2j + 1, that of M(j), which is the first to read it, with one
        // tile after it still on its way.
        auto await = [&](bool newer) {
            if (newer) wait_vm<2 * LPW>();
            else wait_vm<0>();
        };
        if (j0 < j1) {
            await(false);
            barrier();
            if (late) {
                await(j0 + 2 < j1);  // tile j0 + 1
                barrier();
            }
            // the wave's own tiles are j0 .. jw - 1: past them its rows attend nothing
            const int jw = active && lim_hi >= j0 * kTile ? min(j1, lim_hi / kTile + 1) : j0;
            auto begin_w = [&](int j) {
                if (j + lead < j1) {
                    issue(j + lead);
                    find_pages(j + lead + 1);
                }
                if (!late && unsafe(j)) make_safe(j, threadIdx.x, 32 * NW);
            };
            auto end_w = [&](int j) {
                if (!late) await(j + 2 < j1);  // tile j + 1
                barrier();
            };
            auto end_m = [&](int j) {
                if (late) await(j + 3 < j1);  // tile j + 2
                barrier();
            };
            if (j0 < jw) {
                scores(j0);
                order_turn<0, 2 * KD>();
            }
            if (late) await(j0 + 2 < j1);
            barrier();
            for (int j = j0; j < jw - 1; ++j) {
                begin_w(j);
                weigh(j);
                end_w(j);
                __builtin_amdgcn_s_setprio(1);
                collect(j);
                scores(j + 1);
                order_turn<4 * ND, 2 * KD>();
                __builtin_amdgcn_s_setprio(0);
                end_m(j);
            }
            if (j0 < jw) {
                begin_w(jw - 1);
                weigh(jw - 1);
                end_w(jw - 1);
                collect(jw - 1);
                order_turn<4 * ND, 0>();
                end_m(jw - 1);
            }
            for (int j = jw; j < j1; ++j) {
                begin_w(j);
                end_w(j);
                end_m(j);
            }
            if (!late) barrier();
        }
    } else {
        for (int j = j0; j < j1; ++j) {
            wait_vm<0>();
            barrier();  // every wave's part of tile j is there, and nobody reads the other stage any more
            if (!TURNS && j + 1 < j1) {
                issue(j + 1);
                find_pages(j + 2);
            }
            if (unsafe(j)) {
                make_safe(j, threadIdx.x, 64 * NW);
                barrier();
            }
            if (active && lim_hi >= j * kTile) {
                scores(j);
                if constexpr (D == 256) order_turn<0, 2 * KD>();  // (one wave a SIMD: 132 us, 155 without, at 3,000 tokens)
                weigh(j);
                collect(j);
                if constexpr (D == 256) order_turn<4 * ND, 0>();
            }
        }
    }

    if (bad) bad_l = 1;  // any wave's
    barrier();
    if (!active) return;
    l = add_xor32(l);
    const int p_odd = max(j0 * kTile, (lim_wg + 1) & ~(kTile - 1));  // the first tile with positions that not all rows attend
    if constexpr (F16) {
        // (bfloat16 weights have binary32's range; a float16 one below 2^-33 of the largest is 0.) The tiles up to p_odd:
        const int n_even = min(p_odd, min(j1 * kTile, t.end)) - j0 * kTile;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                f4_t x = {o[d][4 * e], o[d][4 * e + 1], o[d][4 * e + 2], o[d][4 * e + 3]};
                if (!__any(spoiled(l, x))) continue;
                mend(l, x, odd_sum<F16, 1>(n_even, lane, 64 * d + 16 * e, 64 * d + 16 * e + 8 * hf, [&](int i) {
                         return vbase + page_offset(a.kv, trow, a.width, j0 * kTile + i, bad);
                     }));
#pragma unroll
                for (int i = 0; i < 4; ++i) o[d][4 * e + i] = x[i];
            }
    }
    if (odd_l) {
#pragma unroll 1
        for (int p = p_odd; p < min(j1 * kTile, t.end); ++p) {
            const uint8_t* vr = vbase + page_offset(a.kv, trow, a.width, p, bad) + 8 * hf;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint2 u = *reinterpret_cast<const uint2*>(vr + 64 * d + 16 * e);
                    if (p <= lim && (nonfinite2<F16>(u.x) | nonfinite2<F16>(u.y))) {
                        f4_t odd = {0.f, 0.f, 0.f, 0.f};
                        add_odd<F16>(u, odd);
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[d][4 * e + i] += odd[i];
                    }
                }
        }
    }
    const bool poison = bad_l != 0;
    // A lane's values lie in four-value runs of one row: through LDS, in the wave's own part of it (16-byte chunks permuted
    // as K's), to stores of whole rows.
    const int orow = (t.first + tok) * a.hq + head * G + g;
    uint8_t* mine = &buf[0][0][0] + wv * (32 * 4 * D);
    if (a.out && parts == 1) {
        const float inv = poison ? __int_as_float(0x7FC00000) : l == 0.f ? 0.f : 1.f / l;
        constexpr int SW = RB / 16 < 16 ? RB / 16 - 1 : 15;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                *reinterpret_cast<uint2*>(mine + n * RB + 16 * ((4 * d + e) ^ (n & SW)) + 8 * hf) =
                    make_uint2(pack2<F16>(o[d][4 * e] * inv, o[d][4 * e + 1] * inv),
                               pack2<F16>(o[d][4 * e + 2] * inv, o[d][4 * e + 3] * inv));
        wait_lds();
#pragma unroll
        for (int i = 0; i < 32 / RPI; ++i) {
            const int r = RPI * i + dr, to = __shfl(orow, r, 64);
            const uint4 u = *reinterpret_cast<const uint4*>(mine + r * RB + 16 * (dc ^ (r & SW)));
            if (32 * wv + r < t.left) *reinterpret_cast<uint4*>(a.out + (int64_t)to * D + 8 * dc) = u;
        }
    } else {
        const int64_t rec = (int64_t)orow * a.nsplit + part;
        if (hf == 0 && x < t.left) {
            a.ml[2 * rec] = m;
            a.ml[2 * rec + 1] = poison ? __int_as_float(0x7FC00000) : l;
        }
        constexpr int FB = 4 * D, FPI = 1024 / FB;  // bytes of a record's row, rows per instruction
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                *reinterpret_cast<f4_t*>(mine + n * FB + 16 * ((8 * d + 2 * e + hf) ^ (n & 15))) =
                    f4_t{o[d][4 * e], o[d][4 * e + 1], o[d][4 * e + 2], o[d][4 * e + 3]};
        wait_lds();
#pragma unroll
        for (int i = 0; i < 32 / FPI; ++i) {
            const int r = FPI * i + lane / (FB / 16), fc = lane % (FB / 16), to = __shfl(orow, r, 64);
            const f4_t u = *reinterpret_cast<const f4_t*>(mine + r * FB + 16 * (fc ^ (r & 15)));
            if (32 * wv + r < t.left) *reinterpret_cast<f4_t*>(a.po + ((int64_t)to * a.nsplit + part) * D + 4 * fc) = u;
        }
    }
}

// ---------------------------------------------------------------------------
struct FlatArgs {
    const uint16_t* q;
    int64_t q_ts, q_hs;
    PagedKV kv;
    const int *kv_len, *table;
    int width, B, hq, hk, G, want;
    float c;
    int* first;      // [B][2]: number of the sequence's first piece, its pieces
    float *ml, *po;  // records [(first + piece) * hq + head]
    const float *rml, *rpo;  // with a prefix: its records [(b * hq + head) * nsplit + part]
    int nsplit;
    int single;      // every sequence is one piece, and what this kernel leaves is the result
    uint16_t* out;   // [B][hq][D]; null: every piece leaves a record (a prefix's are to be added)
};

// Steps of kStep positions that a sequence needs.
__device__ __forceinline__ int steps_of(const FlatArgs& a, int b) {
    bool over = false;
    return b < a.B ? (held(a.kv_len[b], a.width, a.kv.shift, over) + kStep - 1) / kStep : 0;
}

// Grid: x = piece, or the sequence where each is taken whole (takes_whole); y = K/V head, times tiles of 16 of its rows. A wave's
// slot holds one K and one V block, each requested again as soon as it is read, so that a block of each wave is always on
// its way; waves share nothing until the end, so there is no barrier in the loop.
// Measured: two sequences of 100,000 to 130,000 positions (8 K/V heads of 64) 92 us, 5.0 TB/s; 32 of 200 to 16,000 (4 of
// 128) 38 us, 4.5 TB/s with k_attn_join.
template <bool F16, int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void k_attn_flat(const FlatArgs a) {
    constexpr int RB = 2 * D, RPI = 1024 / RB, LI = kSub / RPI, KD = D / 32, ND = D / 16;
    constexpr int SB = kSub * RB;
    constexpr int OS = D + 4;  // floats between rows of the join
    __shared__ __align__(1024) uint8_t slot[4][2][SB];
    __shared__ float red[4][16][2];
    static_assert(sizeof(float) * 4 * 16 * OS <= sizeof(slot), "the join reuses the slots");
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, r = lane >> 4;
    const int G = a.G;
    const int hr = blockIdx.y, rt = a.hk == (int)gridDim.y ? 0 : hr / a.hk, head = hr - rt * a.hk, g0 = 16 * rt;
    const int id = blockIdx.x;

    int b = id, piece = 0, pieces = 1, before = 0, grain = 1 << 23;
    if (!a.single) {
        // The grain of the pieces, in steps: the same for every sequence, so that all pieces are of like size however
        // different the lengths are, and no more than a.want of them in all, if it can be. Then this workgroup's.
        const int steps0 = steps_of(a, lane);  // of the first 64 sequences
        int total = 0;
        for (int b0 = 0; b0 < a.B; b0 += 64) total += __builtin_amdgcn_readlane(wave_scan(b0 ? steps_of(a, b0 + lane) : steps0), 63);
        grain = max(1, (int)(((uint32_t)total + a.want - 1) / (uint32_t)a.want));
        b = -1;
        for (int b0 = 0; b0 < a.B && b < 0; b0 += 64) {
            const int np = small_div((b0 ? steps_of(a, b0 + lane) : steps0) + grain - 1, grain);
            const int sum = before + wave_scan(np);
            const uint64_t mine = __ballot(id < sum);
            if (mine) {
                const int w = __builtin_ctzll(mine);
                b = b0 + w;
                pieces = __builtin_amdgcn_readlane(np, w);
                before = __builtin_amdgcn_readlane(sum, w) - pieces;
                piece = id - before;
            } else {
                before = __builtin_amdgcn_readlane(sum, 63);
            }
        }
        if (b < 0) return;
        if (piece == 0 && hr == 0 && threadIdx.x == 0) {
            a.first[2 * b] = before;
            a.first[2 * b + 1] = pieces;
        }
    }
    bool bad = false;
    const int len = held(scalar_at(a.kv_len, b), a.width, a.kv.shift, bad);
    const int from = piece * grain * kStep, to = (int)min((int64_t)len, from + (int64_t)grain * kStep);

    const int* trow = a.table + (int64_t)b * a.width;
    const uint8_t* kbase = a.kv.kc + head * a.kv.hs;
    const uint8_t* vbase = a.kv.vc + head * a.kv.hs;
    uint8_t *ks = &slot[wv][0][0], *vs = &slot[wv][1][0];
    const int dr = lane / (RB / 16), dc = lane % (RB / 16);
    // The page ids of the 32 positions from p on (16 are always in one page; rows past the end repeat the last 16: their
    // page exists), read an iteration before its loads are issued.
    int page[2];
    auto half_at = [&](int p, int h) { return min(p + 16 * h, (to - 1) & ~15); };
    auto find_pages = [&](int p) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = half_at(p, h) >> a.kv.shift;
            page[h] = scalar_at(trow, min(at, a.width - 1));
            if (at >= a.width) page[h] = -1;
        }
    };
    // the lane's offset in an instruction's rows: the permutations have period 16 in the row
    constexpr int SAME = 16 / RPI;
    uint32_t ko[SAME], vo[SAME];
#pragma unroll
    for (int i = 0; i < SAME; ++i) {
        const int rr = RPI * i + dr;
        ko[i] = (uint32_t)((rr & 15) * (int)a.kv.rs + 16 * swz_k<D>(rr, dc));
        vo[i] = (uint32_t)((rr & 15) * (int)a.kv.rs + 16 * swz_v<D, true>(rr, dc));
    }
    auto issue = [&](int p, bool v) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const bool ok = (unsigned)page[h] < (unsigned)a.kv.pages;
            bad = bad || !ok;
            const int64_t off = (ok ? (int64_t)page[h] : 0) * a.kv.ps + (int64_t)(half_at(p, h) & ((1 << a.kv.shift) - 1)) * a.kv.rs;
            const uint8_t* base = uniform((v ? vbase : kbase) + off);
#pragma unroll
            for (int i = 0; i < LI / 2; ++i) dma16(lds_addr((v ? vs : ks) + 1024 * (h * (LI / 2) + i)), base, v ? vo[i] : ko[i]);
        }
    };
    const int p_first = from + kSub * wv;
    uint4 qb[KD];
    {
        const uint16_t* qr = a.q + (int64_t)b * a.q_ts + (int64_t)(head * G + min(g0 + n, G - 1)) * a.q_hs + 8 * r;
#pragma unroll
        for (int k = 0; k < KD; ++k) qb[k] = *reinterpret_cast<const uint4*>(qr + 32 * k);
    }
    // the compiler's own loads are complete before the first counted one
#pragma unroll
    for (int k = 0; k < KD; ++k) asm volatile("" : "+v"(qb[k].x), "+v"(qb[k].y), "+v"(qb[k].z), "+v"(qb[k].w));
    if (p_first < to) {
        find_pages(p_first);
        issue(p_first, false);
        issue(p_first, true);
        find_pages(p_first + kStep);
    }

    f4_t o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] = f4_t{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, mb = 0.f, l = 0.f;
    const float c = a.c, th = follow(a.c);
    for (int p = p_first; p < to; p += kStep) {
        const bool more = p + kStep < to;
        wait_vm<LI>();  // K is there, V may be in flight
        f4_t s[2] = {f4_t{0.f, 0.f, 0.f, 0.f}, f4_t{0.f, 0.f, 0.f, 0.f}};
        uint4 ka[2][KD];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int k = 0; k < KD; ++k) {
                const int rr = 16 * u + n;
                ka[u][k] = *reinterpret_cast<const uint4*>(ks + rr * RB + 16 * swz_k<D>(rr, 4 * k + r));
            }
        wait_lds();  // the K slot is read: it may be refilled
        if (more) issue(p + kStep, false);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int k = 0; k < KD; ++k) s[u] = mfma16<F16>(ka[u][k], qb[k], s[u]);
        if (p + kSub > to) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (p + 16 * u + 4 * r + i >= to) s[u][i] = -INFINITY;
        }
        float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                         fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        mx = max_xor32(max_xor16(mx));
        if (__any(mx > m + th)) {
            const float mn = fmaxf(m, mx);
            const float nb = mn == -INFINITY ? 0.f : mn * c - kBiasP<F16>;
            const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mb - nb);
            l *= f;
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d] = f4_t{o[d][0] * f, o[d][1] * f, o[d][2] * f, o[d][3] * f};
            m = mn;
            mb = nb;
        }
        // p as two terms of the type, so that its rounding costs nothing: hi + lo is p to 2^-17 of it
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float pe[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                pe[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][i], c, -mb));
                l += pe[i];
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t w = pack2<F16>(pe[2 * h], pe[2 * h + 1]);
                hi[2 * u + h] = w;
                lo[2 * u + h] = pack2<F16>(pe[2 * h] - lo_of<F16>(w), pe[2 * h + 1] - hi_of<F16>(w));
            }
        }
        if (more) wait_vm<LI>();  // V is there, the next K may be in flight
        else wait_vm<0>();
        if (p + kSub > to) {  // rows past the end
            for (int e = (to - p) * (RB / 16) + lane; e < kSub * (RB / 16); e += 64)
                *reinterpret_cast<uint4*>(vs + 16 * e) = make_uint4(0, 0, 0, 0);
            wait_lds();
        }
        uint4 va[ND];
        const int vr = 4 * r + (n >> 2), vcn = (n & 3) >> 1, vb = 8 * (n & 1);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            const uint2 x = read_tr(vs + vr * RB + 16 * swz_v<D, true>(vr, 2 * d + vcn) + vb);
            const uint2 y = read_tr(vs + (vr + 16) * RB + 16 * swz_v<D, true>(vr + 16, 2 * d + vcn) + vb);
            va[d] = make_uint4(x.x, x.y, y.x, y.y);
        }
        wait_lds();  // the V slot is read
        if (more) {
            issue(p + kStep, true);
            find_pages(p + 2 * kStep);
        }
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] = mfma16<F16>(va[d], make_uint4(hi[0], hi[1], hi[2], hi[3]), o[d]);
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] = mfma16<F16>(va[d], make_uint4(lo[0], lo[1], lo[2], lo[3]), o[d]);
    }
    wait_vm<0>();

    // the four waves' sums: o[d][i] = O[row n][dim 16 d + 4 r + i]
    l = add_xor32(add_xor16(l));
    if (bad) l = __int_as_float(0x7FC00000);
    const int mine = max(0, to - p_first), n_mine = mine / kStep * kSub + min(mine % kStep, kSub);  // the wave's positions
#pragma unroll
    for (int d = 0; d < ND; ++d)
        if (__any(spoiled(l, o[d])))
            mend(l, o[d], odd_sum<F16, 2>(n_mine, lane, 32 * d, 32 * d + 8 * r, [&](int i) {
                     return vbase + page_offset(a.kv, trow, a.width, p_first + i / kSub * kStep + i % kSub, bad);
                 }));
    if (r == 0) {
        red[wv][n][0] = m;
        red[wv][n][1] = l;
    }
    barrier();  // the slots are free, too
    float M = red[0][n][0];
#pragma unroll
    for (int w = 1; w < 4; ++w) M = fmaxf(M, red[w][n][0]);
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - M) * c);
    float* join = reinterpret_cast<float*>(&slot[0][0][0]);
#pragma unroll
    for (int d = 0; d < ND; ++d)
        *reinterpret_cast<f4_t*>(join + (wv * 16 + n) * OS + 16 * d + 4 * r) = f4_t{o[d][0] * f, o[d][1] * f, o[d][2] * f, o[d][3] * f};
    barrier();
    const int rows = min(16, G - g0);
    const int64_t row0 = (int64_t)b * a.hq + head * G + g0;  // of out
    const int parts = a.single ? a.nsplit : 0;
    // This piece's share of each row, and those of the prefix's parts, as factors of their O, 1/L of the whole included:
    // 16 lanes a row.
    __shared__ float own[16], share[16][kMaxParts];
    if (parts) {
        const int row = min((int)threadIdx.x >> 4, rows - 1), e = threadIdx.x & 15;
        float Mr = red[0][row][0], L = 0.f;
#pragma unroll
        for (int w = 1; w < 4; ++w) Mr = fmaxf(Mr, red[w][row][0]);
#pragma unroll
        for (int w = 0; w < 4; ++w) L += red[w][row][0] == -INFINITY ? red[w][row][1] : red[w][row][1] * __builtin_amdgcn_exp2f((red[w][row][0] - Mr) * c);
        float m[kMaxParts / 16], ll[kMaxParts / 16], Mx = Mr;
        bool none[kMaxParts / 16];  // a record without weights
#pragma unroll
        for (int k = 0; k < kMaxParts / 16; ++k) {
            const int p = e + 16 * k;
            m[k] = p < parts ? a.rml[2 * ((row0 + row) * parts + p)] : -INFINITY;
            ll[k] = p < parts ? a.rml[2 * ((row0 + row) * parts + p) + 1] : 0.f;
            Mx = fmaxf(Mx, m[k]);
        }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) Mx = fmaxf(Mx, __shfl_xor(Mx, o, 64));
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < kMaxParts / 16; ++k) {
            none[k] = m[k] == -INFINITY;
            const float w = none[k] ? 0.f : __builtin_amdgcn_exp2f((m[k] - Mx) * c);
            sum += none[k] ? ll[k] : ll[k] * w;  // (a record without weights has m = -inf; its l may be a bad page's NaN)
            m[k] = w;
        }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) sum += __shfl_xor(sum, o, 64);
        const float f0 = Mr == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((Mr - Mx) * c);
        sum += Mr == -INFINITY ? L : L * f0;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        if ((int)threadIdx.x >> 4 < rows) {
            if (e == 0) own[row] = f0 * inv;
#pragma unroll
            for (int k = 0; k < kMaxParts / 16; ++k)
                if (e + 16 * k < parts) share[row][e + 16 * k] = none[k] ? -1.f : m[k] * inv;
        }
        __syncthreads();
    }
    for (int e = threadIdx.x; e < rows * (D / 2); e += 256) {
        const int row = e / (D / 2), d = 2 * (e - row * (D / 2));
        float x = 0.f, y = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            x += join[(w * 16 + row) * OS + d];
            y += join[(w * 16 + row) * OS + d + 1];
        }
        uint16_t* const to_out = a.out + (row0 + row) * D + d;
        if (parts) {
            x *= own[row];
            y *= own[row];
            const float* po = a.rpo + (row0 + row) * parts * D + d;
#pragma unroll 8
            for (int p = 0; p < parts; ++p) {
                const float f = share[row][p];
                const float2 v = *reinterpret_cast<const float2*>(po + p * D);
                x += f < 0.f ? 0.f : f * v.x;  // (the O of a record without weights is zeros, or of NaN values that have none)
                y += f < 0.f ? 0.f : f * v.y;
            }
            *reinterpret_cast<uint32_t*>(to_out) = pack2<F16>(x, y);
            continue;
        }
        float Mr = red[0][row][0], L = 0.f;
#pragma unroll
        for (int w = 1; w < 4; ++w) Mr = fmaxf(Mr, red[w][row][0]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float mw = red[w][row][0], lw = red[w][row][1];
            // (a wave without positions has m = -inf and l = 0, or NaN from a bad page)
            L += mw == -INFINITY ? lw : lw * __builtin_amdgcn_exp2f((mw - Mr) * c);
        }
        if (a.out && pieces == 1) {
            const float inv = L == 0.f ? 0.f : 1.f / L;
            *reinterpret_cast<uint32_t*>(to_out) = pack2<F16>(x * inv, y * inv);
        } else {
            const int64_t rec = (int64_t)(before + piece) * a.hq + head * G + g0 + row;
            if (d == 0) {
                a.ml[2 * rec] = Mr;
                a.ml[2 * rec + 1] = L;
            }
            *reinterpret_cast<float2*>(a.po + rec * D + d) = make_float2(x, y);
        }
    }
}

// ---------------------------------------------------------------------------
// The records of a query row added up: those of its sequence's pieces (k_attn_flat) and those of its row tile's parts
// (k_attn_rows). One workgroup of 4 waves per row of out; wave w takes every fourth record.
// Bound by the latency of a record's reads and its launch: 3 to 8 us.
struct JoinArgs {
    const int *first, *kv_len;   // pieces of the sequences, or first null
    const float *ml, *po;
    const int *cu, *kv_own;      // prompt: cu and kv_len of the pack (which rows were cut, and into how many parts)
    const float *rml, *rpo;      // parts: records [row * nsplit + part], or null
    int nsplit, part_min, bm, B, T, hq, hk, cap, all;  // cap: positions of a table row; all: every row has nsplit parts (a shared prefix)
    float c;
    uint16_t* out;
};

template <bool F16, int D>
__global__ __launch_bounds__(256) void k_attn_join(const JoinArgs a) {
    constexpr int EPL = D / 64;
    __shared__ float rm[4], rl[4], ro[4][D];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    if (row >= (int64_t)a.T * a.hq) return;
    const int tok = (int)(row / a.hq), hd = (int)(row - (int64_t)tok * a.hq);
    int na = 0, nb = 0;
    int64_t a0 = 0;
    if (a.first) {
        if (a.kv_len[tok] > 0) {
            na = a.first[2 * tok + 1];
            a0 = (int64_t)a.first[2 * tok] * a.hq + hd;
        }
        if (a.all) nb = a.nsplit;
        else if (na == 1) return;  // stored whole
    } else {
        const int G = a.hq / a.hk;
        int lo = 0, hi = a.B;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.cu[mid] <= tok) lo = mid;
            else hi = mid;
        }
        int t0, t1;
        token_range(a.cu, lo, a.T, t0, t1);
        if (tok < t0 || tok >= t1) return;
        const int rows = (t1 - t0) * G, r = (tok - t0) * G + hd % G, len = min(a.kv_own[lo], a.cap);
        const int last = min(r / a.bm * a.bm + a.bm, rows) - 1;  // of the row's tile
        const int end = max(0, len - (t1 - t0) + last / G + 1);
        nb = parts_of((end + kTile - 1) / kTile, a.nsplit, a.part_min);
        if (nb == 1) return;
    }
    float M = -INFINITY, L = 0.f, O[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) O[e] = 0.f;
    auto take = [&](const float* ml, const float* po, int64_t rec) {
        const float m = ml[2 * rec], l = ml[2 * rec + 1];
        const float mn = fmaxf(M, m);
        const float fo = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((M - mn) * a.c);
        const float fn = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mn) * a.c);
        L = L * (M == -INFINITY ? 1.f : fo) + (m == -INFINITY ? l : l * fn);  // (NaN of a bad page stays)
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
            const float v = po[rec * D + EPL * lane + e];
            O[e] = O[e] * fo + (m == -INFINITY ? 0.f : v * fn);
        }
        M = mn;
    };
    for (int i = wv; i < na; i += 4) take(a.ml, a.po, a0 + (int64_t)i * a.hq);
    for (int i = wv; i < nb; i += 4) take(a.rml, a.rpo, row * a.nsplit + i);
    if (lane == 0) rm[wv] = M, rl[wv] = L;
#pragma unroll
    for (int e = 0; e < EPL; ++e) ro[wv][EPL * lane + e] = O[e];
    __syncthreads();
    if (threadIdx.x < D / 2) {
        const int d = 2 * threadIdx.x;
        const float Mx = fmaxf(fmaxf(rm[0], rm[1]), fmaxf(rm[2], rm[3]));
        float x = 0.f, y = 0.f, Lt = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = rm[w] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((rm[w] - Mx) * a.c);
            Lt += rm[w] == -INFINITY ? rl[w] : rl[w] * f;
            x += ro[w][d] * f;
            y += ro[w][d + 1] * f;
        }
        const float inv = Lt == 0.f ? 0.f : 1.f / Lt;
        *reinterpret_cast<uint32_t*>(a.out + row * D + d) = pack2<F16>(x * inv, y * inv);
    }
}

// ---------------------------------------------------------------------------
// Query rows of a k_attn_rows workgroup. D = 256: four waves, whose registers the CU's whole file holds (16 query and 2 K/V
// heads, 3,000 tokens: 113 us; eight waves with tiles of 32 positions 207, 16 over 8 heads and 8,000 tokens 598 and 582).
// D = 128: eight.
// D = 64, where a tile's weights cost twice its matrix products: four waves, four workgroups to a CU, where there are enough
// to keep them all busy, else eight waves that take turns. 64 query and 8 K/V heads, four and eight waves: 1,280 tokens, the
// rule's border, 29.7 and 30.9 us alone, 76 and 92 behind 2,000 positions, 646 and 823 behind 24,000; 4,000 tokens 151 and 166,
// 288 and 305, 1,817 and 1,821; 2,000 tokens behind 24,000 912 and 883. Below it, behind 24,000, 1,000 tokens 482 and 441, 300
// tokens 364 and 182. Without such a context four waves are ahead there, too (1,000 tokens 23.9 and 25.9, and far where eight
// leave tiles few enough to be cut in parts: 300 tokens 11 and 39), but how long the context is only the device knows.
int rows_of(int d, int64_t rows, int hk) { return d == 256 || (d == 64 && rows / 128 * hk >= 640) ? 128 : 256; }

template <bool F16>
void launch_rows(const RowsArgs& a, int d, int bm, int slots, hipStream_t st) {
    const dim3 grid((unsigned)(a.nsplit * a.hk), (unsigned)(slots < kSlotsY ? slots : kSlotsY), (unsigned)((slots + kSlotsY - 1) / kSlotsY));
    if (d == 64 && bm == 128) hipLaunchKernelGGL((k_attn_rows<F16, 64, 4>), grid, dim3(256), 0, st, a, slots);
    else if (d == 64) hipLaunchKernelGGL((k_attn_rows<F16, 64, 8>), grid, dim3(512), 0, st, a, slots);
    else if (d == 128) hipLaunchKernelGGL((k_attn_rows<F16, 128, 8>), grid, dim3(512), 0, st, a, slots);
    else hipLaunchKernelGGL((k_attn_rows<F16, 256, 4>), grid, dim3(256), 0, st, a, slots);
}
template <bool F16>
void launch_flat(const FlatArgs& a, int d, int64_t pieces, hipStream_t st) {
    const dim3 grid((unsigned)(a.single ? a.B : pieces), (unsigned)(a.hk * ((a.G + 15) / 16)));
    if (d == 64) hipLaunchKernelGGL((k_attn_flat<F16, 64>), grid, dim3(256), 0, st, a);
    else if (d == 128) hipLaunchKernelGGL((k_attn_flat<F16, 128>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_attn_flat<F16, 256>), grid, dim3(256), 0, st, a);
}
template <bool F16>
void launch_join(const JoinArgs& a, int d, hipStream_t st) {
    // a workgroup per row of out, in two dimensions: one holds fewer than 2^32 threads, 2^24 workgroups
    const int64_t rows = (int64_t)a.T * a.hq, x = 1 << 23;
    const dim3 grid((unsigned)(rows < x ? rows : x), (unsigned)((rows + x - 1) / x));
    if (d == 64) hipLaunchKernelGGL((k_attn_join<F16, 64>), grid, dim3(256), 0, st, a);
    else if (d == 128) hipLaunchKernelGGL((k_attn_join<F16, 128>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_attn_join<F16, 256>), grid, dim3(256), 0, st, a);
}

// Row tiles that T tokens of B sequences can have: each sequence's last may be partly empty.
int64_t row_slots(int64_t T, int B, int G, int bm) { return (T * G + bm - 1) / bm + B - 1; }

// Parts for each row tile: where the tiles alone leave CUs without work and the positions are many, enough to occupy the
// card once (256 CUs, one workgroup each), but at least kPartTiles tiles of positions each.
constexpr int kPartTiles = 2;
int row_parts(int64_t groups, int64_t positions) {
    const int64_t most = (positions + kTile - 1) / kTile / kPartTiles;
    const int64_t want = groups < 1 ? 1 : 256 / groups;
    return (int)(want < most ? (want < 1 ? 1 : want) : (most < 1 ? 1 : most));
}

// Whether k_attn_flat takes each sequence whole, which spares the records and k_attn_join: where no table holds more than
// 4 steps of positions, or 8 where there are workgroups enough without pieces, or a prefix's records to be added anyway.
// Whole and in pieces, 4 K/V heads of 128, every sequence as long as its table: one sequence of 512 positions 7.6 and 8.9 us, 768
// 9.1 and 9.4, 1,024 10.8 and 9.5; 64 of 512 14.2 and 18.7, of 1,024 23.6 and 27.6. Behind a prefix of 2,000: one of 512 17.1
// and 17.2, of 1,024 20.4 and 17.7 (the loss at few sequences); 16 of 1,024 24.2 and 24.7, 64 43.0 and 46.8. Longer tables gain,
// too, where all are full (64 of 2,048: 43.0 and 47.0), but one long sequence among short ones would then be the call.
bool takes_whole(int B, int hq, int hk, int64_t positions, bool prefix) {
    const int64_t groups = (int64_t)B * hk * ((hq / hk + 15) / 16);
    return positions <= (groups >= 256 || prefix ? 8 : 4) * kStep;
}

// Records: m and l of all, then, from a multiple of 16 bytes on (k_attn_rows stores 16 at a time), their O.
int64_t ml_bytes(int64_t recs) { return (recs * 8 + 15) / 16 * 16; }
int64_t rec_bytes(int64_t recs, int d) { return ml_bytes(recs) + recs * d * 4; }

struct FlatWs {
    int want;  // pieces that the grain aims at
    int64_t pieces, first, ml, po, end;
};
// k_attn_flat's pieces: as many as workgroups that 256 CUs hold at once (their LDS: 4, 2 or 1 a CU).
FlatWs flat_ws(int B, int hq, int hk, int d) {
    const int G = hq / hk, heads = hk * ((G + 15) / 16), most = d == 64 ? 1024 : d == 128 ? 512 : 256;
    FlatWs w;
    w.want = most / heads < 1 ? 1 : most / heads;
    w.pieces = w.want + B;
    w.first = 0;
    w.ml = ((int64_t)B * 8 + 15) / 16 * 16;
    w.po = w.ml + ml_bytes(w.pieces * hq);
    w.end = w.po + w.pieces * hq * d * 4;
    return w;
}

constexpr float kLog2E = 1.44269504088896340736f;
bool good_scale(float s) { return s > 0.f && s * kLog2E < INFINITY; }

int check_q(const void* q, int64_t q_ts, int64_t q_hs, const void* out) {
    if (!aligned(q, 16) || !aligned(out, 16) || q_ts % 8 || q_hs % 8) {
        set_error("q, its strides and out must be 16-byte aligned");
        return WISP_EALIGN;
    }
    return WISP_OK;
}

int check_ws(const void* ws) {
    if (!aligned(ws, 16)) {
        set_error("ws must be 16-byte aligned");
        return WISP_EALIGN;
    }
    return WISP_OK;
}

}  // namespace
}  // namespace wisp

using namespace wisp;

extern "C" int64_t wisp_attn_prompt_ws_bytes(int64_t T, int B, int hq, int hk, int d, int page, int width) {
    if (T < 0 || T > (1 << 30) || B < 1 || hk < 1 || hq < hk || hq > 1024 || hq % hk || d < 64 || page < 1 || width < 1) return -1;
    const int parts = row_parts(row_slots(T, B, hq / hk, rows_of(d, T * (hq / hk), hk)) * hk, (int64_t)page * width);
    return parts > 1 ? rec_bytes(T * hq * parts, d) : 0;
}

extern "C" int wisp_attn_prompt(const void* q, int64_t q_ts, int64_t q_hs, const void* kc, const void* vc, int64_t pages,
                                int page, int64_t page_stride, int64_t head_stride, int64_t row_stride, const int32_t* cu,
                                const int32_t* kv_len, const int32_t* table, int width, int B, int64_t T, int hq, int hk,
                                int d, int dtype, float scale, void* ws, void* out, void* stream) {
    clear_error();
    if (int rc = check_paged(kc, vc, pages, page, page_stride, head_stride, row_stride, width, B, hq, hk, d, dtype)) return rc;
    if (T < 0 || T > (1 << 30) || T * hq > (1 << 30)) return fail_inval("T * hq must be in [0, 2^30]");
    if (!good_scale(scale)) return fail_inval("scale must be positive, and finite times log2(e)");
    if (T == 0) return WISP_OK;
    if (!q || !cu || !kv_len || !table || !out) return fail_inval("null pointer");
    if (int rc = check_q(q, q_ts, q_hs, out)) return rc;
    const int bm = rows_of(d, T * (hq / hk), hk);
    const int64_t slots = row_slots(T, B, hq / hk, bm);
    const int parts = row_parts(slots * hk, (int64_t)page * width);
    if (parts > 1 && !ws) return fail_inval("null workspace");
    if (int rc = check_ws(ws)) return rc;
    float* ml = (float*)ws;
    float* po = ml ? (float*)((uint8_t*)ws + ml_bytes(T * hq * parts)) : nullptr;
    RowsArgs a{(const uint16_t*)q, q_ts, q_hs, paged_kv((void*)kc, (void*)vc, pages, page, page_stride, head_stride, row_stride),
               cu, kv_len, table, width, B, (int)T, hq, hk, hq / hk, 1.f / (float)(hq / hk), scale * kLog2E, parts, kPartTiles, ml, po, (uint16_t*)out};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == WISP_DT_F16) launch_rows<true>(a, d, bm, (int)slots, st);
    else launch_rows<false>(a, d, bm, (int)slots, st);
    if (parts > 1) {
        JoinArgs j{nullptr, nullptr, nullptr, nullptr, cu, kv_len, ml, po, parts, kPartTiles, bm, B, (int)T, hq, hk, width * page, 0, a.c, (uint16_t*)out};
        if (dtype == WISP_DT_F16) launch_join<true>(j, d, st);
        else launch_join<false>(j, d, st);
    }
    return check_launch("k_attn_rows");
}

// The parts of a shared prefix: rows of all B sequences together.
static int prefix_parts(int B, int hq, int hk, int d, int64_t positions) {
    const int bm = rows_of(d, (int64_t)B * (hq / hk), hk);
    const int n = row_parts((int64_t)(((int64_t)B * (hq / hk) + bm - 1) / bm) * hk, positions);
    return n < kMaxParts ? n : kMaxParts;
}

extern "C" int64_t wisp_attn_batch_ws_bytes(int B, int hq, int hk, int d, int page, int width, int prefix_width) {
    if (B < 1 || hk < 1 || hq < hk || hq % hk || d < 64 || page < 1 || width < 1 || prefix_width < 0) return -1;
    const bool whole = takes_whole(B, hq, hk, (int64_t)width * page, prefix_width > 0);
    const int64_t own = whole ? 0 : flat_ws(B, hq, hk, d).end;
    return prefix_width ? own + rec_bytes((int64_t)B * hq * prefix_parts(B, hq, hk, d, (int64_t)page * prefix_width), d) : own;
}

extern "C" int wisp_attn_batch(const void* q, int64_t q_ts, int64_t q_hs, const void* kc, const void* vc, int64_t pages,
                               int page, int64_t page_stride, int64_t head_stride, int64_t row_stride,
                               const int32_t* kv_len, const int32_t* table, int width, const int32_t* prefix_len,
                               const int32_t* prefix_table, int prefix_width, int B, int hq, int hk, int d, int dtype,
                               float scale, void* ws, void* out, void* stream) {
    clear_error();
    if (int rc = check_paged(kc, vc, pages, page, page_stride, head_stride, row_stride, width, B, hq, hk, d, dtype)) return rc;
    if (!good_scale(scale)) return fail_inval("scale must be positive, and finite times log2(e)");
    if (prefix_width < 0 || (int64_t)prefix_width * page > (1 << 30)) return fail_inval("the prefix's positions must be in [0, 2^30]");
    if (!q || !kv_len || !table || !out || (prefix_width && (!prefix_len || !prefix_table))) return fail_inval("null pointer");
    const bool whole = takes_whole(B, hq, hk, (int64_t)width * page, prefix_width > 0);
    if (!ws && (!whole || prefix_width)) return fail_inval("null workspace");
    if (int rc = check_q(q, q_ts, q_hs, out)) return rc;
    if (int rc = check_ws(ws)) return rc;
    FlatWs w = flat_ws(B, hq, hk, d);
    if (whole) w.ml = w.po = w.end = 0;  // (no records of its own)
    if ((int64_t)B * hq > (1 << 30) || (int64_t)B * ((int64_t)width * page / kStep + 1) > 0x7FFFFFFF)
        return fail_inval("too many sequences, or positions in their tables, for one call");
    const PagedKV kv = paged_kv((void*)kc, (void*)vc, pages, page, page_stride, head_stride, row_stride);
    const float c = scale * kLog2E;
    uint8_t* p = (uint8_t*)ws;
    hipStream_t st = (hipStream_t)stream;
    const bool f16 = dtype == WISP_DT_F16;
    FlatArgs f{(const uint16_t*)q, q_ts, q_hs, kv, kv_len, table, width, B, hq, hk, hq / hk, w.want, c, (int*)p, (float*)(p + w.ml),
               (float*)(p + w.po), nullptr, nullptr, 0, whole, (uint16_t*)out};
    if (prefix_width && !f.single) f.out = nullptr;
    JoinArgs j{f.first, kv_len, f.ml, f.po, nullptr, nullptr, nullptr, nullptr, 0, 1, 1, B, B, hq, hk, 0, 0, c, (uint16_t*)out};
    if (prefix_width) {
        const int bm = rows_of(d, (int64_t)B * (hq / hk), hk), slots = (int)(((int64_t)B * (hq / hk) + bm - 1) / bm);
        const int parts = prefix_parts(B, hq, hk, d, (int64_t)page * prefix_width);
        float* rml = (float*)(p + w.end);
        RowsArgs a{(const uint16_t*)q, q_ts, q_hs, kv, nullptr, prefix_len, prefix_table, prefix_width, B, B, hq, hk, hq / hk, 1.f / (float)(hq / hk), c, parts, 1,
                   rml, (float*)((uint8_t*)rml + ml_bytes((int64_t)B * hq * parts)), nullptr};
        if (f16) launch_rows<true>(a, d, bm, slots, st);
        else launch_rows<false>(a, d, bm, slots, st);
        j.rml = f.rml = a.ml;
        j.rpo = f.rpo = a.po;
        j.nsplit = f.nsplit = parts;
        j.all = 1;
    }
    if (f16) launch_flat<true>(f, d, w.pieces, st);
    else launch_flat<false>(f, d, w.pieces, st);
    if (!f.single) {
        if (f16) launch_join<true>(j, d, st);
        else launch_join<false>(j, d, st);
    }
    return check_launch("k_attn_flat");
}
