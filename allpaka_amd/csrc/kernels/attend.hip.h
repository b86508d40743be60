// gfx950 device code, part of apk_kernels.hip: attention over the paged fp16 K/V cache.
//
// Row r of a sequence with n cached keys, its m new rows among them, is at position p = n - m + r and sees the keys
// max(0, p - window + 1) .. p (window 0: from 0).  With x_j = scale * log2(e) * <q, K_j>:
//     o = sum_j 2^(x_j - M) V_j / sum_j 2^(x_j - M),   M the running maximum of the x_j met so far,
// one pass over the keys; sums and maxima in f32.  A row that sees no key gives zeros.
//
// Scores and outputs are held transposed (S^T = K Q^T, O^T = V^T P^T): a lane then holds one query's scores, so its
// maximum, its sum and the rescaling of its outputs need no other lane but the two to four that share the query, and the
// probabilities are already laid out as the second product's operand.  fp16 products are exact in f32.  With f32
// activations a query element is the sum of two fp16 values (its row scaled by a power of two first), and so is a
// probability: 22 bits of each take part.  With fp16 activations probabilities are rounded to fp16 once (an error of
// 2^-12 relative at most, next to the 2^-12 of the fp16 result); they are held times 2^14, so that a key of weight down
// to 2^-28 of the largest keeps all its bits, which a long cache of small weights needs.
#pragma once
#include "../apk_attend.h"

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

static constexpr float kProbShift = 14.0f;  // probabilities are held as 2^14 p
#define NEG_INF (-__builtin_inff())

// {lane's own value, that of lane ^ X} in some order, X = 16 or 32: one swap of half rows, no LDS.  Written out, because
// the compiler's builtin hands back one of the two registers twice; the instruction needs two wait states after the vector
// instruction that wrote its operand (never a matrix instruction here: the operand is a sum or a maximum).
template <int X> DEV f32x2 pair_xor(float v) {
    f32x2 r = {v, v};
    if constexpr (X == 32) asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(r.x), "+v"(r.y));
    else asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(r.x), "+v"(r.y));
    return r;
}
template <int X> DEV float max_xor(float v) {
    const f32x2 t = pair_xor<X>(v);
    return fmaxf(t.x, t.y);
}
template <int X> DEV float sum_xor(float v) {
    const f32x2 t = pair_xor<X>(v);
    return t.x + t.y;
}
DEV float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// key / page and key % page for any key < 2^32: the host's magic is floor(2^32 / page) (2^32 - 1 for page 1), which
// is short by less than one page.
DEV void split_key(const apk_attend_args& a, uint32_t key, uint32_t& idx, uint32_t& off) {
    idx = __umulhi(key, a.page_magic);
    off = key - idx * a.page;
    if (off >= a.page) {
        idx++;
        off -= a.page;
    }
}

// ------------------------------------------------------------------------------------------- division of the work
// A tile is tile_rows flat rows (token * group + head of the group) of one sequence and kv head.  Every sequence's tiles
// are cut into the same number of parts along the keys: one, where there are tiles enough to fill the chip, else as many
// as bring the launch to about `target` workgroups, parts of at least unit_min units.  The lengths are on the device, so
// each workgroup works its own place out: two short passes of a wave over the sequences.
struct att_seq {
    uint32_t row0, m;  // first row, rows
    int32_t n, p0;     // keys, position of the first row
    uint32_t tiles, parts, umax;
};
struct att_item {
    uint32_t seq, tile, part, slot;
    att_seq s;
};
DEV att_seq att_load_seq(const apk_attend_args& a, uint32_t i) {
    att_seq s;
    uint32_t n = a.kv_len[i];
    const uint64_t cap = (uint64_t)a.max_pages * a.page;
    bool bad = n > cap;
    if (bad) n = (uint32_t)cap;
    uint32_t r0 = i, r1 = i + 1;
    if (a.q_off) {
        r0 = a.q_off[i];
        r1 = a.q_off[i + 1];
        if (r1 > a.rows || r0 > r1) {
            atomicOr(a.fault, APK_FAULT_ROW_RANGE);
            r1 = r1 < a.rows ? r1 : a.rows;
            r0 = r0 < r1 ? r0 : r1;
        }
    }
    if (bad) atomicOr(a.fault, APK_FAULT_CACHE_RANGE);
    s.row0 = r0;
    s.m = r1 - r0;
    s.n = (int32_t)n;
    s.p0 = (int32_t)n - (int32_t)s.m;
    const uint64_t flat = (uint64_t)s.m * a.group;
    s.tiles = a.q_off ? (uint32_t)((flat + a.tile_rows - 1) / a.tile_rows) : (s.m ? 1u : 0u);
    uint32_t span = n;
    if (a.window) {  // keys that the rows of one tile see between them
        const uint64_t w = (uint64_t)a.window + (a.q_off ? a.tile_rows / a.group + 1 : 0) + a.unit;
        if (w < span) span = (uint32_t)w;
    }
    s.umax = (span + a.unit - 1) / a.unit;
    s.parts = 1;
    return s;
}
DEV uint32_t rl(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }
DEV uint64_t rl64(uint64_t v, int lane) { return ((uint64_t)rl((uint32_t)(v >> 32), lane) << 32) | rl((uint32_t)v, lane); }
DEV uint64_t wave_scan_u64(uint64_t v) {  // inclusive sums over the lanes
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t t = ((uint64_t)(uint32_t)__shfl_up((uint32_t)(v >> 32), d) << 32) | (uint32_t)__shfl_up((uint32_t)v, d);
        if ((int)(threadIdx.x & 63) >= d) v += t;
    }
    return v;
}
DEV uint64_t wave_sum_u64(uint64_t v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t lo = __shfl_xor((uint32_t)v, d), hi = __shfl_xor((uint32_t)(v >> 32), d);
        v += ((uint64_t)hi << 32) | lo;
    }
    return v;
}
// Units a part has at least, so that no more than `target` parts come of splitting.
DEV uint32_t att_units_per_part(const apk_attend_args& a) {
    const uint32_t lane = threadIdx.x & 63;
    uint64_t u = 0;
    for (uint32_t i = lane; i < a.n_seq; i += 64) {
        const att_seq s = att_load_seq(a, i);
        u += (uint64_t)s.tiles * s.umax;
    }
    u = (a.n_seq > 1 ? wave_sum_u64(u) : rl64(u, 0)) * a.n_kv * a.head_tiles;
    const uint64_t c = (u + a.target - 1) / a.target;
    return c > a.unit_min ? (uint32_t)c : a.unit_min;
}
DEV uint32_t att_parts(const att_seq& s, uint32_t c) { return s.umax > c ? (s.umax + c - 1) / c : 1u; }
// The tile and part that item `pg` (0, 1, ...; without the kv head) of the launch is; false: past the last one.  SPLIT:
// items are the tiles that were cut, `slot` the first of a tile's parts.
template <bool SPLIT> DEV bool att_find(const apk_attend_args& a, uint32_t pg, att_item& it) {
    const uint32_t lane = threadIdx.x & 63, c = att_units_per_part(a);
    uint64_t before = 0, slots = 0;
    for (uint32_t base = 0; base < a.n_seq; base += 64) {
        const uint32_t i = base + lane;
        att_seq s = {0, 0, 0, 0, 0, 1, 0};
        if (i < a.n_seq) {
            s = att_load_seq(a, i);
            s.parts = att_parts(s, c);
        }
        const uint64_t parts = (uint64_t)s.tiles * s.parts, cut = s.parts > 1 ? parts : 0;
        const uint64_t cnt = SPLIT ? (s.parts > 1 ? s.tiles : 0) : parts;
        uint64_t inc = cnt, sinc = cut;
        if (a.n_seq > 1) {
            inc = wave_scan_u64(inc);
            sinc = wave_scan_u64(sinc);
        }
        const uint64_t hit = __ballot(before + inc > pg && before + inc - cnt <= pg);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            it.seq = base + (uint32_t)l;
            it.s.row0 = rl(s.row0, l);
            it.s.m = rl(s.m, l);
            it.s.n = (int32_t)rl((uint32_t)s.n, l);
            it.s.p0 = (int32_t)rl((uint32_t)s.p0, l);
            it.s.tiles = rl(s.tiles, l);
            it.s.parts = rl(s.parts, l);
            it.s.umax = rl(s.umax, l);
            const uint32_t idx = pg - (uint32_t)(before + rl64(inc - cnt, l));
            const uint32_t slot0 = (uint32_t)(slots + rl64(sinc - cut, l));
            it.tile = it.s.tiles - 1 - (SPLIT ? idx : idx / it.s.parts);  // the last rows see the most keys: they go first
            it.part = SPLIT ? 0 : idx % it.s.parts;
            it.slot = slot0 + (SPLIT ? idx * it.s.parts : idx);
            return true;
        }
        if (a.n_seq > 64) {
            before += rl64(inc, 63);
            slots += rl64(sinc, 63);
        }
    }
    return false;
}

// The keys [lo, hi) that any row of a tile sees (tok0 .. tok1: its first and last row of the sequence) and, of their
// units, those of one part.
struct att_span {
    int32_t lo, hi;    // keys
    uint32_t u0, u1;   // units of this part: keys [u0 * unit, u1 * unit)
};
DEV att_span att_tile_span(const apk_attend_args& a, const att_seq& s, uint32_t part, uint32_t tok0, uint32_t tok1) {
    att_span r;
    int64_t lo = a.window ? (int64_t)s.p0 + tok0 - (int64_t)a.window + 1 : 0;
    int64_t hi = (int64_t)s.p0 + tok1 + 1;
    r.lo = (int32_t)(lo < 0 ? 0 : lo);
    r.hi = (int32_t)(hi < 0 ? 0 : hi);
    uint32_t first = (uint32_t)r.lo / a.unit, last = ((uint32_t)r.hi + a.unit - 1) / a.unit;
    if (last < first) last = first;
    const uint64_t nu = last - first;
    r.u0 = first + (uint32_t)(nu * part / s.parts);
    r.u1 = first + (uint32_t)(nu * (part + 1) / s.parts);
    return r;
}

// Cache row of a key of sequence `seq`; keys outside [lo, hi) are not looked up and read row 0, whose values are not used.
// A table entry that names no page raises a fault and reads row 0 as well.
DEV uint32_t att_row(const apk_attend_args& a, const uint32_t* tab, int32_t key, int32_t lo, int32_t hi) {
    if (key < lo || key >= hi) return 0;
    uint32_t idx, off;
    split_key(a, (uint32_t)key, idx, off);
    const uint32_t e = tab[idx];
    if (e >= a.n_pages) {
        atomicOr(a.fault, APK_FAULT_CACHE_RANGE);
        return 0;
    }
    return e * a.page + off;
}

// ------------------------------------------------------------------------------------------- query fragments
// Eight consecutive elements of a query row as fp16: one fragment for fp16 rows, a high and a low one for f32 rows whose
// elements are multiplied by `mul` (a power of two) first.
template <typename T> struct att_q;
template <> struct att_q<f16_t> {
    static constexpr int N = 1;
    DEV void load(const f16_t* p, bool on, float sign, float, f16x8* f) {
        f16x8 t = {0, 0, 0, 0, 0, 0, 0, 0};
        if (on) t = *(const f16x8*)p;
        f[0] = sign < 0.f ? -t : t;
    }
    DEV float absmax(const f16_t*, bool) { return 0.f; }
};
template <> struct att_q<float> {
    static constexpr int N = 2;
    DEV void load(const float* p, bool on, float sign, float mul, f16x8* f) {
        float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (on) {
            io<float>::load(p, v);
            io<float>::load(p + 4, v + 4);
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float x = v[j] * (mul * sign);
            f[0][j] = (f16_t)x;
            f[1][j] = (f16_t)(x - (float)f[0][j]);
        }
    }
    DEV float absmax(const float* p, bool on) {
        float v[8], m = 0.f;
        if (!on) return 0.f;
        io<float>::load(p, v);
        io<float>::load(p + 4, v + 4);
#pragma unroll
        for (int j = 0; j < 8; j++) m = fmaxf(m, __builtin_fabsf(v[j]));
        return m;
    }
};
// The power of two that brings a row's largest magnitude to [2^13, 2^14), and its inverse; 1 for a row of zeros.
DEV void att_q_scale(float mx, float& mul, float& inv) {
    const int e = (int)((__builtin_bit_cast(uint32_t, mx) >> 23) & 0xff);  // biased exponent
    int k = 127 + 13 - e;                                                  // multiply by 2^k
    if (e == 0 || e == 255) k = 0;
    k = k > 126 ? 126 : k < -126 ? -126 : k;
    mul = __builtin_bit_cast(float, (uint32_t)(127 + k) << 23);
    inv = __builtin_bit_cast(float, (uint32_t)(127 - k) << 23);
}

template <typename T> DEV void att_store8(T* p, const float* v);
template <> __device__ __forceinline__ void att_store8<f16_t>(f16_t* p, const float* v) { io<f16_t>::store(p, v); }
template <> __device__ __forceinline__ void att_store8<float>(float* p, const float* v) {
    io<float>::store(p, v);
    io<float>::store(p + 4, v + 4);
}
template <typename T> DEV void att_store4(T* p, const float* v);
template <> __device__ __forceinline__ void att_store4<f16_t>(f16_t* p, const float* v) {
    f32x2 lo = {v[0], v[1]}, hi = {v[2], v[3]};
    *(u32x2*)p = u32x2{__builtin_bit_cast(uint32_t, __builtin_convertvector(lo, f16x2)), __builtin_bit_cast(uint32_t, __builtin_convertvector(hi, f16x2))};
}
template <> __device__ __forceinline__ void att_store4<float>(float* p, const float* v) { io<float>::store(p, v); }

// ------------------------------------------------------------------------------------------- single tokens
// One workgroup per (sequence, kv head, tile of up to 16 query heads, part of the keys); its waves take blocks of 32 keys
// in turn and are joined through LDS at the end.  K and V go from memory straight to registers: a wave's K block is the
// first operand of 16x16x32 products as it lies (16 bytes of a key a lane), its V block becomes one by an in-lane
// transpose (8 keys x 8 channels a lane).  Bound by the stream of K and V.
template <typename T, int HD, int W>
DEV void attend_token_body(const apk_attend_args& a, float* smem) {
    constexpr int KF = HD / 32;           // K fragments of 16 keys
    constexpr int CH = HD / 16;           // channels a lane holds of a V row
    constexpr int NQ = att_q<T>::N;
    const uint32_t H = a.n_kv * a.head_tiles;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n16 = lane & 15, g = lane >> 4;
    att_item it;
    if (!att_find<false>(a, blockIdx.x / H, it)) return;
    const uint32_t hh = blockIdx.x % H, kvh = hh / a.head_tiles, ht = hh % a.head_tiles;
    const uint32_t rows_here = min(APK_ATT_TOKEN_ROWS, a.group - ht * APK_ATT_TOKEN_ROWS);
    const att_span sp = att_tile_span(a, it.s, it.part, 0, 0);
    const uint32_t* tab = a.table + (uint64_t)it.seq * a.max_pages;
    const uint64_t kv_stride = (uint64_t)a.n_kv * HD;
    const f16_t* kb = (const f16_t*)a.k + (uint64_t)kvh * HD;
    const f16_t* vb = (const f16_t*)a.v + (uint64_t)kvh * HD;
    const uint64_t qat = (uint64_t)it.s.row0 * a.n_q * HD + (uint64_t)(kvh * a.group + ht * APK_ATT_TOKEN_ROWS) * HD;
    const T* qb = (const T*)a.q + qat;

    f16x8 qf[KF][NQ];
    float qinv = 1.f;
    {
        const bool on = n16 < rows_here;
        float mul = 1.f;
        if constexpr (NQ == 2) {
            float mx = 0.f;
#pragma unroll
            for (int s = 0; s < KF; s++) mx = fmaxf(mx, att_q<T>::absmax(qb + n16 * HD + s * 32 + g * 8, on));
            mx = max_xor<32>(max_xor<16>(mx));
            att_q_scale(mx, mul, qinv);
        }
#pragma unroll
        for (int s = 0; s < KF; s++) att_q<T>::load(qb + n16 * HD + s * 32 + g * 8, on, a.sign, mul, qf[s]);
    }
    const float c = a.c * qinv;

    f32x4 o[CH];
#pragma unroll
    for (int i = 0; i < CH; i++) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = NEG_INF, l = 0.f;

    typedef uint32_t vrow_t __attribute__((ext_vector_type(CH / 2)));
    const int32_t k_end = min((int32_t)(sp.u1 * APK_ATT_TOKEN_UNIT), sp.hi);
    int32_t key0 = (int32_t)(sp.u0 * APK_ATT_TOKEN_UNIT) + (int32_t)wave * 32;
    const int32_t k_lo = max(sp.lo, (int32_t)(sp.u0 * APK_ATT_TOKEN_UNIT));
    f16x8 kf[2][KF];
    vrow_t vr[8];
    auto load_k = [&](uint32_t row) {
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const uint32_t r = __shfl(row, b * 16 + n16);
            const f16_t* p = kb + (uint64_t)r * kv_stride + g * 8;
#pragma unroll
            for (int s = 0; s < KF; s++) kf[b][s] = *(const f16x8*)(p + s * 32);
        }
    };
    auto load_v = [&](uint32_t row) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t r = __shfl(row, (j >> 2) * 16 + g * 4 + (j & 3));
            const f16_t* p = vb + (uint64_t)r * kv_stride;
            if constexpr (CH == 4) vr[j] = *(const vrow_t*)(p + n16 * 4);
            if constexpr (CH == 8) vr[j] = *(const vrow_t*)(p + n16 * 8);
            if constexpr (CH == 16) {
                const u32x4 x = *(const u32x4*)(p + n16 * 8), y = *(const u32x4*)(p + 128 + n16 * 8);
                vr[j] = vrow_t{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
            }
        }
    };
    uint32_t row = 0;
    if (key0 < k_end) {
        row = att_row(a, tab, key0 + (int32_t)(lane & 31), k_lo, k_end);
        load_k(row);
        load_v(row);
    }
    while (key0 < k_end) {
        const int32_t next = key0 + 32 * W;
        const bool more = next < k_end;
        uint32_t nrow = 0;
        if (more) nrow = att_row(a, tab, next + (int32_t)(lane & 31), k_lo, k_end);
        f32x4 s[2];
#pragma unroll
        for (int b = 0; b < 2; b++) {
            s[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < KF; i++)
#pragma unroll
                for (int t = 0; t < NQ; t++) s[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[b][i], qf[i][t], s[b], 0, 0, 0);
        }
        if (more) load_k(nrow);
        const bool edge = key0 < k_lo || key0 + 32 > k_end;
        if (edge) {
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int32_t key = key0 + b * 16 + (int32_t)g * 4 + i;
                    if (key < k_lo || key >= k_end) s[b][i] = NEG_INF;
                }
        }
        float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        mx = max_xor<32>(max_xor<16>(mx)) * c;
        const float mn = fmaxf(m, mx);
        const float ms = mn == NEG_INF ? 0.f : mn;
        if (__any(mn > m)) {
            const float alpha = exp2_hw(m - ms);
            l *= alpha;
#pragma unroll
            for (int i = 0; i < CH; i++) o[i] *= alpha;
            m = mn;
        }
        const float sub = kProbShift - ms;
        f16x8 ph, pl;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float p = exp2_hw(__builtin_fmaf(s[j >> 2][j & 3], c, sub));
            l += p;
            ph[j] = (f16_t)p;
            if constexpr (NQ == 2) pl[j] = (f16_t)(p - (float)ph[j]);
        }
        if (edge) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int32_t key = key0 + (j >> 2) * 16 + (int32_t)g * 4 + (j & 3);
                if (key < k_lo || key >= k_end) vr[j] = (vrow_t)(0u);
            }
        }
        f16x8 vt[CH];
#pragma unroll
        for (int w = 0; w < CH / 2; w++) {
            u32x4 e, d;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                e[j] = __builtin_amdgcn_perm(vr[2 * j + 1][w], vr[2 * j][w], 0x05040100u);
                d[j] = __builtin_amdgcn_perm(vr[2 * j + 1][w], vr[2 * j][w], 0x07060302u);
            }
            vt[2 * w] = __builtin_bit_cast(f16x8, e);
            vt[2 * w + 1] = __builtin_bit_cast(f16x8, d);
        }
        if (more) load_v(nrow);
#pragma unroll
        for (int i = 0; i < CH; i++) {
            o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt[i], ph, o[i], 0, 0, 0);
            if constexpr (NQ == 2) o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt[i], pl, o[i], 0, 0, 0);
        }
        key0 = next;
    }
    l = sum_xor<32>(sum_xor<16>(l));

    // join the waves: their maxima, then the sums of the rescaled outputs
    const uint32_t R = rows_here;
    float* sm_m = smem;               // [W][16]
    float* sm_l = smem + W * 16;      // [W][16]
    float* sm_o = smem + 2 * W * 16;  // [W][R][HD]
    if (g == 0) sm_m[wave * 16 + n16] = m;
    __syncthreads();
    float M = NEG_INF;
#pragma unroll
    for (int w = 0; w < W; w++) M = fmaxf(M, sm_m[w * 16 + n16]);
    const float f = m == NEG_INF ? 0.f : exp2_hw(m - M);
    if (g == 0) sm_l[wave * 16 + n16] = l * f;
    if (n16 < R) {
        float* dst = sm_o + ((uint64_t)wave * R + n16) * HD;
        // o[ci][i]: channel CHW * (4 g + i) + ci, the lanes of 256 channels holding two runs of eight 128 apart
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int ci = 0; ci < CH; ci++) {
                const int m16 = (int)g * 4 + i;
                const int chan = CH == 16 ? (ci >> 3) * 128 + m16 * 8 + (ci & 7) : m16 * CH + ci;
                dst[chan] = o[ci][i] * f;
            }
    }
    __syncthreads();
    const bool split = it.s.parts > 1;
    float* part = a.part + ((uint64_t)it.slot * H + hh) * ((uint64_t)APK_ATT_TOKEN_ROWS * (HD + 2));
    for (uint32_t i = threadIdx.x; i < R * (HD / 4); i += W * 64) {
        const uint32_t r = i / (HD / 4), col = (i % (HD / 4)) * 4;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        float ls = 0.f;
#pragma unroll
        for (int w = 0; w < W; w++) {
            v += *(const f32x4*)(sm_o + ((uint64_t)w * R + r) * HD + col);
            ls += sm_l[w * 16 + r];
        }
        if (split) {
            *(f32x4*)(part + r * HD + col) = v;
            if (col == 0) {
                float mm = NEG_INF;
#pragma unroll
                for (int w = 0; w < W; w++) mm = fmaxf(mm, sm_m[w * 16 + r]);
                part[APK_ATT_TOKEN_ROWS * HD + r] = mm;
                part[APK_ATT_TOKEN_ROWS * (HD + 1) + r] = ls;
            }
        } else {
            const float inv = ls > 0.f ? 1.f / ls : (ls == 0.f ? 0.f : ls);
            float t[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
            att_store4<T>((T*)a.out + qat + (uint64_t)r * HD + col, t);
        }
    }
}
extern __shared__ float att_smem[];
#define ATTEND_TOKEN(T, t, HD, W)                                                                                            \
    extern "C" __global__ __launch_bounds__(W * 64) void apk_attend_token_##t##_hd##HD##_w##W(apk_attend_args a) {           \
        attend_token_body<T, HD, W>(a, att_smem);                                                                            \
    }
#define ATTEND_TOKEN_ALL(W) \
    ATTEND_TOKEN(f16_t, f16, 64, W) ATTEND_TOKEN(f16_t, f16, 128, W) ATTEND_TOKEN(f16_t, f16, 256, W) \
    ATTEND_TOKEN(float, f32, 64, W) ATTEND_TOKEN(float, f32, 128, W) ATTEND_TOKEN(float, f32, 256, W)
ATTEND_TOKEN_ALL(4)

// ------------------------------------------------------------------------------------------- chunks of new tokens
// One workgroup of four waves per (sequence, kv head, tile of 128 flat (token, head) rows, part of the keys).  Units of
// BN keys go through LDS (fetched into registers while the unit before is worked on, two buffers, one barrier a unit); a
// wave holds 32 rows.  K rows are the first operand of 32x32x16 products as they lie; V comes out of LDS transposed
// (ds_read_b64_tr_b16), in the key order in which a lane holds its probabilities.  The 16-byte chunks of LDS row r are
// permuted by f(r), so that both kinds of reads meet all banks.  Bound by the matrix and vector pipes together: for 32
// rows x 32 keys x 128 channels 512 cycles of products stand next to about as many for the softmax.
template <int HD> DEV uint32_t att_swz(uint32_t r) {
    if constexpr (HD == 64) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    else return ((r & 3) << 2) | ((r >> 2) & 3);
}
DEV bool att_nonfinite(u32x4 t) {  // any of eight fp16 values infinite or NaN
    bool b = false;
#pragma unroll
    for (int i = 0; i < 4; i++) b |= (t[i] & 0x7c00u) == 0x7c00u || (t[i] & 0x7c000000u) == 0x7c000000u;
    return b;
}
DEV u32x4 att_clear_nonfinite(u32x4 t) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if ((t[i] & 0x7c00u) == 0x7c00u) t[i] &= 0xffff0000u;
        if ((t[i] & 0x7c000000u) == 0x7c000000u) t[i] &= 0xffffu;
    }
    return t;
}
template <typename T, int HD, int BN>
DEV void attend_chunk_body(const apk_attend_args& a, f16_t* smem) {
    constexpr int KF = HD / 16, NQ = att_q<T>::N, KB = BN / 32, HB = HD / 32, CPR = HD / 8;
    constexpr int NCH = BN * CPR / 256;  // 16-byte chunks of K (and of V) a thread stages
    const uint32_t H = a.n_kv, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n32 = lane & 31, hf = lane >> 5;
    f16_t* const sk = smem;                    // [2][BN][HD]
    f16_t* const sv = smem + 2 * BN * HD;      // [2][BN][HD]
    att_item it;
    if (!att_find<false>(a, blockIdx.x / H, it)) return;
    const uint32_t kvh = blockIdx.x % H;
    const uint64_t flat_n = (uint64_t)it.s.m * a.group, flat0 = (uint64_t)it.tile * APK_ATT_CHUNK_ROWS;
    const uint32_t tok0 = (uint32_t)(flat0 / a.group);
    const uint32_t tok1 = (uint32_t)(min(flat0 + APK_ATT_CHUNK_ROWS, flat_n) - 1) / a.group;
    const att_span sp = att_tile_span(a, it.s, it.part, tok0, tok1);
    const uint32_t* tab = a.table + (uint64_t)it.seq * a.max_pages;
    const uint64_t kv_stride = (uint64_t)a.n_kv * HD;
    const f16_t* kb = (const f16_t*)a.k + (uint64_t)kvh * HD;
    const f16_t* vb = (const f16_t*)a.v + (uint64_t)kvh * HD;

    // this lane's row, and the first and last position of the wave's rows
    const uint64_t flat = flat0 + wave * 32 + n32;
    const bool on = flat < flat_n;
    const uint32_t tok = (uint32_t)(flat / a.group), head = (uint32_t)(flat % a.group);
    const int32_t pos = on ? it.s.p0 + (int32_t)tok : -1;
    const int32_t pos_lo = a.window ? pos - (int32_t)a.window : -1;  // keys above this one
    const bool wave_on = flat0 + wave * 32 < flat_n;
    const int32_t wpos0 = it.s.p0 + (int32_t)((flat0 + wave * 32) / a.group);
    const int32_t wpos1 = it.s.p0 + (int32_t)((min(flat0 + wave * 32 + 32, flat_n) - 1) / a.group);
    const int32_t tpos0 = it.s.p0 + (int32_t)tok0, tpos1 = it.s.p0 + (int32_t)tok1;
    const uint64_t qat = ((uint64_t)(it.s.row0 + tok) * a.n_q + kvh * a.group + head) * HD;

    f16x8 qf[KF][NQ];
    float c = a.c;
    {
        const T* qb = (const T*)a.q + (on ? qat : 0);
        float mul = 1.f, inv = 1.f;
        if constexpr (NQ == 2) {
            float mx = 0.f;
#pragma unroll
            for (int s = 0; s < KF; s++) mx = fmaxf(mx, att_q<T>::absmax(qb + s * 16 + hf * 8, on));
            att_q_scale(max_xor<32>(mx), mul, inv);
        }
#pragma unroll
        for (int s = 0; s < KF; s++) att_q<T>::load(qb + s * 16 + hf * 8, on, a.sign, mul, qf[s]);
        c *= inv;
    }
    f32x16 o[HB];
#pragma unroll
    for (int i = 0; i < HB; i++)
#pragma unroll
        for (int j = 0; j < 16; j++) o[i][j] = 0.f;
    float m = NEG_INF, l = 0.f;

    // some row of the tile does not see all keys of this unit
    auto is_partial = [&](int32_t key0) { return key0 + BN - 1 > tpos0 || (a.window && key0 <= tpos1 - (int32_t)a.window); };
    bool odd = false;  // a value of V that is not finite was cleared
    // staging: thread t takes chunks t, t + 256, ... of a unit
    uint32_t rows[NCH];
    u32x4 rk[NCH], rv[NCH];
    auto look = [&](uint32_t u) {
#pragma unroll
        for (int i = 0; i < NCH; i++) {
            const uint32_t r = (i * 256 + tid) / CPR;
            rows[i] = att_row(a, tab, (int32_t)(u * BN + r), sp.lo, sp.hi);
        }
    };
    auto fetch = [&]() {
#pragma unroll
        for (int i = 0; i < NCH; i++) {
            const uint32_t p = i * 256 + tid, r = p / CPR, ch = (p % CPR) ^ att_swz<HD>(r);
            const uint64_t at = (uint64_t)rows[i] * kv_stride + ch * 8;
            rk[i] = *(const u32x4*)(kb + at);
            rv[i] = *(const u32x4*)(vb + at);
        }
    };
    auto stage = [&](uint32_t u) {
        const int32_t key0 = (int32_t)(u * BN);
        const bool edge = key0 < sp.lo || key0 + BN > sp.hi;
        const bool partial = is_partial(key0);
        f16_t* dk = sk + (u & 1) * (BN * HD);
        f16_t* dv = sv + (u & 1) * (BN * HD);
#pragma unroll
        for (int i = 0; i < NCH; i++) {
            const uint32_t p = i * 256 + tid;
            if (edge) {
                const int32_t key = key0 + (int32_t)(p / CPR);
                if (key < sp.lo || key >= sp.hi) rv[i] = u32x4{0u, 0u, 0u, 0u};
            }
            if (partial && att_nonfinite(rv[i])) {
                odd = true;
                rv[i] = att_clear_nonfinite(rv[i]);
            }
            *(u32x4*)(dk + p * 8) = rk[i];
            *(u32x4*)(dv + p * 8) = rv[i];
        }
    };
    if (sp.u0 < sp.u1) {
        look(sp.u0);
        fetch();
        if (sp.u0 + 1 < sp.u1) look(sp.u0 + 1);
        stage(sp.u0);
    }
    __syncthreads();
    for (uint32_t u = sp.u0; u < sp.u1; u++) {
        if (u + 1 < sp.u1) {
            fetch();
            if (u + 2 < sp.u1) look(u + 2);
        }
        const f16_t* tk = sk + (u & 1) * (BN * HD);
        const f16_t* tv = sv + (u & 1) * (BN * HD);
        const int32_t key0 = (int32_t)(u * BN);
        const bool active = wave_on && key0 <= wpos1 && (!a.window || key0 + BN - 1 > wpos0 - (int32_t)a.window);
        f16x8 ph[KB][2], pl[KB][2];
        if (active) {
            f32x16 s[KB];
#pragma unroll
            for (int b = 0; b < KB; b++) {
#pragma unroll
                for (int j = 0; j < 16; j++) s[b][j] = 0.f;
                const uint32_t r = b * 32 + n32;
#pragma unroll
                for (int i = 0; i < KF; i++) {
                    const f16x8 kf = *(const f16x8*)(tk + r * HD + (((i * 2 + hf) ^ att_swz<HD>(r)) * 8));
#pragma unroll
                    for (int t = 0; t < NQ; t++) s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[i][t], s[b], 0, 0, 0);
                }
            }
            if (key0 + BN - 1 > wpos0 || (a.window && key0 <= wpos1 - (int32_t)a.window)) {
#pragma unroll
                for (int b = 0; b < KB; b++)
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        const int32_t key = key0 + b * 32 + 8 * (j >> 2) + 4 * (int32_t)hf + (j & 3);
                        if (key > pos || (a.window && key <= pos_lo)) s[b][j] = NEG_INF;
                    }
            }
            float mx = NEG_INF;
#pragma unroll
            for (int b = 0; b < KB; b++)
#pragma unroll
                for (int j = 0; j < 16; j++) mx = fmaxf(mx, s[b][j]);
            mx = max_xor<32>(mx) * c;
            const float mn = fmaxf(m, mx), ms = mn == NEG_INF ? 0.f : mn;
            if (__any(mn > m)) {
                const float alpha = exp2_hw(m - ms);
                l *= alpha;
#pragma unroll
                for (int i = 0; i < HB; i++) o[i] *= alpha;
                m = mn;
            }
            const float sub = kProbShift - ms;
#pragma unroll
            for (int b = 0; b < KB; b++)
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    const float p = exp2_hw(__builtin_fmaf(s[b][j], c, sub));
                    l += p;
                    const f16_t h = (f16_t)p;
                    ph[b][j >> 3][j & 7] = h;
                    if constexpr (NQ == 2) pl[b][j >> 3][j & 7] = (f16_t)(p - (float)h);
                }
        }
        if (active) {
            const uint32_t l16 = lane & 15, half = (lane >> 4) & 1;
#pragma unroll
            for (int hb = 0; hb < HB; hb++)
#pragma unroll
                for (int b = 0; b < KB; b++)
#pragma unroll
                    for (int q = 0; q < 2; q++) {
                        union {
                            s16x4 h[2];
                            f16x8 v;
                        } vf;
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const uint32_t r = b * 32 + q * 16 + e * 8 + hf * 4 + (l16 >> 2);
                            const uint32_t ch = hb * 4 + half * 2 + ((l16 & 3) >> 1);
                            const f16_t* p = tv + r * HD + ((ch ^ att_swz<HD>(r)) * 8) + (l16 & 1) * 4;
                            vf.h[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
                        }
                        o[hb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf.v, ph[b][q], o[hb], 0, 0, 0);
                        if constexpr (NQ == 2) o[hb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf.v, pl[b][q], o[hb], 0, 0, 0);
                    }
        }
        if (u + 1 < sp.u1) stage(u + 1);
        __syncthreads();
    }
    // A value of V that is not finite, in a unit that some rows see only in part, was cleared on its way in, so that it
    // met no weight of zero; the rows that do see it get it here, as it is (any weight above zero leaves it so).
    if (__syncthreads_or(odd)) {
#pragma unroll 1
        for (uint32_t u = sp.u0; u < sp.u1; u++) {
            if (!is_partial((int32_t)(u * BN))) continue;
#pragma unroll 1
            for (int32_t key = (int32_t)(u * BN); key < (int32_t)(u * BN) + BN; key++) {
                if (key < sp.lo || key > pos || (a.window && key <= pos_lo)) continue;
                const f16_t* p = vb + (uint64_t)att_row(a, tab, key, sp.lo, sp.hi) * kv_stride + 4 * hf;
#pragma unroll
                for (int hb = 0; hb < HB; hb++)
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        const f16x4 t = *(const f16x4*)(p + hb * 32 + 2 * j);
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (!(__builtin_fabsf((float)t[e]) < __builtin_inff())) o[hb][j + e] += (float)t[e];
                    }
            }
        }
    }
    l = sum_xor<32>(l);
    if (!on) return;
    if (it.s.parts > 1) {
        const uint32_t r = wave * 32 + n32;
        float* part = a.part + ((uint64_t)it.slot * H + kvh) * ((uint64_t)APK_ATT_CHUNK_ROWS * (HD + 2));
#pragma unroll
        for (int hb = 0; hb < HB; hb++)
#pragma unroll
            for (int j = 0; j < 16; j += 4)
                *(f32x4*)(part + r * HD + hb * 32 + 8 * (j >> 2) + 4 * hf) = f32x4{o[hb][j], o[hb][j + 1], o[hb][j + 2], o[hb][j + 3]};
        if (hf == 0) {
            part[APK_ATT_CHUNK_ROWS * HD + r] = m;
            part[APK_ATT_CHUNK_ROWS * (HD + 1) + r] = l;
        }
        return;
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    T* out = (T*)a.out + qat;
#pragma unroll
    for (int hb = 0; hb < HB; hb++)
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            float t[4] = {o[hb][j] * inv, o[hb][j + 1] * inv, o[hb][j + 2] * inv, o[hb][j + 3] * inv};
            att_store4<T>(out + hb * 32 + 8 * (j >> 2) + 4 * hf, t);
        }
}
#define ATTEND_CHUNK(T, t, HD, BN, WPE)                                                                              extern "C" __global__ __launch_bounds__(256, WPE) void apk_attend_chunk_##t##_hd##HD(apk_attend_args a) {            attend_chunk_body<T, HD, BN>(a, (f16_t*)att_smem);                                                           }
ATTEND_CHUNK(f16_t, f16, 64, 64, 2)
ATTEND_CHUNK(f16_t, f16, 128, 64, 2)
ATTEND_CHUNK(f16_t, f16, 256, 32, 1)
ATTEND_CHUNK(float, f32, 64, 64, 2)
ATTEND_CHUNK(float, f32, 128, 64, 1)
ATTEND_CHUNK(float, f32, 256, 32, 1)

// ------------------------------------------------------------------------------------------- joining the parts
// The tiles that were cut, and only those: a wave (WPR = 1) or a workgroup of four (WPR = 4: single tokens, few rows of
// many parts) per row.  Bound by its launch.
template <typename T, int WPR>
DEV void attend_join_body(const apk_attend_args& a) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t per_tile = WPR == 4 ? a.tile_rows : a.tile_rows / 4;  // workgroups of a tile
    const uint32_t H = a.n_kv * a.head_tiles, t = blockIdx.x / per_tile;
    att_item it;
    if (!att_find<true>(a, t / H, it)) return;
    const uint32_t hh = t % H, kvh = hh / a.head_tiles, ht = hh % a.head_tiles, hd = a.hd;
    const uint32_t r = WPR == 4 ? blockIdx.x % per_tile : (blockIdx.x % per_tile) * 4 + wave;
    uint64_t qat;
    if (a.q_off) {
        const uint64_t flat = (uint64_t)it.tile * a.tile_rows + r;
        if (flat >= (uint64_t)it.s.m * a.group) return;
        qat = ((uint64_t)(it.s.row0 + (uint32_t)(flat / a.group)) * a.n_q + kvh * a.group + (uint32_t)(flat % a.group)) * hd;
    } else {
        if (ht * APK_ATT_TOKEN_ROWS + r >= a.group) return;
        qat = ((uint64_t)it.s.row0 * a.n_q + kvh * a.group + ht * APK_ATT_TOKEN_ROWS + r) * hd;
    }
    const uint32_t parts = it.s.parts;
    const uint64_t slot_floats = (uint64_t)a.tile_rows * (hd + 2);
    const float* base = a.part + ((uint64_t)it.slot * H + hh) * slot_floats;
    const uint64_t step = (uint64_t)H * slot_floats;
    const float* mp = base + (uint64_t)a.tile_rows * hd + r;
    float M = NEG_INF;
    for (uint32_t p = lane; p < parts; p += 64) M = fmaxf(M, mp[p * step]);
    M = wave_max_f32(M);
    const float Ms = M == NEG_INF ? 0.f : M;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
    const uint32_t col = lane * 4;
    const bool on = col < hd;
#pragma unroll 4
    for (uint32_t p = WPR == 1 ? 0 : wave; p < parts; p += WPR) {
        const float w = exp2_hw(mp[p * step] - Ms);
        l = __builtin_fmaf(mp[p * step + a.tile_rows], w, l);
        const f32x4 v = *(const f32x4*)(base + p * step + (uint64_t)r * hd + (on ? col : 0));
        acc.x = __builtin_fmaf(v.x, w, acc.x);
        acc.y = __builtin_fmaf(v.y, w, acc.y);
        acc.z = __builtin_fmaf(v.z, w, acc.z);
        acc.w = __builtin_fmaf(v.w, w, acc.w);
    }
    if constexpr (WPR == 4) {
        __shared__ f32x4 so[4][64];
        __shared__ float sl[4];
        so[wave][lane] = acc;
        if (lane == 0) sl[wave] = l;
        __syncthreads();
        if (wave) return;
        acc = (so[0][lane] + so[1][lane]) + (so[2][lane] + so[3][lane]);
        l = (sl[0] + sl[1]) + (sl[2] + sl[3]);
    }
    if (on) {
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
        float v[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
        att_store4<T>((T*)a.out + qat + col, v);
    }
}
extern "C" __global__ __launch_bounds__(256) void apk_attend_join_f16_w1(apk_attend_args a) { attend_join_body<f16_t, 1>(a); }
extern "C" __global__ __launch_bounds__(256) void apk_attend_join_f32_w1(apk_attend_args a) { attend_join_body<float, 1>(a); }
extern "C" __global__ __launch_bounds__(256) void apk_attend_join_f16_w4(apk_attend_args a) { attend_join_body<f16_t, 4>(a); }
extern "C" __global__ __launch_bounds__(256) void apk_attend_join_f32_w4(apk_attend_args a) { attend_join_body<float, 4>(a); }

// ------------------------------------------------------------------------------------------- any head size
// A workgroup of four waves per (row, query head), element by element: heads of other sizes than 64, 128 and 256 (up to
// 1024).  A wave takes blocks of 64 keys in turn, a key a lane for the scores, then a channel a lane for the values.
template <typename T>
DEV void attend_generic_body(const apk_attend_args& a, float* smem) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hd = a.hd;
    const uint32_t row = blockIdx.x / a.n_q, h = blockIdx.x % a.n_q, kvh = h / a.group;
    att_seq s = {0, 0, 0, 0, 0, 1, 0};
    uint32_t seq = 0;
    bool found = false;
    for (uint32_t base = 0; base < a.n_seq && !found; base += 64) {
        const uint32_t i = base + lane;
        att_seq t = {0, 0, 0, 0, 0, 1, 0};
        if (i < a.n_seq) t = att_load_seq(a, i);
        const uint64_t hit = __ballot(row >= t.row0 && row - t.row0 < t.m);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            found = true;
            seq = base + (uint32_t)l;
            s.row0 = rl(t.row0, l);
            s.p0 = (int32_t)rl((uint32_t)t.p0, l);
        }
    }
    if (!found) return;
    const int32_t pos = s.p0 + (int32_t)(row - s.row0);
    const int32_t hi = pos + 1, lo = a.window ? max(0, pos - (int32_t)a.window + 1) : 0;
    const uint32_t* tab = a.table + (uint64_t)seq * a.max_pages;
    const uint64_t kv_stride = (uint64_t)a.n_kv * hd;
    const f16_t* kb = (const f16_t*)a.k + (uint64_t)kvh * hd;
    const f16_t* vb = (const f16_t*)a.v + (uint64_t)kvh * hd;
    const uint64_t qat = ((uint64_t)row * a.n_q + h) * hd;
    float* sq = smem;             // [hd]
    float* so = smem + hd;        // [4][hd]
    float* sml = smem + 5 * hd;   // [4][2]
    for (uint32_t i = threadIdx.x; i < hd; i += 256) sq[i] = (float)((const T*)a.q)[qat + i] * a.sign;
    __syncthreads();
    float o[16];
#pragma unroll
    for (int i = 0; i < 16; i++) o[i] = 0.f;
    float m = NEG_INF, l = 0.f;
    for (int32_t k0 = lo + (int32_t)wave * 64; k0 < hi; k0 += 256) {
        const int32_t key = k0 + (int32_t)lane;
        const uint32_t r = att_row(a, tab, key, lo, hi);
        float x = NEG_INF;
        if (key < hi) {
            float d = 0.f;
            const f16_t* kr = kb + (uint64_t)r * kv_stride;
            for (uint32_t i = 0; i < hd; i++) d = __builtin_fmaf((float)kr[i], sq[i], d);
            x = d * a.c;
        }
        const float mn = fmaxf(m, wave_max_f32(x)), ms = mn == NEG_INF ? 0.f : mn;
        const float alpha = exp2_hw(m - ms), p = exp2_hw(x - ms);
        m = mn;
        l = l * alpha + p;
#pragma unroll
        for (int i = 0; i < 16; i++) o[i] *= alpha;
        const int cnt = min(64, hi - k0);
        for (int j = 0; j < cnt; j++) {
            const float pj = __builtin_bit_cast(float, rl(__builtin_bit_cast(uint32_t, p), j));
            const f16_t* vr = vb + (uint64_t)rl(r, j) * kv_stride;
#pragma unroll
            for (int i = 0; i < 16; i++)
                if (i * 64 + lane < hd) o[i] = __builtin_fmaf((float)vr[i * 64 + lane], pj, o[i]);
        }
    }
    l = group_sum<64>(l);
#pragma unroll
    for (int i = 0; i < 16; i++)
        if (i * 64 + lane < hd) so[wave * hd + i * 64 + lane] = o[i];
    if (lane == 0) {
        sml[wave * 2] = m;
        sml[wave * 2 + 1] = l;
    }
    __syncthreads();
    const float M = fmaxf(fmaxf(sml[0], sml[2]), fmaxf(sml[4], sml[6])), Ms = M == NEG_INF ? 0.f : M;
    float f[4], ls = 0.f;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        f[w] = exp2_hw(sml[w * 2] - Ms);
        ls += sml[w * 2 + 1] * f[w];
    }
    const float inv = ls > 0.f ? 1.f / ls : (ls == 0.f ? 0.f : ls);
    for (uint32_t i = threadIdx.x; i < hd; i += 256) {
        const float v = (so[i] * f[0] + so[hd + i] * f[1]) + (so[2 * hd + i] * f[2] + so[3 * hd + i] * f[3]);
        ((T*)a.out)[qat + i] = (T)(v * inv);
    }
}
extern "C" __global__ __launch_bounds__(256) void apk_attend_any_f16(apk_attend_args a) { attend_generic_body<f16_t>(a, att_smem); }
extern "C" __global__ __launch_bounds__(256) void apk_attend_any_f32(apk_attend_args a) { attend_generic_body<float>(a, att_smem); }
