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
// activations a query element is the sum of two fp16 values, its row scaled by a power of two first: 22 bits of it, or 2^-38 of
// the row's largest magnitude where that is more.
//
// Probabilities are 2^(x_j - r + a constant), r a reference near the largest x_j, as fp16 values: below 2^16, with 11 bits from
// 2^-14 on and steps of 2^-24 below.  What they keep of a small weight goes by where r lies:
// * Few rows: two fp16 values, the second one 2^11 times the rest that the first leaves, its product with V added with
//   2^-11: 22 bits, of weights down to 2^-28 of the largest key's, 2^-50 of that one below (r stays within 2 of the running
//   maximum, at 2^14).  The launch is bound by memory: a second product costs nothing that shows (fp16 rows, 64 sequences of
//   6000 keys: 277 us with it and without).
// * Chunks: one fp16 value for fp16 rows (2^-11), the sum of two for f32 rows (2^-22), plain, both added up in the same place.
//   r follows the largest x_j of the unit of keys, down as well as up: that one lies at 2^-3 at least, so that a weight that is far
//   smaller than the largest of its unit is off by 2^-22 of that one, whatever came before.  With r the running maximum
//   all keys behind a dominant one were held to 2^-33 of it, and where that key's value is small (a sink) nothing else is
//   in the result.  r comes down at once the first times and once in 8 units then, so that scores that jump up and down
//   all along do not cost a rescaling each time; they are held to 2^-33 of the largest meanwhile.  (512 tokens over 32000 keys,
//   us with the running maximum / this way: fp16, heads of 64 420 / 420, of 128 596 / 601, of 256 1480 / 1479, f32 of 128 998 / 989;
//   with scores three times as wide 604 / 615 and 983 / 1024; coming down freely 677 and 1197 there.  A second product for
//   fp16 rows: 944 for 603.  The second value scaled as for few rows, in accumulators of its own: f32 heads of 64 6 % more, of
//   128 43 %, of 256 three times as long, for want of registers.)
#pragma once
#include <type_traits>
#include <utility>

#include "../apk_attend.h"

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

static constexpr float kLog2e = 1.44269504088896341f;
// few rows: r at 2^14, moved up where a maximum is more than 2 times larger; the factor of the second values
static constexpr float kFewShift = 14.0f, kFewLag = 1.0f, kLowUp = 2048.0f, kLowDown = 1.0f / 2048.0f;
// chunks: r at 2^6.  Where a block's maximum is 2^9 times larger r moves to 2^2 below it, where it is 2^9 times smaller to 2^6
// above it (the next ones may be larger); not down to one 2^40 below the largest met, which counts for nothing, so that sums
// stay in range.  A move takes 8 units of keys from an account that begins with three moves; down only what is on it.
static constexpr float kMid = 6.0f, kReach = 9.0f, kAbove = 2.0f, kRoom = 6.0f, kDepth = 40.0f;
static constexpr int32_t kMoves = 3, kMoveUnits = 8;
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
// A tile is tile_rows flat rows (token * group + head of the group) of one sequence and kv head, its work the units of keys
// that its rows see.  The lengths are on the device, so each workgroup works its own place out: two short passes of a wave
// over the sequences (sums and prefix sums by DPP).  The tiles that were cut are listed in the scratch for the launch that
// joins their parts.
// Chunks (att_find): a workgroup per tile, the heaviest first; where there are too few tiles to fill the chip, the tiles of
// a sequence are cut into as many parts as bring the launch to about `target` workgroups, of at least unit_min units.
// Few rows (att_share): all units in one line, cut into `target` equal pieces, one for each workgroup, which goes through
// the tiles its piece touches.  Such launches are streams of the cache: equal pieces end together whatever the lengths are.
struct att_seq {
    uint32_t row0, m;  // first row, rows
    int32_t n, p0;     // keys, position of the first row
    uint32_t tiles, umax, parts;
};
struct att_item {
    uint32_t seq, tile, part, slot;  // slot: of this part, among all parts of cut tiles
    att_seq s;
};
DEV att_seq att_load_seq(const apk_attend_args& a, uint32_t i) {
    att_seq s = {0, 0, 0, 0, 0, 0, 1};
    if (i >= a.n_seq) return s;
    uint32_t n = a.kv_len[i];
    uint32_t r0 = i, r1 = i + 1, bad = 0;
    if (a.q_off) {
        r0 = a.q_off[i];
        r1 = a.q_off[i + 1];
        if (r1 > a.rows || r0 > r1) {
            bad = APK_FAULT_ROW_RANGE;
            r1 = r1 < a.rows ? r1 : a.rows;
            r0 = r0 < r1 ? r0 : r1;
        }
    }
    const uint32_t cap = a.max_pages * a.page;  // at most 2^30
    if (n > cap) {
        n = cap;
        bad |= APK_FAULT_CACHE_RANGE;
    }
    if (bad) atomicOr(a.fault, bad);
    s.row0 = r0;
    s.m = r1 - r0;
    s.n = (int32_t)n;
    s.p0 = (int32_t)n - (int32_t)s.m;
    s.tiles = (s.m * a.group + a.tile_rows - 1) >> a.tile_shift;  // the host holds rows * group below 2^31
    uint32_t span = n;
    if (a.window) {  // keys that the rows of one tile see between them
        const uint64_t w = (uint64_t)a.window + a.tile_rows / a.group + 1 + a.unit;
        if (w < span) span = (uint32_t)w;
    }
    s.umax = (span + a.unit - 1) >> a.unit_shift;
    if (s.umax == 0) s.umax = 1;  // rows without keys are work too: they get zeros
    if (a.whole_units) s.umax = a.whole_units;
    return s;
}
DEV uint32_t rl(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }
template <int CTRL, int ROWS> DEV uint32_t dpp_add(uint32_t v) {
    return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, true);
}
DEV uint32_t wave_scan_u32(uint32_t v) {  // inclusive sums over the lanes
    v = dpp_add<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8
    v = dpp_add<0x112, 0xf>(v);
    v = dpp_add<0x114, 0xf>(v);
    v = dpp_add<0x118, 0xf>(v);
    v = dpp_add<0x142, 0xa>(v);  // row_bcast 15, 31
    v = dpp_add<0x143, 0xc>(v);
    return v;
}
// Units a part has at least, so that at most `target` workgroups' worth of parts comes of cutting.  Equal shares of all
// units would be parts of c; but a tile is cut into equal parts, so that there are more of them, and what is more than
// `target` takes a second round of the chip.  Of c, 9/8 c .. 15/8 c the first that needs no second round.  (Sums of whole
// numbers in double: exact, and the same in every wave.  16 sequences of 1 to 7 drafts over 500 to 8000
// keys: 81 us by equal shares, 69 this way.  Sequences sorted by their length first: no gain above 2 %, and 7 us for 64.)
DEV uint32_t att_parts(const att_seq& s, uint32_t c) { return s.umax > c ? (s.umax + c - 1) / c : 1u; }
DEV uint32_t att_units_per_part(const apk_attend_args& a, const att_seq& first) {
    const uint32_t lane = threadIdx.x & 63;
    double u = (double)first.tiles * (double)first.umax, tiles = (double)first.tiles;
    for (uint32_t i = 64 + lane; i < a.n_seq; i += 64) {
        const att_seq s = att_load_seq(a, i);
        u += (double)s.tiles * (double)s.umax;
        tiles += (double)s.tiles;
    }
    const double hb = (double)(a.n_kv / a.heads), t = group_sum<64>(tiles) * hb;
    u = group_sum<64>(u) * hb;
    const double cd = ceil(u / (double)a.target);
    const uint32_t c = cd > (double)a.unit_min ? (cd < 1073741824.0 ? (uint32_t)cd : 1073741824u) : a.unit_min;
    if (t >= (double)a.target) return c;
    for (uint32_t k = 0; k < 8; k++) {
        const uint32_t ck = c + c / 8 * k + c % 8 * k / 8;
        double n = (double)first.tiles * (double)att_parts(first, ck);
        for (uint32_t i = 64 + lane; i < a.n_seq; i += 64) {
            const att_seq s = att_load_seq(a, i);
            n += (double)s.tiles * (double)att_parts(s, ck);
        }
        if (group_sum<64>(n) * hb <= (double)a.target) return ck;
    }
    return c;
}
// The tile and part that item `pg` (0, 1, ...; without the kv heads) of the launch is; false: past the last one.
DEV bool att_find(const apk_attend_args& a, uint32_t pg, att_item& it) {
    const uint32_t lane = threadIdx.x & 63;
    att_seq s = att_load_seq(a, lane);
    const uint32_t c = att_units_per_part(a, s);
    uint32_t before = 0, slots = 0, tiles = 0;
    bool found = false;
    for (uint32_t base = 0;;) {
        s.parts = att_parts(s, c);
        const uint32_t cnt = s.tiles * s.parts, cut = s.parts > 1 ? cnt : 0, ct = s.parts > 1 ? s.tiles : 0;
        const uint32_t inc = before + wave_scan_u32(cnt), sinc = slots + wave_scan_u32(cut), tinc = tiles + wave_scan_u32(ct);
        const uint64_t hit = __ballot(inc > pg && inc - cnt <= pg);
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
            const uint32_t idx = pg - rl(inc - cnt, l), rank = idx / it.s.parts;
            it.tile = it.s.tiles - 1 - rank;  // the last rows see the most keys: they go first
            it.part = idx - rank * it.s.parts;
            it.slot = rl(sinc - cut, l) + idx;
            found = true;
            const uint32_t at = rl(tinc - ct, l) + rank;  // (lanes are read where all of them are active)
            if (it.s.parts > 1 && it.part == 0 && threadIdx.x == 0 && blockIdx.x % (a.n_kv / a.heads) == 0) {
                uint32_t* d = a.scratch + 16 + 8 * at;
                *(u32x4*)d = u32x4{it.s.row0, it.s.m, it.tile, it.s.parts};
                *(u32x4*)(d + 4) = u32x4{it.slot, it.slot + 1, 1, 0};
            }
            if (blockIdx.x) return true;  // the first workgroup goes on to the number of cut tiles
        }
        base += 64;
        before = rl(inc, 63);
        slots = rl(sinc, 63);
        tiles = rl(tinc, 63);
        if (base >= a.n_seq) {
            if (blockIdx.x == 0 && threadIdx.x == 0 && a.scratch) a.scratch[0] = tiles;
            return found;
        }
        s = att_load_seq(a, base + lane);
    }
}
DEV uint64_t rl64(uint64_t v, int lane) { return ((uint64_t)rl((uint32_t)(v >> 32), lane) << 32) | rl((uint32_t)v, lane); }
template <int CTRL, int ROWS> DEV uint64_t dpp_add64(uint64_t v) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xf, true);
    return v + (((uint64_t)hi << 32) | lo);
}
DEV uint64_t wave_scan_u64(uint64_t v) {
    v = dpp_add64<0x111, 0xf>(v);
    v = dpp_add64<0x112, 0xf>(v);
    v = dpp_add64<0x114, 0xf>(v);
    v = dpp_add64<0x118, 0xf>(v);
    v = dpp_add64<0x142, 0xa>(v);
    v = dpp_add64<0x143, 0xc>(v);
    return v;
}
// The line of all units as a wave keeps it: 64 sequences at a time, one a lane, with the sums up to and with each.
struct att_line {
    uint32_t base;      // the sequence of lane 0
    att_seq s;          // this lane's
    uint64_t end;       // where its units end
    uint32_t tiles;     // tiles up to and with it
};
DEV void att_line_load(const apk_attend_args& a, uint32_t base, uint64_t units, uint32_t tiles, att_line& ln) {
    ln.base = base;
    ln.s = att_load_seq(a, base + (threadIdx.x & 63));
    ln.end = units + wave_scan_u64((uint64_t)ln.s.tiles * ln.s.umax);
    ln.tiles = tiles + wave_scan_u32(ln.s.tiles);
}
// The piece [x0, x1) of the line that workgroup w of `target` takes; empty for workgroups that are not needed.  The line
// is left at its beginning.  Returns the number of tiles.
DEV uint32_t att_share(const apk_attend_args& a, uint32_t w, uint64_t& x0, uint64_t& x1, uint64_t& share, att_line& ln) {
    att_line_load(a, 0, 0, 0, ln);
    uint64_t all = rl64(ln.end, 63);
    uint32_t tiles = rl(ln.tiles, 63);
    for (uint32_t base = 64; base < a.n_seq; base += 64) {
        att_line t;
        att_line_load(a, base, all, tiles, t);
        all = rl64(t.end, 63);
        tiles = rl(t.tiles, 63);
    }
    // (32-bit division where the numbers allow it)
    share = all < 0x80000000u ? ((uint32_t)all + a.target - 1) / a.target : (all + a.target - 1) / a.target;
    if (share < a.unit_min) share = a.unit_min;
    // (no tile is ever cut there, also where wrong row offsets make more tiles than the launch has workgroups)
    if (a.whole_units) share = (share + a.whole_units - 1) / a.whole_units * a.whole_units;
    x0 = min(all, share * w);
    x1 = min(all, x0 + share);
    return tiles;
}
// The tile that unit x of the line falls into (x does not go back), where its units begin, and its number among all tiles.
struct att_place {
    uint32_t seq, tile, number;
    uint64_t begin;
    att_seq s;
};
DEV void att_locate(const apk_attend_args& a, uint64_t x, att_line& ln, att_place& pl) {
    while (rl64(ln.end, 63) <= x && ln.base + 64 < a.n_seq) att_line_load(a, ln.base + 64, rl64(ln.end, 63), rl(ln.tiles, 63), ln);
    const uint64_t cnt = (uint64_t)ln.s.tiles * ln.s.umax;
    const int l = __builtin_ctzll(__ballot(ln.end > x && ln.end - cnt <= x) | (1ull << 63));
    pl.seq = ln.base + (uint32_t)l;
    pl.s.row0 = rl(ln.s.row0, l);
    pl.s.m = rl(ln.s.m, l);
    pl.s.n = (int32_t)rl((uint32_t)ln.s.n, l);
    pl.s.p0 = (int32_t)rl((uint32_t)ln.s.p0, l);
    pl.s.tiles = rl(ln.s.tiles, l);
    pl.s.umax = rl(ln.s.umax, l);
    pl.s.parts = 1;
    const uint64_t first = rl64(ln.end - cnt, l), off = x - first;
    pl.tile = off < 0x80000000u ? (uint32_t)off / pl.s.umax : (uint32_t)(off / pl.s.umax);
    pl.number = rl(ln.tiles - ln.s.tiles, l) + pl.tile;
    pl.begin = first + (uint64_t)pl.tile * pl.s.umax;
}
// What is the same in all lanes, told to the compiler, which then keeps it in scalar registers and its branches uniform.
DEV uint32_t uni(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }
DEV int32_t uni(int32_t v) { return __builtin_amdgcn_readfirstlane(v); }
DEV uint64_t uni(uint64_t v) { return ((uint64_t)uni((uint32_t)(v >> 32)) << 32) | uni((uint32_t)v); }
DEV void uni_seq(att_seq& s) {
    s.row0 = uni(s.row0);
    s.m = uni(s.m);
    s.n = uni(s.n);
    s.p0 = uni(s.p0);
    s.tiles = uni(s.tiles);
    s.parts = uni(s.parts);
    s.umax = uni(s.umax);
}
DEV float* att_part(const apk_attend_args& a, uint32_t slot, uint32_t kvh) {
    return (float*)((char*)a.scratch + APK_ATT_PART_AT) + ((uint64_t)slot * a.n_kv + kvh) * ((uint64_t)a.tile_rows * (a.hd + 2));
}
DEV float att_inverse(float l) { return l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l); }  // no key: zeros; NaN stays

// The keys [lo, hi) that any row of a tile sees (tok0 .. tok1: its first and last row of the sequence) and their units.
struct att_span {
    int32_t lo, hi;    // keys
    uint32_t u0, u1;   // units: keys [u0 * UNIT, u1 * UNIT)
};
template <int UNIT> DEV att_span att_tile_span(const apk_attend_args& a, const att_seq& s, uint32_t tok0, uint32_t tok1) {
    att_span r;
    r.lo = a.window ? max(0, s.p0 + (int32_t)tok0 - (int32_t)a.window + 1) : 0;
    r.hi = max(0, s.p0 + (int32_t)tok1 + 1);
    r.u0 = (uint32_t)r.lo / UNIT;
    r.u1 = max(r.u0, ((uint32_t)r.hi + UNIT - 1) / UNIT);
    return r;
}

// The cache row of a key in two steps, so that the table entry is under way while the loads issued before it are (loads
// return in order: an entry used at once would wait for all of them).  Keys outside [lo, hi) read row 0, whose values are
// not used; a table entry that names no page reads row 0 as well, and is reported once at the end.
struct att_entry {
    uint32_t e, off;
};
DEV att_entry att_look(const apk_attend_args& a, const uint32_t* tab, int32_t key, int32_t lo, int32_t hi) {
    uint32_t idx, off;
    const bool in = key >= lo && key < hi;
    split_key(a, in ? (uint32_t)key : 0u, idx, off);
    return {tab[idx], in ? off : 0xffffffffu};
}
DEV uint32_t att_row(const apk_attend_args& a, att_entry t, bool& bad) {
    const bool in = t.off != 0xffffffffu, ok = in && t.e < a.n_pages;
    bad |= in && !ok;
    return ok ? t.e * a.page + t.off : 0;
}
DEV void att_report(const apk_attend_args& a, bool bad) {
    if (bad) atomicOr(a.fault, APK_FAULT_CACHE_RANGE);
}

// ------------------------------------------------------------------------------------------- query fragments
// Eight consecutive elements of a query row, as they are loaded (zeros for a row that is not there) and as fp16: one
// fragment for fp16 rows, a high and a low one for f32 rows, whose elements are multiplied by `mul` (a power of two) first.
template <typename T> struct att_q;
template <> struct att_q<f16_t> {
    static constexpr int N = 1;
    typedef f16x8 raw_t;
    DEV raw_t load(const f16_t* p, bool on) { return on ? *(const f16x8*)p : f16x8{0, 0, 0, 0, 0, 0, 0, 0}; }
    DEV float absmax(raw_t) { return 0.f; }
    DEV void split(raw_t t, float mul, f16x8* f) { f[0] = mul < 0.f ? -t : t; }
};
template <> struct att_q<float> {
    static constexpr int N = 2;
    struct raw_t {
        f32x4 a, b;
    };
    DEV raw_t load(const float* p, bool on) {
        const f32x4 z = {0.f, 0.f, 0.f, 0.f};
        return {on ? *(const f32x4*)p : z, on ? *(const f32x4*)(p + 4) : z};
    }
    DEV float absmax(raw_t t) {
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 4; j++) m = fmaxf(m, fmaxf(__builtin_fabsf(t.a[j]), __builtin_fabsf(t.b[j])));
        return m;
    }
    DEV void split(raw_t t, float mul, f16x8* f) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float x = (j < 4 ? t.a[j & 3] : t.b[j & 3]) * mul;
            f[0][j] = (f16_t)x;
            f[1][j] = (f16_t)(x - (float)f[0][j]);
        }
    }
};
// The power of two that brings a row's largest magnitude to [2^13, 2^14) or, for the smallest ones, as near as 2^126 does,
// and its inverse; 1 for a row that is not finite.
DEV void att_q_scale(float mx, float& mul, float& inv) {
    const int e = (int)((__builtin_bit_cast(uint32_t, mx) >> 23) & 0xff);  // biased exponent
    int k = 127 + 13 - e;                                                  // multiply by 2^k
    if (e == 255) k = 0;
    k = k > 126 ? 126 : k < -126 ? -126 : k;
    mul = __builtin_bit_cast(float, (uint32_t)(127 + k) << 23);
    inv = __builtin_bit_cast(float, (uint32_t)(127 - k) << 23);
}
// What an f32 row's products are multiplied by: |scale| * log2(e) / its power of two, the exact product first, so that a scale and
// a row whose sizes undo each other lose nothing.  Kept a normal number: a masked score stays -inf when multiplied by it
// (with 0 it would be NaN), and a score of 0 stays 0.  The least one moves no weight: a row's products are below 2^40.
// (fp16 rows are not scaled: theirs is a.c, one number that stays in a scalar register.)
DEV float att_factor(const apk_attend_args& a, float inv) {
    return __builtin_amdgcn_fmed3f(a.scale * inv * kLog2e, __FLT_MIN__, __FLT_MAX__);
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

// ------------------------------------------------------------------------------------------- few rows
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
// Single tokens, and chunks of a few: tiles of 16 flat rows.  A workgroup of W waves takes `heads` kv heads of one tile
// and part, W / heads waves to a head, each of them blocks of 32 keys in turn; so a workgroup reads whole rows of the
// cache where there are W heads or more, and its waves need not be joined.  K and V go from memory straight to registers:
// a wave's K block is the first operand of 16x16x32 products as it lies (16 bytes of a key a lane), its V block becomes
// one by an in-lane transpose (8 keys x 8 channels a lane).  K of the next block is under way from the moment K of this
// one is used up, V likewise.  Bound by the stream of K and V: 131071 keys of 8 heads of 128 in 96 us (5.6 TB/s), 64
// sequences of 100 to 12000 keys in 280 us (5.8 TB/s), where reads in this pattern without any arithmetic reach 5.9 to
// 6.2.  Short caches are bound by the chain launch, length, table entry, K, V, joins: 13 us for 600 keys.
template <typename T, int HD, int W>
DEV void attend_few_body(const apk_attend_args& a, float* smem) {
    constexpr int KF = HD / 32;           // K fragments of 16 keys
    constexpr int CH = HD / 16;           // channels a lane holds of a V row
    constexpr int NQ = att_q<T>::N, R = 16;
    const uint32_t lane = threadIdx.x & 63, wave = (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n16 = lane & 15, g = lane >> 4;
    const uint32_t hblocks = a.n_kv / a.heads, WK = W / a.heads;
    const uint32_t kvh = blockIdx.x % hblocks * a.heads + wave % a.heads, wk = wave / a.heads, piece = blockIdx.x / hblocks;
    uint64_t x0, x1, share;
    att_line line;
    const uint32_t all_tiles = att_share(a, piece, x0, x1, share, line);
    x0 = uni(x0);
    x1 = uni(x1);
    share = uni(share);
    const bool lists = threadIdx.x == 0 && blockIdx.x % hblocks == 0 && a.scratch;
    if (lists && piece == 0) a.scratch[0] = a.list_tiles ? all_tiles : a.target;
    if (lists && !a.list_tiles) a.scratch[16 + 8 * piece + 3] = 0;  // no tile that goes on in the next piece, so far
    bool first_seg = true;
    for (uint64_t x = x0; x < x1; first_seg = false) {
    att_place it;
    att_locate(a, x, line, it);
    it.seq = uni(it.seq);
    it.tile = uni(it.tile);
    it.number = uni(it.number);
    it.begin = uni(it.begin);
    uni_seq(it.s);
    const uint64_t tile_end = it.begin + it.s.umax, seg_end = min(tile_end, x1);
    const bool split = it.begin < x || tile_end > x1;
    const uint32_t slot = 2 * piece + (first_seg ? 0 : 1);
    if (lists && it.begin == x) {  // the tile begins here: its parts are this one and the first segments of the next pieces
        uint32_t* d = a.scratch + 16 + 8 * (a.list_tiles ? it.number : piece);
        const uint32_t parts = split ? 1 + (uint32_t)((tile_end - x1 + share - 1) / share) : 0;
        if (a.list_tiles || split) {
            *(u32x4*)d = u32x4{it.s.row0, it.s.m, it.tile, parts};
            *(u32x4*)(d + 4) = u32x4{slot, 2 * (piece + 1), 2, 0};
        }
    }
    const uint32_t flat_n = it.s.m * a.group, flat0 = it.tile * R, rows_here = min(flat_n - flat0, (uint32_t)R);
    const uint32_t tok0 = uni(flat0 / a.group), tok1 = uni((flat0 + rows_here - 1) / a.group);
    att_span sp = att_tile_span<32>(a, it.s, tok0, tok1);
    sp.u1 = min(sp.u1, sp.u0 + (uint32_t)(seg_end - it.begin));
    sp.u0 = min(sp.u1, sp.u0 + (uint32_t)(x - it.begin));
    x = seg_end;
    const uint32_t* tab = a.table + (uint64_t)it.seq * a.max_pages;
    const uint32_t kv_stride = a.n_kv * HD;
    const f16_t* kb = (const f16_t*)a.k + (uint64_t)kvh * HD;
    const f16_t* vb = (const f16_t*)a.v + (uint64_t)kvh * HD;

    typename att_q<T>::raw_t qr[KF];
    const uint32_t flat = flat0 + n16, tok = flat / a.group;
    const bool on = n16 < rows_here;
    const uint64_t qat = on ? ((uint64_t)(it.s.row0 + tok) * a.n_q + kvh * a.group + flat % a.group) * HD : 0;
    const int32_t pos = on ? it.s.p0 + (int32_t)tok : -1;
#pragma unroll
    for (int s = 0; s < KF; s++) qr[s] = att_q<T>::load((const T*)a.q + qat + g * 8 + s * 32, on);
    float m = NEG_INF, l = 0.f;
    f32x4 o[CH];
#pragma unroll
    for (int i = 0; i < CH; i++) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};

    typedef uint32_t vrow_t __attribute__((ext_vector_type(CH / 2)));
    const int32_t k_end = min((int32_t)(sp.u1 * 32), sp.hi), k_lo = max(sp.lo, (int32_t)(sp.u0 * 32));
    const int32_t key_first = (int32_t)(sp.u0 * 32 + wk * 32), stride = (int32_t)(32 * WK);
    const int32_t tpos0 = it.s.p0 + (int32_t)tok0, tpos1 = it.s.p0 + (int32_t)tok1;
    // some row of the tile does not see all keys of this block
    auto is_partial = [&](int32_t key0) { return key0 + 31 > tpos0 || (a.window && key0 <= tpos1 - (int32_t)a.window); };
    f16x8 kf[2][KF];
    vrow_t vr[8];
    auto load_k = [&](uint32_t row) {
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const f16_t* p = kb + (uint64_t)__shfl(row, b * 16 + n16) * kv_stride + g * 8;
#pragma unroll
            for (int s = 0; s < KF; s++) kf[b][s] = *(const f16x8*)(p + s * 32);
        }
    };
    auto load_v = [&](uint32_t row) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const f16_t* p = vb + (uint64_t)__shfl(row, (j >> 2) * 16 + g * 4 + (j & 3)) * kv_stride;
            if constexpr (CH == 4) vr[j] = *(const vrow_t*)(p + n16 * 4);
            if constexpr (CH == 8) vr[j] = *(const vrow_t*)(p + n16 * 8);
            if constexpr (CH == 16) {
                const u32x4 x = *(const u32x4*)(p + n16 * 8), y = *(const u32x4*)(p + 128 + n16 * 8);
                vr[j] = vrow_t{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
            }
        }
    };
    auto look = [&](int32_t key) { return att_look(a, tab, key + (int32_t)(lane & 31), k_lo, k_end); };
    bool bad = false, odd = false;  // a table entry that names no page; a value of V that is not finite was cleared
    att_entry ahead = {0, 0};       // the table entries of the block after the one that is worked on
    int32_t key0 = key_first;
    if (key0 < k_end) {
        const att_entry t = look(key0);
        ahead = look(key0 + stride);
        const uint32_t row = att_row(a, t, bad);
        load_k(row);
        __builtin_amdgcn_sched_barrier(0);
        load_v(row);
        __builtin_amdgcn_sched_barrier(0);
    }
    f16x8 qf[KF][NQ];
    float mul = 1.f, inv = 1.f;
    if constexpr (NQ == 2) {
        float mx = 0.f;
#pragma unroll
        for (int s = 0; s < KF; s++) mx = fmaxf(mx, att_q<T>::absmax(qr[s]));
        att_q_scale(max_xor<32>(max_xor<16>(mx)), mul, inv);
    }
#pragma unroll
    for (int s = 0; s < KF; s++) att_q<T>::split(qr[s], mul * a.sign, qf[s]);
    const float c = NQ == 2 ? att_factor(a, inv) : a.c;
    while (key0 < k_end) {
        const int32_t next = key0 + stride;
        f32x4 s[2];
#pragma unroll
        for (int b = 0; b < 2; b++) {
            s[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < KF; i++)
#pragma unroll
                for (int t = 0; t < NQ; t++) s[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[b][i], qf[i][t], s[b], 0, 0, 0);
        }
        // (without a condition on there being a next block: behind the last one this reads row 0, and a condition here
        // makes the compiler copy what it loads, that is wait for it)
        const uint32_t nrow = att_row(a, ahead, bad);
        ahead = look(next + stride);
        load_k(nrow);
        __builtin_amdgcn_sched_barrier(0);  // K before V, so that K can be waited for with V under way
        const bool partial = key0 < k_lo || is_partial(key0);  // (a block that ends behind the last key is one)
        if (partial) {
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int32_t key = key0 + b * 16 + (int32_t)g * 4 + i;
                    if (key < k_lo || key > pos || (a.window && key <= pos - (int32_t)a.window)) s[b][i] = NEG_INF;
                }
        }
        f16x8 ph, pl;
        float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        mx = max_xor<32>(max_xor<16>(mx)) * c;
        if (__any(mx > m + kFewLag)) {
            const float mn = fmaxf(m, mx), alpha = mn == NEG_INF ? 1.f : exp2_hw(m - mn);
            l *= alpha;
#pragma unroll
            for (int i = 0; i < CH; i++) o[i] *= alpha;
            m = mn;
        }
        const float sub = m == NEG_INF ? 0.f : kFewShift - m;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float p = exp2_hw(__builtin_fmaf(s[j >> 2][j & 3], c, sub));
            l += p;
            ph[j] = (f16_t)p;
            pl[j] = (f16_t)((p - (float)ph[j]) * kLowUp);
        }
        if (partial) {  // keys that no row sees: zero; values that are not finite: see below
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int32_t key = key0 + (j >> 2) * 16 + (int32_t)g * 4 + (j & 3);
                if (key < k_lo || key >= k_end) vr[j] = (vrow_t)(0u);
#pragma unroll
                for (int w = 0; w < CH / 2; w++) {
                    const uint32_t t = vr[j][w];
                    const bool lo = (t & 0x7c00u) == 0x7c00u, hi = (t & 0x7c000000u) == 0x7c000000u;
                    odd |= lo || hi;
                    vr[j][w] = t & ((lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u));
                }
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
        load_v(nrow);
#pragma unroll
        for (int i = 0; i < CH; i++) {
            o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt[i], ph, o[i], 0, 0, 0);
            const f32x4 low = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt[i], pl, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
            for (int j = 0; j < 4; j++) o[i][j] = __builtin_fmaf(low[j], kLowDown, o[i][j]);
        }
        key0 = next;
        __builtin_amdgcn_sched_barrier(0);  // V is issued here, not at the head of the next round
    }
    att_report(a, bad);
    // o[ci][i]: row n16, channel chan(4 g + i, ci); heads of 256 channels hold two runs of eight, 128 apart
    auto chan = [&](int i, int ci) { return CH == 16 ? (ci >> 3) * 128 + ((int)g * 4 + i) * 8 + (ci & 7) : ((int)g * 4 + i) * CH + ci; };
    // A value of V that is not finite, in a block that some rows see only in part, was cleared on its way in, so that it
    // met no weight of zero; the rows that do see it get it here, as it is (any weight above zero leaves it so).
    if (__any(odd)) {
#pragma unroll 1
        for (int32_t k0 = key_first; k0 < k_end; k0 += stride) {
            if (!(k0 < k_lo || is_partial(k0))) continue;
#pragma unroll 1
            for (int32_t key = max(k0, k_lo); key < min(k0 + 32, k_end); key++) {
                bool no = false;
                const f16_t* p = vb + (uint64_t)att_row(a, att_look(a, tab, key, k_lo, k_end), no) * kv_stride;
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int ci = 0; ci < CH; ci++) {
                        const float x = (float)p[chan(i, ci)];
                        const bool nonfinite = !(__builtin_fabsf(x) < __builtin_inff());
                        if (nonfinite && key <= pos && !(a.window && key <= pos - (int32_t)a.window)) o[ci][i] += x;
                    }
            }
        }
    }
    l = sum_xor<32>(sum_xor<16>(l));
    float* part = att_part(a, split ? slot : 0, kvh);
    if (WK == 1) {  // a wave has the whole result of its head
        if (on) {
            const float f = split ? 1.f : att_inverse(l);
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int ci = 0; ci < CH; ci += 4) {
                    float t[4] = {o[ci][i] * f, o[ci + 1][i] * f, o[ci + 2][i] * f, o[ci + 3][i] * f};
                    if (split) io<float>::store(part + (uint64_t)n16 * HD + chan(i, ci), t);
                    else att_store4<T>((T*)a.out + qat + chan(i, ci), t);
                }
            if (split && g == 0) {
                part[R * HD + n16] = m;
                part[R * (HD + 1) + n16] = l;
            }
        }
        continue;
    }
    // join the waves of a head: their maxima, then the sums of the rescaled outputs
    const uint32_t RR = rows_here;
    float* sm_m = smem;              // [W][R]
    float* sm_l = smem + W * R;      // [W][R]
    float* sm_o = smem + 2 * W * R;  // [W][RR][HD]
    const uint32_t hl = wave % a.heads;  // the head's waves: hl, hl + heads, ...
    if (g == 0) sm_m[wave * R + n16] = m;
    __syncthreads();
    float M = NEG_INF;
    for (uint32_t w = hl; w < W; w += a.heads) M = fmaxf(M, sm_m[w * R + n16]);
    const float f = m == NEG_INF ? 0.f : exp2_hw(m - M);
    if (g == 0) sm_l[wave * R + n16] = l * f;
    if (on) {
        float* dst = sm_o + ((uint64_t)wave * RR + n16) * HD;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int ci = 0; ci < CH; ci += 4)
                *(f32x4*)(dst + chan(i, ci)) = f32x4{o[ci][i] * f, o[ci + 1][i] * f, o[ci + 2][i] * f, o[ci + 3][i] * f};
    }
    __syncthreads();
    const uint32_t kvh0 = blockIdx.x % hblocks * a.heads;
    for (uint32_t i = threadIdx.x; i < a.heads * RR * (HD / 4); i += W * 64) {
        const uint32_t col = i % (HD / 4) * 4, r = i / (HD / 4) % RR, h = i / (HD / 4) / RR;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        float ls = 0.f, mm = NEG_INF;
        for (uint32_t w = h; w < W; w += a.heads) {
            v += *(const f32x4*)(sm_o + ((uint64_t)w * RR + r) * HD + col);
            ls += sm_l[w * R + r];
            mm = fmaxf(mm, sm_m[w * R + r]);
        }
        if (split) {
            float* to = att_part(a, slot, kvh0 + h);
            *(f32x4*)(to + (uint64_t)r * HD + col) = v;
            if (col == 0) {
                to[R * HD + r] = mm;
                to[R * (HD + 1) + r] = ls;
            }
        } else {
            const float inv = att_inverse(ls);
            const uint32_t flat = flat0 + r;
            float t[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
            att_store4<T>((T*)a.out + ((uint64_t)(it.s.row0 + flat / a.group) * a.n_q + (kvh0 + h) * a.group + flat % a.group) * HD + col, t);
        }
    }
    __syncthreads();  // the next segment writes there again
    }
}
extern __shared__ float att_smem[];
#define ATTEND_FEW(HD, W)                                                                                          \
    extern "C" __global__ __launch_bounds__(W * 64, W / 4) void apk_attend_few_f16_hd##HD(apk_attend_args a) {     \
        attend_few_body<f16_t, HD, W>(a, att_smem);                                                                \
    }                                                                                                              \
    extern "C" __global__ __launch_bounds__(W * 64, W / 4) void apk_attend_few_f32_hd##HD(apk_attend_args a) {     \
        attend_few_body<float, HD, W>(a, att_smem);                                                                \
    }
ATTEND_FEW(64, 8)
ATTEND_FEW(128, 8)
ATTEND_FEW(256, 4)

// ------------------------------------------------------------------------------------------- chunks of new tokens
// One workgroup of four waves per (sequence, kv head, tile of 128 flat (token, head) rows, part of the keys); a wave holds 32
// rows.  Units of BN keys go through LDS, written there by the loads themselves (no registers in between) into one of two
// buffers while the unit in the other is worked on; one barrier a unit.  K rows are the first operand of 32x32x16 products
// as they lie; V comes out of LDS transposed (ds_read_b64_tr_b16), in the key order in which a lane holds its
// probabilities.  The 16-byte chunks of LDS row r are permuted by f(r), so that both kinds of reads meet all banks.
// Bound by the three that do not overlap fully, matrix instructions, LDS reads and exponentials, each near 2000 cycles for
// the units that the two workgroups of a CU (one for f32 heads of 128 and heads of 256) work on together: 512 tokens over
// 32000 keys, 64 / 8 heads of 128, fp16: 595 us, 0.9 PFLOP/s, where a large matrix product reaches 1.3; without the loads
// 15 % less, without the exponentials 17 % less.  64 rows a wave read LDS half as often, but leave one wave per SIMD,
// whose products and exponentials then wait for each other: 760 us.
template <int HD> DEV uint32_t att_swz(uint32_t r) {
    if constexpr (HD == 64) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    else return ((r & 3) << 2) | ((r >> 2) & 3);
}
typedef __attribute__((address_space(3))) char lds_t;
template <typename F, int... I> DEV void static_for_(F&& f, std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>()), ...); }
template <int N, typename F> DEV void static_for(F&& f) { static_for_(f, std::make_integer_sequence<int, N>()); }
// The value of lane J of this lane's run of 16.
template <int J> DEV uint32_t run_lane(uint32_t v) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x150 + J, 0xf, 0xf, true); }
// 16 bytes a lane from memory to LDS, lane l's to `at` + 16 l.  Counted by vmcnt like any load; the caller waits.
DEV void lds_load16(const void* g, uint32_t at) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g), "s"(at) : "memory");
}
DEV void lds_arrived() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}
template <typename T, int HD, int BN>
DEV void attend_chunk_body(const apk_attend_args& a, char* smem) {
    constexpr int KF = HD / 16, NQ = att_q<T>::N, KB = BN / 32, HB = HD / 32, CPR = HD / 8;
    constexpr int NCH = BN * CPR / 256;  // 16-byte chunks of K (and of V) a thread stages
    constexpr uint32_t BUF = BN * HD * 2;  // bytes of a unit's K or V; K in buffers 0 and 1, V in 2 and 3
    const uint32_t H = a.n_kv, tid = threadIdx.x, lane = tid & 63, n32 = lane & 31, hf = lane >> 5;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane(tid >> 6);
    lds_t* const lds = (lds_t*)smem;
    const uint32_t lds0 = (uint32_t)(uintptr_t)lds;
    att_item it;
    if (!att_find(a, blockIdx.x / H, it)) return;
    it.seq = uni(it.seq);
    it.tile = uni(it.tile);
    it.part = uni(it.part);
    it.slot = uni(it.slot);
    uni_seq(it.s);
    const uint32_t kvh = blockIdx.x % H;
    const uint32_t flat_n = it.s.m * a.group, flat0 = it.tile * APK_ATT_CHUNK_ROWS;
    const uint32_t tok0 = uni(flat0 / a.group), tok1 = uni((min(flat0 + APK_ATT_CHUNK_ROWS, flat_n) - 1) / a.group);
    att_span sp = att_tile_span<BN>(a, it.s, tok0, tok1);
    if (it.s.parts > 1) {
        const uint64_t nu = sp.u1 - sp.u0;
        const uint32_t first = sp.u0;
        sp.u0 = uni(first + (uint32_t)(nu * it.part / it.s.parts));
        sp.u1 = uni(first + (uint32_t)(nu * (it.part + 1) / it.s.parts));
    }
    const uint32_t* tab = a.table + (uint64_t)it.seq * a.max_pages;
    const uint32_t kv_stride = a.n_kv * HD;
    const f16_t* kb = (const f16_t*)a.k + (uint64_t)kvh * HD;
    const f16_t* vb = (const f16_t*)a.v + (uint64_t)kvh * HD;

    // this lane's row, and the first and last position of the wave's and the tile's rows
    const uint32_t flat = flat0 + wave * 32 + n32;
    const bool on = flat < flat_n;
    const uint32_t tok = flat / a.group, head = flat % a.group;
    // (no key behind the part counts: heads of 256 go through units in pairs, and the one behind an odd last one is the
    // next part's)
    const int32_t part_last = (int32_t)(sp.u1 * BN) - 1, row_pos = it.s.p0 + (int32_t)tok;
    const int32_t pos = on ? min(row_pos, part_last) : -1;
    const int32_t pos_lo = a.window ? row_pos - (int32_t)a.window : -1;  // keys above this one
    const bool wave_on = flat0 + wave * 32 < flat_n;
    const int32_t wpos0 = it.s.p0 + uni((int32_t)((flat0 + wave * 32) / a.group));
    const int32_t wpos1 = it.s.p0 + uni((int32_t)((min(flat0 + wave * 32 + 32, flat_n) - 1) / a.group));
    const int32_t tpos0 = min(it.s.p0 + (int32_t)tok0, part_last), tpos1 = it.s.p0 + (int32_t)tok1;
    const uint64_t qat = ((uint64_t)(it.s.row0 + tok) * a.n_q + kvh * a.group + head) * HD;

    // staging: thread t takes chunks t, t + 256, ... of a unit.  A lane looks one key up, a unit ahead; rows are handed round.
    bool bad = false, odd = false;  // a table entry that names no page; a value of V that is not finite was cleared
    // (thread t's chunk i is one of row (256 i + t) / CPR.  In a run of 16 lanes lane j < NCH * RPR looks up the row that
    // chunk j % NCH of the lanes 16 / RPR * (j / NCH) .. needs, and hands it to them.)
    constexpr int RPR = CPR < 16 ? 16 / CPR : 1;  // rows that 16 lanes touch
    static_assert(NCH * RPR <= 16, "rows of a run of lanes");
    att_entry ent;
    auto look = [&](uint32_t u) {
        const uint32_t j = lane & 15, i = j % NCH, h = j / NCH % RPR;
        ent = att_look(a, tab, (int32_t)(u * BN + (i * 256 + (tid & ~15u)) / CPR + h), sp.lo, sp.hi);
    };
    auto fetch = [&](uint32_t buf) {
        const uint32_t row = att_row(a, ent, bad);
        const uint32_t to = lds0 + buf * BUF + wave * 1024;
        static_for<NCH>([&](auto i_) {
            constexpr int i = decltype(i_)::value;
            const uint32_t r = (i * 256 + tid) / CPR, ch = (tid % CPR) ^ att_swz<HD>(r);
            uint32_t from = run_lane<i>(row);
            if constexpr (RPR == 2) {  // (both read by all lanes: a lane that is off hands nothing on)
                const uint32_t other = run_lane<NCH + i>(row);
                from = (lane & 8) ? other : from;
            }
            const uint64_t at = (uint64_t)from * kv_stride + ch * 8;
            lds_load16(kb + at, to + i * 4096);
            lds_load16(vb + at, to + i * 4096 + 2 * BUF);
        });
    };
    // some row of the tile does not see all keys of this unit
    auto is_partial = [&](int32_t key0) { return key0 + BN - 1 > tpos0 || (a.window && key0 <= tpos1 - (int32_t)a.window); };
    f16x8 qf[KF][NQ];
    float c = a.c;
    {
        typename att_q<T>::raw_t qr[KF];
        float mul = 1.f, inv = 1.f;
#pragma unroll
        for (int s = 0; s < KF; s++) qr[s] = att_q<T>::load((const T*)a.q + (on ? qat : 0) + s * 16 + hf * 8, on);
        if constexpr (NQ == 2) {
            float mx = 0.f;
#pragma unroll
            for (int s = 0; s < KF; s++) mx = fmaxf(mx, att_q<T>::absmax(qr[s]));
            att_q_scale(max_xor<32>(mx), mul, inv);
        }
#pragma unroll
        for (int s = 0; s < KF; s++) att_q<T>::split(qr[s], mul * a.sign, qf[s]);
        if constexpr (NQ == 2) c = att_factor(a, inv);
    }
    f32x16 o[HB];
#pragma unroll
    for (int i = 0; i < HB; i++)
#pragma unroll
        for (int j = 0; j < 16; j++) o[i][j] = 0.f;
    float m = NEG_INF, l = 0.f;
    // where this lane finds its fragments: K chunk 2 i + hf of row n32 (+ 32 b); V channels 32 hb + .. of four keys
    uint32_t ka[KF], va[HB][2];
#pragma unroll
    for (int i = 0; i < KF; i++) ka[i] = n32 * (HD * 2) + (((i * 2 + hf) ^ att_swz<HD>(n32)) * 16);
#pragma unroll
    for (int hb = 0; hb < HB; hb++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const uint32_t r = e * 8 + hf * 4 + ((lane & 15) >> 2), ch = hb * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
            va[hb][e] = r * (HD * 2) + ((ch ^ att_swz<HD>(r)) * 16) + (lane & 1) * 8;
        }

    f32x16 s[KB];
    f16x8 ph[KB][2], pl[KB][2];
    auto load_k = [&](int b, int i, uint32_t k_at) { return *(__attribute__((address_space(3))) f16x8*)(lds + (ka[i] + k_at + b * 32 * HD * 2)); };
    auto score = [&](int b, int i, f16x8 kf) {
        if (i == 0) {
#pragma unroll
            for (int j = 0; j < 16; j++) s[b][j] = 0.f;
        }
#pragma unroll
        for (int t = 0; t < NQ; t++) s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[i][t], s[b], 0, 0, 0);
    };
    // 16 keys of 32 channels, transposed.  (The compiler neither moves these reads nor lets others pass them: where they
    // stand is where they are issued.)
    auto load_v = [&](int hb, int b, int q, uint32_t v_at) {
        union {
            s16x4 h[2];
            f16x8 v;
        } t;
#pragma unroll
        for (int e = 0; e < 2; e++)
            t.h[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds + (va[hb][e] + v_at + (b * 32 + q * 16) * HD * 2)));
        return t.v;
    };
    auto value = [&](int hb, int b, int q, f16x8 vf) {
        o[hb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, ph[b][q], o[hb], 0, 0, 0);
        if constexpr (NQ == 2) o[hb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pl[b][q], o[hb], 0, 0, 0);
    };
    float neg = -1.f;  // hidden from the compiler, which then takes a fp16 factor into one instruction with the subtraction
    asm("" : "+v"(neg));
    auto weight = [&](int b, int j, float sub) {  // the block's scores 2 j and 2 j + 1
        const f32x2 p = {exp2_hw(__builtin_fmaf(s[b][2 * j], c, sub)), exp2_hw(__builtin_fmaf(s[b][2 * j + 1], c, sub))};
        l += p.x;
        l += p.y;
        const f16x2 h = __builtin_convertvector(p, f16x2);
        ph[b][j >> 2][2 * j & 7] = h.x;
        ph[b][j >> 2][(2 * j & 7) + 1] = h.y;
        if constexpr (NQ == 2) {
            const f32x2 d = {__builtin_fmaf((float)h.x, neg, p.x), __builtin_fmaf((float)h.y, neg, p.y)};
            const f16x2 e = __builtin_convertvector(d, f16x2);
            pl[b][j >> 2][2 * j & 7] = e.x;
            pl[b][j >> 2][(2 * j & 7) + 1] = e.y;
        }
    };
    auto shift = [&]() { return m == NEG_INF ? 0.f : kMid - m; };
    auto values = [&](int b, uint32_t v_at) {
        f16x8 vf[2][2];
#pragma unroll
        for (int q = 0; q < 2; q++) vf[0][q] = load_v(0, b, q, v_at);
#pragma unroll
        for (int hb = 0; hb < HB; hb++) {
            if (hb + 1 < HB) {
#pragma unroll
                for (int q = 0; q < 2; q++) vf[(hb + 1) & 1][q] = load_v(hb + 1, b, q, v_at);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int q = 0; q < 2; q++) value(hb, b, q, vf[hb & 1][q]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // Moves the reference to where block b of unit u asks for it, up or down; `again` redoes what refers to the old one.  Not
    // down (DOWN false) for block 1 where block 0 has weights already, which must stay in range: a row that sees block 0 has a
    // reference by it, and one that does not has none yet.  The largest maximum met at such times lies in LDS, read back by
    // its own lane; its address is made where it is used, since kept it would cost a register all the way.
    auto top_at = [&]() {
        uint32_t l;
        asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(l));
        return (__attribute__((address_space(3))) float*)(lds + (4 * BUF + wave * 256) + l * 4);
    };
    *top_at() = NEG_INF;
    int32_t spent = (int32_t)sp.u0 - kMoves * kMoveUnits;
    auto refer = [&](uint32_t u, int b, auto down_, auto&& again) {
        constexpr bool DOWN = decltype(down_)::value;
        float mx = NEG_INF;
#pragma unroll
        for (int j = 0; j < 16; j++) mx = fmaxf(mx, s[b][j]);
        mx = max_xor<32>(mx) * c;
        const float d = mx - m, below = (int32_t)u - spent >= kMoveUnits ? -kReach : NEG_INF;
        const bool low = DOWN && d < below && d != NEG_INF;  // (-inf: a row that sees nothing of the block)
        if (__builtin_expect(__any(d > kReach || low), 0)) {
            spent += kMoveUnits;
            __attribute__((address_space(3))) float* const top = top_at();
            const float t = *top;
            *top = fmaxf(t, mx);
            const float mn = low && mx > t - kDepth ? mx + kRoom : fmaxf(m, mx - kAbove), alpha = mn == NEG_INF ? 1.f : exp2_hw(m - mn);
            m = mn;
            again(alpha);
#pragma unroll
            for (int i = 0; i < HB; i++) o[i] *= alpha;
        }
    };
    // Keys that no row sees are cleared in V, so that what lies there meets no weight of zero; so are values that are not
    // finite, which the rows that see them get at the end.
    auto clear = [&](int32_t key0, uint32_t buf) {
#pragma unroll 1
        for (int i = 0; i < NCH; i++) {
            const uint32_t p = i * 256 + tid;
            const int32_t key = key0 + (int32_t)(p / CPR);
            __attribute__((address_space(3))) u32x4* at = (__attribute__((address_space(3))) u32x4*)(lds + (2 + buf) * BUF + p * 16);
            if (key < sp.lo || key >= sp.hi) {
                *at = u32x4{0u, 0u, 0u, 0u};
            } else {
                const u32x4 t = *at;
                if (att_nonfinite(t)) {
                    odd = true;
                    *at = att_clear_nonfinite(t);
                }
            }
        }
        __syncthreads();
    };
    auto hide = [&](int b, int32_t key0) {
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const int32_t key = key0 + b * 32 + 8 * (j >> 2) + 4 * (int32_t)hf + (j & 3);
            if (key > pos || (a.window && key <= pos_lo)) s[b][j] = NEG_INF;
        }
    };
    // A unit in buffer `buf`; unless ANY, one that all rows see whole.  Blocks of 32 keys, so that a wave has products and softmax to run
    // side by side: the products of block 1's scores next to block 0's exponentials, those of block 0's values next to
    // block 1's; LDS reads stand a few products before their use.  (fetch: behind the last unit it reads row 0, which is
    // not used; a condition would make the compiler wait for the table entries.)
    auto whole = [&](uint32_t u, auto buf_, auto any_) {
        constexpr bool ANY = decltype(any_)::value;
        const int32_t key0 = (int32_t)(u * BN);
        const bool partial = ANY && (key0 < sp.lo || is_partial(key0));
        constexpr uint32_t buf = decltype(buf_)::value, k_at = buf * BUF, v_at = (2 + buf) * BUF;
        constexpr int AHEAD = KF < 4 ? KF : 4;  // fragments read ahead
        f16x8 kf[KF];
#pragma unroll
        for (int i = 0; i < KF; i++) {
            kf[i] = load_k(0, i, k_at);
            if (i >= 2 * AHEAD - 1) {  // (all of them for heads of up to 128)
                score(0, i - (2 * AHEAD - 1), kf[i - (2 * AHEAD - 1)]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int i = KF < 2 * AHEAD ? 0 : KF - (2 * AHEAD - 1); i < KF; i++) score(0, i, kf[i]);
        fetch(1 - buf);
        look(u + 2);
#pragma unroll
        for (int i = 0; i < AHEAD; i++) kf[i] = load_k(1, i, k_at);
        if (partial) {
            clear(key0, buf);
            hide(0, key0);
        }
        refer(u, 0, std::true_type(), [&](float alpha) { l *= alpha; });
        float sub = shift();
        const float before = l;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < KF; i++) {
            if (i + AHEAD < KF) kf[i + AHEAD] = load_k(1, i + AHEAD, k_at);
            score(1, i, kf[i]);
#pragma unroll
            for (int j = i * 8 / KF; j < (i + 1) * 8 / KF; j++) weight(0, j, sub);
            __builtin_amdgcn_sched_barrier(0);
        }
        f16x8 vf[2][2];
#pragma unroll
        for (int q = 0; q < 2; q++) vf[0][q] = load_v(0, 0, q, v_at);
        if (partial) hide(1, key0);
        refer(u, 1, std::false_type(), [&](float alpha) {
            l = before * alpha;
            sub = shift();
#pragma unroll
            for (int j = 0; j < 8; j++) weight(0, j, sub);
        });
        sub = shift();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < 2 * HB; k++) {  // block 0's values, then block 1's
                const int hb = k % HB, b = k / HB, nhb = (k + 1) % HB, nb = (k + 1) / HB;
                if (k + 1 < 2 * HB) {
#pragma unroll
                    for (int q = 0; q < 2; q++) vf[(k + 1) & 1][q] = load_v(nhb, nb, q, v_at);
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    value(hb, b, q, vf[k & 1][q]);
                    if (b == 0) {
                        const int x = hb * 2 + q;
#pragma unroll
                        for (int j = x * 8 / (2 * HB); j < (x + 1) * 8 / (2 * HB); j++) weight(1, j, sub);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        lds_arrived();
    };
    // Any unit: rows that do not see all of it have scores of -inf.  Keys that no row sees are cleared in V, so that what
    // lies there meets no weight of zero; so are values that are not finite, which the rows that see them get at the end.
    auto part_seen = [&](uint32_t u, uint32_t buf) {
        fetch(1 - buf);
        look(u + 2);
        const int32_t key0 = (int32_t)(u * BN);
        if (key0 < sp.lo || is_partial(key0)) clear(key0, buf);
        if (wave_on && key0 <= wpos1 && (!a.window || key0 + BN - 1 > wpos0 - (int32_t)a.window)) {
#pragma unroll
            for (int b = 0; b < KB; b++) {
#pragma unroll
                for (int i = 0; i < KF; i++) score(b, i, load_k(b, i, buf * BUF));
                hide(b, key0);
                refer(u, b, std::true_type(), [&](float alpha) { l *= alpha; });
                const float sub = shift();
#pragma unroll
                for (int j = 0; j < 8; j++) weight(b, j, sub);
                values(b, (2 + buf) * BUF);
            }
        }
        lds_arrived();
    };
    // Units [f0, f1), an even number, are seen whole by all rows.  A wave without rows takes them by part_seen next to the
    // others' `whole`: both have to meet the same barriers there.  They do: one each at the end, and none in `clear`, which
    // runs only in units that some row does not see whole, for all waves or none.
    int32_t w0 = a.window ? tpos1 - (int32_t)a.window + 1 : 0, w1 = tpos0 + 1;
    uint32_t f0 = max(sp.u0, (uint32_t)max(0, (max(w0, sp.lo) + BN - 1) / BN)), f1 = min(sp.u1, (uint32_t)max(0, w1 / BN));
    f0 = min(f0, sp.u1);
    f1 = f1 > f0 && wave_on ? f0 + ((f1 - f0) & ~1u) : f0;
    // Heads of 256: two such bodies do not fit the registers (5 chunks of 333 to 2500 tokens: 608 us; 32 keys at a time, with
    // nothing side by side, 429), so one serves all units, in pairs from the first (318 us).
    constexpr bool ONE = HD == 256;
    const uint32_t parity = ONE ? sp.u0 & 1 : f0 & 1;
    if (sp.u0 < sp.u1) {
        look(sp.u0);
        fetch((sp.u0 ^ parity) & 1);
        look(sp.u0 + 1);
    }
    lds_arrived();
    uint32_t u = sp.u0, stop = f0;
    if constexpr (ONE) {
#pragma unroll 1
        for (; u < sp.u1; u += 2) {  // (behind the last unit: keys that no row sees)
            whole(u, std::integral_constant<uint32_t, 0>(), std::true_type());
            whole(u + 1, std::integral_constant<uint32_t, 1>(), std::true_type());
        }
    } else {
#pragma unroll 1
        for (;;) {
#pragma unroll 1
            for (; u < stop; u++) part_seen(u, (u ^ parity) & 1);
            if (u >= sp.u1) break;
            for (; u < f1; u += 2) {
                whole(u, std::integral_constant<uint32_t, 0>(), std::false_type());
                whole(u + 1, std::integral_constant<uint32_t, 1>(), std::false_type());
            }
            stop = sp.u1;
        }
    }
    att_report(a, bad);
    if (tid == 0) *(__attribute__((address_space(3))) uint32_t*)lds = 0;
    __syncthreads();
    if (odd) *(__attribute__((address_space(3))) uint32_t*)lds = 1;
    __syncthreads();
    if (*(__attribute__((address_space(3))) uint32_t*)lds) {
#pragma unroll 1
        for (uint32_t u = sp.u0; u < sp.u1; u++) {
            if (!is_partial((int32_t)(u * BN))) continue;
#pragma unroll 1
            for (int32_t key = (int32_t)(u * BN); key < (int32_t)(u * BN) + BN; key++) {
                if (key < sp.lo || key > pos || (a.window && key <= pos_lo)) continue;
                bool no = false;
                const f16_t* p = vb + (uint64_t)att_row(a, att_look(a, tab, key, sp.lo, sp.hi), no) * kv_stride + 4 * hf;
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
        float* part = att_part(a, it.slot, kvh);
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
    const float inv = att_inverse(l);
    T* out = (T*)a.out + qat;
#pragma unroll
    for (int hb = 0; hb < HB; hb++)
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            float t[4] = {o[hb][j] * inv, o[hb][j + 1] * inv, o[hb][j + 2] * inv, o[hb][j + 3] * inv};
            att_store4<T>(out + hb * 32 + 8 * (j >> 2) + 4 * hf, t);
        }
}
#define ATTEND_CHUNK(T, t, HD, BN, WPE)                                                                          \
    extern "C" __global__ __launch_bounds__(256, WPE) void apk_attend_chunk_##t##_hd##HD(apk_attend_args a) {    \
        attend_chunk_body<T, HD, BN>(a, (char*)att_smem);                                                        \
    }
ATTEND_CHUNK(f16_t, f16, 64, 64, 2)
ATTEND_CHUNK(f16_t, f16, 128, 64, 2)
ATTEND_CHUNK(f16_t, f16, 256, 64, 1)
ATTEND_CHUNK(float, f32, 64, 64, 2)
ATTEND_CHUNK(float, f32, 128, 64, 1)
ATTEND_CHUNK(float, f32, 256, 64, 1)

// ------------------------------------------------------------------------------------------- joining the parts
// The tiles that were cut: a workgroup of eight waves takes join_rows rows of one listed tile and kv head.  Bound by the
// round trips of the parts' loads, 4 us where little was cut, 15 for 256 tiles of 128 rows in two parts (34 MB).  Of up
// to 32 parts a wave joins a row on its own, hd / 4 lanes to a part; of more the whole workgroup shares the parts of one
// row after the other, so that the loads of all of them are under way together.
template <typename T>
DEV void attend_join_body(const apk_attend_args& a) {
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = (uint32_t)__builtin_amdgcn_readfirstlane(tid >> 6), hd = a.hd, R = a.tile_rows;
    const uint32_t per_tile = R / a.join_rows, x = blockIdx.x / per_tile;
    const uint32_t kvh = x % a.n_kv, j = x / a.n_kv, r0 = blockIdx.x % per_tile * a.join_rows;
    if (j >= a.scratch[0]) return;
    const uint32_t* d = a.scratch + 16 + 8 * j;
    const uint32_t row0 = d[0], m = d[1], tile = d[2], parts = d[3], slot0 = d[4], slot1 = d[5], step = d[6];
    const uint32_t flat0 = tile * R + r0, flat_n = m * a.group;
    if (parts < 2 || flat0 >= flat_n) return;
    const uint32_t rows = min(a.join_rows, flat_n - flat0);
    const uint64_t to = (uint64_t)a.n_kv * R * (hd + 2);  // floats from slot to slot
    const float* base = att_part(a, 0, kvh);
    auto slot_of = [&](uint32_t p) { return base + (uint64_t)(p ? slot1 + (p - 1) * step : slot0) * to; };
    auto finish = [&](uint32_t r, uint32_t col, f32x4 t, float l) {
        const uint32_t flat = flat0 + r;
        const float inv = att_inverse(l);
        float v[4] = {t.x * inv, t.y * inv, t.z * inv, t.w * inv};
        att_store4<T>((T*)a.out + ((uint64_t)(row0 + flat / a.group) * a.n_q + kvh * a.group + flat % a.group) * hd + col, v);
    };
    auto add = [](f32x4& acc, f32x4 v, float w) {
        acc.x = __builtin_fmaf(v.x, w, acc.x);
        acc.y = __builtin_fmaf(v.y, w, acc.y);
        acc.z = __builtin_fmaf(v.z, w, acc.z);
        acc.w = __builtin_fmaf(v.w, w, acc.w);
    };
    const uint32_t per = hd / 4, col = tid % per * 4;  // lanes of a part (16, 32 or 64)
    if (parts <= 32 && a.join_rows > 1) {
        const uint32_t groups = 64 / per, grp = lane / per;
        for (uint32_t r = wave; r < rows; r += 8) {
        float mp = NEG_INF, lp = 0.f;  // of part `lane`
        if (lane < parts) {
            const float* q = slot_of(lane) + (uint64_t)R * hd + r0 + r;
            mp = q[0];
            lp = q[R];
        }
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        float M = NEG_INF, w = 0.f;
        for (uint32_t p0 = 0; p0 < parts; p0 += 4 * groups) {
            f32x4 v[4];
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] = *(const f32x4*)(slot_of(min(p0 + k * groups + grp, parts - 1)) + (uint64_t)(r0 + r) * hd + col);
            if (p0 == 0) {
                M = wave_max_f32(mp);
                w = exp2_hw(mp - (M == NEG_INF ? 0.f : M));
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const uint32_t p = p0 + k * groups + grp;
                const float wp = __shfl(w, p & 63);
                if (p < parts) add(acc, v[k], wp);
            }
        }
        const float l = group_sum<64>(lane < parts ? lp * w : 0.f);
        for (uint32_t g = per; g < 64; g <<= 1) {
            acc.x += __shfl_xor(acc.x, g);
            acc.y += __shfl_xor(acc.y, g);
            acc.z += __shfl_xor(acc.z, g);
            acc.w += __shfl_xor(acc.w, g);
        }
        if (grp == 0) finish(r, col, acc, l);
        }
        return;
    }
    const uint32_t groups = 512 / per, grp = tid / per;
    __shared__ float sw[512], sred[8];
    __shared__ f32x4 so[512];
    for (uint32_t r = 0; r < rows; r++) {
        float M = NEG_INF;
        for (uint32_t p = tid; p < parts; p += 512) M = fmaxf(M, slot_of(p)[(uint64_t)R * hd + r0 + r]);
        M = wave_max_f32(M);
        if (lane == 0) sred[wave] = M;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; w++) M = fmaxf(M, sred[w]);
        const float Ms = M == NEG_INF ? 0.f : M;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        float l = 0.f;
        for (uint32_t p0 = 0; p0 < parts; p0 += 512) {
            const uint32_t n = min(512u, parts - p0);
            __syncthreads();
            if (tid < n) {
                const float* q = slot_of(p0 + tid) + (uint64_t)R * hd + r0 + r;
                const float w = exp2_hw(q[0] - Ms);
                sw[tid] = w;
                l = __builtin_fmaf(q[R], w, l);
            }
            __syncthreads();
            for (uint32_t p = grp; p < n; p += 8 * groups) {
                f32x4 v[8];
#pragma unroll
                for (int k = 0; k < 8; k++) v[k] = *(const f32x4*)(slot_of(p0 + min(p + k * groups, n - 1)) + (uint64_t)(r0 + r) * hd + col);
#pragma unroll
                for (int k = 0; k < 8; k++)
                    if (p + k * groups < n) add(acc, v[k], sw[p + k * groups]);
            }
        }
        l = group_sum<64>(l);
        so[tid] = acc;
        __syncthreads();
        if (lane == 0) sred[wave] = l;
        __syncthreads();
        if (tid < per) {
            float ls = 0.f;
#pragma unroll
            for (int w = 0; w < 8; w++) ls += sred[w];
            f32x4 t = so[tid];
            for (uint32_t g = 1; g < groups; g++) t += so[g * per + tid];
            finish(r, col, t, ls);
        }
        __syncthreads();
    }
}
extern "C" __global__ __launch_bounds__(512) void apk_attend_join_f16(apk_attend_args a) { attend_join_body<f16_t>(a); }
extern "C" __global__ __launch_bounds__(512) void apk_attend_join_f32(apk_attend_args a) { attend_join_body<float>(a); }

// ------------------------------------------------------------------------------------------- any head size
// A workgroup of four waves per (row, query head), element by element: heads of other sizes than 64, 128 and 256 (up to
// 1024).  A wave takes blocks of 64 keys in turn, a key a lane for the scores, then a channel a lane for the values.
template <typename T>
DEV void attend_generic_body(const apk_attend_args& a, float* smem) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hd = a.hd;
    const uint32_t row = blockIdx.x / a.n_q, h = blockIdx.x % a.n_q, kvh = h / a.group;
    att_seq s = {0, 0, 0, 0, 0, 0, 1};
    uint32_t seq = 0;
    bool found = false;
    for (uint32_t base = 0; base < a.n_seq && !found; base += 64) {
        const att_seq t = att_load_seq(a, base + lane);
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
    const uint32_t kv_stride = a.n_kv * hd;
    const f16_t* kb = (const f16_t*)a.k + (uint64_t)kvh * hd;
    const f16_t* vb = (const f16_t*)a.v + (uint64_t)kvh * hd;
    const uint64_t qat = ((uint64_t)row * a.n_q + h) * hd;
    float* sq = smem;             // [hd]
    float* so = smem + hd;        // [4][hd]
    float* sml = smem + 5 * hd;   // [4][2]
    // (the scale goes into the query, so that no sum leaves the range that its score has)
    for (uint32_t i = threadIdx.x; i < hd; i += 256) sq[i] = (float)((const T*)a.q)[qat + i] * a.sign * a.scale;
    __syncthreads();
    float o[16];
#pragma unroll
    for (int i = 0; i < 16; i++) o[i] = 0.f;
    float m = NEG_INF, l = 0.f;
    bool bad = false;
    for (int32_t k0 = lo + (int32_t)wave * 64; k0 < hi; k0 += 256) {
        const int32_t key = k0 + (int32_t)lane;
        const uint32_t r = att_row(a, att_look(a, tab, key, lo, hi), bad);
        float x = NEG_INF;
        if (key < hi) {
            float d = 0.f;
            const f16_t* kr = kb + (uint64_t)r * kv_stride;
            for (uint32_t i = 0; i < hd; i++) d = __builtin_fmaf((float)kr[i], sq[i], d);
            x = d * kLog2e;
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
    att_report(a, bad);
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
    const float inv = att_inverse(ls);
    for (uint32_t i = threadIdx.x; i < hd; i += 256) {
        const float v = (so[i] * f[0] + so[hd + i] * f[1]) + (so[2 * hd + i] * f[2] + so[3 * hd + i] * f[3]);
        ((T*)a.out)[qat + i] = (T)(v * inv);
    }
}
extern "C" __global__ __launch_bounds__(256) void apk_attend_any_f16(apk_attend_args a) { attend_generic_body<f16_t>(a, att_smem); }
extern "C" __global__ __launch_bounds__(256) void apk_attend_any_f32(apk_attend_args a) { attend_generic_body<float>(a, att_smem); }
