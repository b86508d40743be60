// gfx950 device code, part of apk_kernels.hip: the pages of the paged K/V cache (who holds which) and their copies.
//
// The state is three device arrays of the caller: the pool, the page tables [n_seq][max_pages] and the lengths.  The
// bookkeeping kernels are one workgroup each: their work is a few thousand words, so what bounds them is the chain of
// dependent round trips to memory (about 1 us each), not bandwidth, and one workgroup needs no device-wide ordering.
// Every choice (which page, in which order) is a function of the state alone: sums and bit ranks, and atomics only where
// their order cannot show (counts, maxima, set bits).
#pragma once

// The pool: a header, a reference count per page, a bit per free page, and scratch that is zero between calls.
struct page_pool {
    uint32_t *head, *refs, *bits, *cnt, *last, *list;
    uint32_t n, words;
    DEV page_pool at(uint32_t* p, uint32_t n) {
        page_pool r;
        r.n = n;
        r.words = (n + 31) / 32;
        r.head = p;              // [0]: free pages
        r.refs = p + 4;          // [n]
        r.bits = r.refs + n;     // [words], bit set: free
        r.cnt = r.bits + r.words;  // [n] zero between calls
        r.last = r.cnt + n;      // [n] zero between calls
        r.list = r.last + n;     // [n] scratch
        return r;
    }
};
// State that atomics or other waves of the workgroup have changed is read past the L1.
DEV uint32_t pg_ld(const uint32_t* p) { return __hip_atomic_load((uint32_t*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
DEV void pg_st(uint32_t* p, uint32_t v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
DEV uint32_t pg_add(uint32_t* p, uint32_t v) { return __hip_atomic_fetch_add(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
DEV void pg_sync() {  // everything the workgroup has written is in the L2 before anybody goes on
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
}
#define PG_BLOCK 1024
#define PG_LIST 4096  // new pages of a step that fit LDS
// Inclusive sums over the workgroup of up to 1024 lanes; `total`: of all.  sm: 17 words.
DEV uint32_t pg_scan(uint32_t v, uint32_t* sm, uint32_t& total) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t t = __shfl_up(v, d);
        if ((int)lane >= d) v += t;
    }
    __syncthreads();  // sm may still be read from the call before
    if (lane == 63) sm[wave] = v;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < PG_BLOCK / 64; w++) {
        const uint32_t t = sm[w];
        before += (uint32_t)w < wave ? t : 0;
        total += t;
    }
    return v + before;
}
// The same for three values at once; v0 .. v2 become their sums up to this lane.  sm: 48 words.
DEV void pg_scan3(uint32_t& v0, uint32_t& v1, uint32_t& v2, uint32_t* sm, uint32_t& t0, uint32_t& t1, uint32_t& t2) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t a = __shfl_up(v0, d), b = __shfl_up(v1, d), c = __shfl_up(v2, d);
        if ((int)lane >= d) {
            v0 += a;
            v1 += b;
            v2 += c;
        }
    }
    __syncthreads();
    if (lane == 63) {
        sm[wave] = v0;
        sm[16 + wave] = v1;
        sm[32 + wave] = v2;
    }
    __syncthreads();
    uint32_t b0 = 0, b1 = 0, b2 = 0;
    t0 = t1 = t2 = 0;
#pragma unroll
    for (int w = 0; w < PG_BLOCK / 64; w++) {
        const bool before = (uint32_t)w < wave;
        b0 += before ? sm[w] : 0;
        b1 += before ? sm[16 + w] : 0;
        b2 += before ? sm[32 + w] : 0;
        t0 += sm[w];
        t1 += sm[16 + w];
        t2 += sm[32 + w];
    }
    v0 += b0;
    v1 += b1;
    v2 += b2;
}
DEV uint64_t pg_wave_sum(uint64_t v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
// The last index i of off[0 .. n) (ascending, off[0] <= k) with off[i] <= k.
DEV uint32_t pg_find(const uint32_t* off, uint32_t n, uint32_t k) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (off[mid] <= k) lo = mid;
        else hi = mid;
    }
    return lo;
}
DEV uint32_t pg_ceil(uint32_t a, uint32_t b) { return a / b + (a % b != 0); }
// Sequences that a round over tables takes, a lane each: as many as have fewer than 2^31 entries between them, so that neither
// their sum nor an index that steps past it leaves 32 bits.
DEV uint32_t pg_round(uint32_t max_pages) { return min((uint32_t)PG_BLOCK, 0x7fffffffu / max(max_pages, 1u)); }

// The pool counted afresh from the page tables (n_seq 0: every page free).
extern "C" __global__ __launch_bounds__(PG_BLOCK) void apk_pages_init_k(uint32_t* pool, uint32_t n_pages, uint32_t page, const uint32_t* table,
                                                                       uint32_t max_pages, const uint32_t* kv_len, uint32_t n_seq, uint32_t* fault) {
    const page_pool P = page_pool::at(pool, n_pages);
    const uint32_t tid = threadIdx.x;
    __shared__ uint32_t live;
    if (tid == 0) live = 0;
    for (uint32_t i = tid; i < n_pages; i += PG_BLOCK) {
        pg_st(P.refs + i, 0);
        pg_st(P.cnt + i, 0);
        pg_st(P.last + i, 0);
    }
    pg_sync();
    for (uint32_t s = tid >> 6; s < n_seq; s += PG_BLOCK / 64) {  // a wave per sequence
        uint32_t used = pg_ceil(kv_len[s], page);
        if (used > max_pages) {
            used = max_pages;
            if ((tid & 63) == 0) atomicOr(fault, APK_FAULT_CACHE_RANGE);
        }
        for (uint32_t j = tid & 63; j < used; j += 64) {
            const uint32_t e = table[(uint64_t)s * max_pages + j];
            if (e < n_pages) pg_add(P.refs + e, 1);
            else atomicOr(fault, APK_FAULT_CACHE_RANGE);
        }
    }
    pg_sync();
    for (uint32_t w = tid; w < P.words; w += PG_BLOCK) {
        uint32_t b = 0;
        for (uint32_t i = 0; i < 32 && w * 32 + i < n_pages; i++) b |= (uint32_t)(pg_ld(P.refs + w * 32 + i) == 0) << i;
        pg_st(P.bits + w, b);
        atomicAdd(&live, (uint32_t)__popc(b));
    }
    pg_sync();
    if (tid == 0) {
        P.head[0] = live;
        P.head[1] = P.head[2] = P.head[3] = 0;
    }
}

// One step of every sequence: n_new[s] tokens more.  All or nothing.  The chain is: lengths; tail pages; their holders;
// where any are shared, who writes; then everything out (9 us for 256 sequences, 17 with the list of new pages in memory
// and every number read again where it is used).
extern "C" __global__ __launch_bounds__(PG_BLOCK) void apk_pages_extend_k(uint32_t* pool, uint32_t n_pages, uint32_t page, uint32_t* table,
                                                                         uint32_t max_pages, uint32_t* kv_len, uint32_t n_seq, const uint32_t* n_new,
                                                                         uint32_t rows, uint32_t* q_off, uint32_t* positions, uint32_t* slots,
                                                                         uint32_t* pairs, uint32_t* n_pairs, uint32_t* fault) {
    const page_pool P = page_pool::at(pool, n_pages);
    const uint32_t tid = threadIdx.x;
    const uint64_t cap = (uint64_t)max_pages * page;
    __shared__ uint32_t sm[3 * PG_BLOCK / 64], bad, shared_tails;
    __shared__ unsigned long long sum_new, sum_need;
    __shared__ uint32_t row_off[PG_BLOCK + 1], first[PG_BLOCK + 1], s_len[PG_BLOCK], s_have[PG_BLOCK], s_tail[PG_BLOCK];
    __shared__ uint32_t s_list[PG_LIST];
    if (tid == 0) {
        bad = shared_tails = 0;
        sum_new = sum_need = 0;
    }
    // What does not depend on the sequences is asked for first: the number of free pages and this lane's first word of them.
    const uint32_t per = (P.words + PG_BLOCK - 1) / PG_BLOCK;
    const uint32_t w0 = min(tid * per, P.words), w1 = min(w0 + per, P.words);
    const uint32_t free0 = pg_ld(P.head), word0 = pg_ld(P.bits + min(w0, P.words - 1));
    // the page that a sequence's next token falls into, where it holds one already; n_pages: none
    auto tail_of = [&](uint32_t s, uint32_t len, uint32_t fresh) -> uint32_t {
        if (!fresh || len % page == 0 || len > cap) return n_pages;
        const uint32_t t = pg_ld(table + (uint64_t)s * max_pages + len / page);
        if (t < n_pages) return t;
        bad = APK_FAULT_CACHE_RANGE;
        return n_pages;
    };
    __syncthreads();
    // (the first block of sequences keeps what it reads)
    uint32_t len_a = 0, new_a = 0, tail_a = n_pages, held_a = 0;
    auto sequence = [&](uint32_t s, uint32_t& len, uint32_t& fresh, uint32_t& t, uint32_t& held) {
        if (s == tid) {
            len = len_a;
            fresh = new_a;
            t = tail_a;
            held = held_a;
        } else {
            len = kv_len[s];
            fresh = n_new[s];
            t = tail_of(s, len, fresh);
            held = t < n_pages ? pg_ld(P.refs + t) : 0;
        }
    };
    if (tid < n_seq) {
        len_a = kv_len[tid];
        new_a = n_new[tid];
        tail_a = tail_of(tid, len_a, new_a);
        held_a = tail_a < n_pages ? pg_ld(P.refs + tail_a) : 0;
    }
    // who writes into a page that others hold: their number and the last of them
    for (uint32_t s = tid; s < n_seq; s += PG_BLOCK) {
        uint32_t len, fresh, t, held;
        sequence(s, len, fresh, t, held);
        if (held > 1) {
            pg_add(P.cnt + t, 1);
            __hip_atomic_fetch_max(P.last + t, s + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            shared_tails = 1;
        }
        if ((uint64_t)len + fresh > cap) bad = APK_FAULT_CACHE_RANGE;
    }
    __syncthreads();
    if (shared_tails) pg_sync();
    // of the holders of a page that all write now the last one keeps it, the others write to a copy
    auto copies = [&](uint32_t s, uint32_t t, uint32_t held) -> uint32_t {
        return held > 1 && !(pg_ld(P.cnt + t) == held && pg_ld(P.last + t) == s + 1);
    };
    uint32_t need_a = 0, copy_a = 0;
    {
        uint64_t my_new = 0, my_need = 0;
        for (uint32_t s = tid; s < n_seq; s += PG_BLOCK) {
            uint32_t len, fresh, t, held;
            sequence(s, len, fresh, t, held);
            if ((uint64_t)len + fresh > cap) continue;
            const uint32_t cp = copies(s, t, held), need = pg_ceil(len + fresh, page) - pg_ceil(len, page) + cp;
            my_new += fresh;
            my_need += need;
            if (s == tid) {
                need_a = need;
                copy_a = cp;
            }
        }
        my_new = pg_wave_sum(my_new);
        my_need = pg_wave_sum(my_need);
        if ((tid & 63) == 0) {
            if (my_new) atomicAdd(&sum_new, (unsigned long long)my_new);
            if (my_need) atomicAdd(&sum_need, (unsigned long long)my_need);
        }
    }
    __syncthreads();
    const bool full = sum_need > min(free0, n_pages), many = sum_new > rows;
    if (bad || full || many) {  // nothing is changed but the scratch put back
        pg_sync();
        for (uint32_t s = tid; s < n_seq; s += PG_BLOCK) {
            const uint32_t t = tail_of(s, kv_len[s], n_new[s]);
            if (t < n_pages) {
                pg_st(P.cnt + t, 0);
                pg_st(P.last + t, 0);
            }
            q_off[s + 1] = 0;
        }
        for (uint32_t r = tid; r < rows; r += PG_BLOCK) {
            positions[r] = 0;
            slots[r] = 0xffffffffu;
        }
        if (tid == 0) {
            q_off[0] = 0;
            *n_pairs = 0;
            atomicOr(fault, bad | (full ? APK_FAULT_NO_PAGES : 0u) | (many ? APK_FAULT_ROW_RANGE : 0u));
        }
        return;
    }
    // the lowest sum_need free pages, ascending; a short list stays in LDS
    const uint32_t total_need = (uint32_t)sum_need;
    auto fresh_page = [&](uint32_t k) { return total_need <= PG_LIST ? s_list[min(k, (uint32_t)PG_LIST - 1)] : pg_ld(P.list + k); };
    if (total_need) {
        auto word = [&](uint32_t w) {
            return (w == w0 ? word0 : pg_ld(P.bits + w)) & (w * 32 + 32 > n_pages ? (1u << (n_pages & 31)) - 1 : 0xffffffffu);
        };
        uint32_t mine = 0, all;
        for (uint32_t w = w0; w < w1; w++) mine += (uint32_t)__popc(word(w));
        uint32_t k = pg_scan(mine, sm, all) - mine;
        for (uint32_t w = w0; w < w1 && k < total_need; w++) {
            uint32_t b = word(w);
            while (b && k < total_need) {
                const uint32_t p = w * 32 + (uint32_t)__builtin_ctz(b);
                b &= b - 1;
                if (total_need <= PG_LIST) s_list[k] = p;
                else pg_st(P.list + k, p);
                k++;
                pg_st(P.refs + p, 1);
            }
            pg_st(P.bits + w, b);
        }
        if (tid == 0) pg_st(P.head, free0 - total_need);
        if (total_need > PG_LIST) pg_sync();  // (a short list: seen behind the next barrier)
    }
    uint32_t row_base = 0, need_base = 0, pair_base = 0;
    for (uint32_t base = 0; base < n_seq; base += PG_BLOCK) {
        const uint32_t s = base + tid, here = min((uint32_t)PG_BLOCK, n_seq - base);
        uint32_t len = 0, fresh = 0, need = 0, cp = 0, have = 0, t = n_pages, held = 0;
        if (s < n_seq) {
            sequence(s, len, fresh, t, held);
            have = pg_ceil(len, page);
            if (base == 0) {
                cp = copy_a;
                need = need_a;
            } else {
                cp = copies(s, t, held);
                need = pg_ceil(len + fresh, page) - have + cp;
            }
        }
        uint32_t i_new = fresh, i_need = need, i_cp = cp, all_new, all_need, all_cp;
        pg_scan3(i_new, i_need, i_cp, sm, all_new, all_need, all_cp);
        if (tid < here) {
            row_off[tid] = i_new - fresh;
            first[tid] = i_need - need;
            s_len[tid] = len;
            s_have[tid] = have - cp;  // item first + k goes to table entry have + k; a copy's replaces the entry before
            s_tail[tid] = t;
            q_off[s + 1] = row_base + i_new;
        }
        __syncthreads();
        // (references of pages that others hold drop only at the very end: later blocks of sequences decide by them)
        if (cp) {
            pairs[2 * (pair_base + i_cp - 1)] = fresh_page(need_base + i_need - need);
            pairs[2 * (pair_base + i_cp - 1) + 1] = t;
        }
        for (uint32_t k = tid; k < all_need; k += PG_BLOCK) {
            const uint32_t i = pg_find(first, here, k);
            pg_st(table + (uint64_t)(base + i) * max_pages + s_have[i] + (k - first[i]), fresh_page(need_base + k));
        }
        for (uint32_t r = tid; r < all_new; r += PG_BLOCK) {
            const uint32_t i = pg_find(row_off, here, r), pos = s_len[i] + (r - row_off[i]), j = pos / page;
            const uint32_t e = j >= s_have[i] ? fresh_page(need_base + first[i] + (j - s_have[i])) : s_tail[i];
            positions[row_base + r] = pos;
            slots[row_base + r] = e * page + pos % page;
        }
        if (s < n_seq) kv_len[s] = len + fresh;
        row_base += all_new;
        need_base += all_need;
        pair_base += all_cp;
        if (base + PG_BLOCK < n_seq) pg_sync();
    }
    if (pair_base) {
        pg_sync();
        for (uint32_t i = tid; i < pair_base; i += PG_BLOCK) {
            const uint32_t t = pg_ld(pairs + 2 * i + 1);
            pg_add(P.refs + t, 0xffffffffu);
            pg_st(P.cnt + t, 0);
            pg_st(P.last + t, 0);
        }
    }
    for (uint32_t r = row_base + tid; r < rows; r += PG_BLOCK) {  // rows of nobody: no cache row, so that a store skips them
        positions[r] = 0;
        slots[r] = 0xffffffffu;
    }
    if (tid == 0) {
        q_off[0] = 0;
        *n_pairs = pair_base;
    }
}

// Sequence dst[i] becomes one more holder of src[i]'s pages; as the tables were when the call began.
extern "C" __global__ __launch_bounds__(PG_BLOCK) void apk_pages_fork_k(uint32_t* pool, uint32_t n_pages, uint32_t page, uint32_t* table,
                                                                       uint32_t max_pages, uint32_t* kv_len, uint32_t n_seq, const uint32_t* src,
                                                                       const uint32_t* dst, uint32_t n, uint32_t* fault) {
    const page_pool P = page_pool::at(pool, n_pages);
    const uint32_t tid = threadIdx.x;
    __shared__ uint32_t s_src[PG_BLOCK], s_dst[PG_BLOCK], s_len[PG_BLOCK];
    if (tid < n) {
        s_src[tid] = src[tid];
        s_dst[tid] = dst[tid];
    }
    __syncthreads();
    if (tid < n) {
        const uint32_t a = s_src[tid], b = s_dst[tid];
        bool ok = a < n_seq && b < n_seq && a != b;
        for (uint32_t j = 0; j < tid; j++) ok = ok && s_dst[j] != b;  // named twice: the first one counts
        uint32_t len = 0;
        if (ok) {
            len = kv_len[a];
            ok = kv_len[b] == 0 && pg_ceil(len, page) <= max_pages;
        }
        if (!ok) atomicOr(fault, APK_FAULT_ROW_RANGE);
        s_len[tid] = ok ? len : 0;
    }
    __syncthreads();
    for (uint32_t i = tid >> 6; i < n; i += PG_BLOCK / 64) {
        const uint32_t used = pg_ceil(s_len[i], page);
        for (uint32_t j = tid & 63; j < used; j += 64) {
            const uint32_t e = table[(uint64_t)s_src[i] * max_pages + j];
            table[(uint64_t)s_dst[i] * max_pages + j] = e;
            if (e < n_pages) pg_add(P.refs + e, 1);
            else atomicOr(fault, APK_FAULT_CACHE_RANGE);
        }
        if ((tid & 63) == 0 && s_len[i]) kv_len[s_dst[i]] = s_len[i];
    }
}

// Sequences cut to new_len[s] tokens (as they are where that is not fewer); pages behind lose a holder.  5 us for 96.
extern "C" __global__ __launch_bounds__(PG_BLOCK) void apk_pages_truncate_k(uint32_t* pool, uint32_t n_pages, uint32_t page, uint32_t* table,
                                                                           uint32_t max_pages, uint32_t* kv_len, uint32_t n_seq,
                                                                           const uint32_t* new_len, uint32_t* fault) {
    const page_pool P = page_pool::at(pool, n_pages);
    const uint32_t tid = threadIdx.x;
    __shared__ uint32_t sm[PG_BLOCK / 64 + 1], freed, off[PG_BLOCK], s_keep[PG_BLOCK];
    if (tid == 0) freed = 0;
    const uint32_t round = pg_round(max_pages);
    for (uint32_t base = 0; base < n_seq; base += round) {
        const uint32_t s = base + tid, here = min(round, n_seq - base);
        uint32_t gone = 0, keep = 0;
        if (tid < here) {
            const uint32_t len = kv_len[s], cut = new_len[s];
            if (cut < len) {
                uint32_t have = pg_ceil(len, page);
                if (have > max_pages) {
                    have = max_pages;
                    atomicOr(fault, APK_FAULT_CACHE_RANGE);
                }
                keep = min(pg_ceil(cut, page), have);
                gone = have - keep;
                kv_len[s] = cut;
            }
        }
        uint32_t all;
        const uint32_t inc = pg_scan(gone, sm, all);
        if (tid < here) {
            off[tid] = inc - gone;
            s_keep[tid] = keep;
        }
        __syncthreads();
        for (uint32_t k = tid; k < all; k += PG_BLOCK) {
            const uint32_t i = pg_find(off, here, k);
            const uint32_t e = table[(uint64_t)(base + i) * max_pages + s_keep[i] + (k - off[i])];
            if (e >= n_pages) {
                atomicOr(fault, APK_FAULT_CACHE_RANGE);
                continue;
            }
            const uint32_t held = pg_add(P.refs + e, 0xffffffffu);
            if (held == 1) {
                __hip_atomic_fetch_or(P.bits + e / 32, 1u << (e & 31), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                atomicAdd(&freed, 1u);
            } else if ((int32_t)held <= 0) {  // nobody held it (below 0: so others found, and have not put theirs back yet)
                pg_add(P.refs + e, 1);
                atomicOr(fault, APK_FAULT_CACHE_RANGE);
            }
        }
        __syncthreads();
    }
    pg_sync();
    if (tid == 0) pg_st(P.head, pg_ld(P.head) + freed);
}

// The pages in use moved to the front: with L of them, the i-th at or behind L goes to the i-th free one before it.  10 us
// for 600 moves in a pool of 3500 pages.
extern "C" __global__ __launch_bounds__(PG_BLOCK) void apk_pages_compact_k(uint32_t* pool, uint32_t n_pages, uint32_t page, uint32_t* table,
                                                                          uint32_t max_pages, const uint32_t* kv_len, uint32_t n_seq,
                                                                          uint32_t* pairs, uint32_t* n_pairs, uint32_t* fault) {
    const page_pool P = page_pool::at(pool, n_pages);
    const uint32_t tid = threadIdx.x;
    __shared__ uint32_t sm[PG_BLOCK / 64 + 1], off[PG_BLOCK];
    const uint32_t L = n_pages - pg_ld(P.head);
    const uint32_t per = (P.words + PG_BLOCK - 1) / PG_BLOCK;
    const uint32_t w0 = min(tid * per, P.words), w1 = min(w0 + per, P.words);
    // of word w: the free pages before L, and the used ones from L on
    auto holes = [&](uint32_t w, uint32_t b) { return w * 32 >= L ? 0u : w * 32 + 32 <= L ? b : b & ((1u << (L & 31)) - 1); };
    auto strays = [&](uint32_t w, uint32_t b) {
        uint32_t used = ~b;
        if (w * 32 + 32 > n_pages) used &= (1u << (n_pages & 31)) - 1;
        return w * 32 >= L ? used : w * 32 + 32 <= L ? 0u : used & ~((1u << (L & 31)) - 1);
    };
    uint32_t nh = 0, ns = 0, all_h, all_s;
    for (uint32_t w = w0; w < w1; w++) {
        const uint32_t b = pg_ld(P.bits + w);
        nh += (uint32_t)__popc(holes(w, b));
        ns += (uint32_t)__popc(strays(w, b));
    }
    uint32_t kh = pg_scan(nh, sm, all_h) - nh, ks = pg_scan(ns, sm, all_s) - ns;
    const uint32_t moves = min(all_h, all_s);  // equal, unless the pool is not this table's
    if (all_h != all_s && tid == 0) atomicOr(fault, APK_FAULT_CACHE_RANGE);
    for (uint32_t w = w0; w < w1; w++) {
        const uint32_t b = pg_ld(P.bits + w);
        uint32_t h = holes(w, b), s = strays(w, b), nb = b;
        while (h) {
            const uint32_t bit = h & (0u - h);
            if (kh < moves) {
                pairs[2 * kh] = w * 32 + (uint32_t)__builtin_ctz(h);
                nb &= ~bit;
            }
            kh++;
            h ^= bit;
        }
        while (s) {
            const uint32_t bit = s & (0u - s);
            if (ks < moves) {
                pairs[2 * ks + 1] = w * 32 + (uint32_t)__builtin_ctz(s);
                nb |= bit;
            }
            ks++;
            s ^= bit;
        }
        if (nb != b) pg_st(P.bits + w, nb);
    }
    pg_sync();
    for (uint32_t k = tid; k < moves; k += PG_BLOCK) {
        const uint32_t to = pg_ld(pairs + 2 * k), from = pg_ld(pairs + 2 * k + 1);
        pg_st(P.last + from, to + 1);  // its new name, plus one
        pg_st(P.refs + to, pg_ld(P.refs + from));
        pg_st(P.refs + from, 0);
    }
    pg_sync();
    if (moves) {
        const uint32_t round = pg_round(max_pages);
        for (uint32_t base = 0; base < n_seq; base += round) {
            const uint32_t s = base + tid, here = min(round, n_seq - base);
            const uint32_t used = tid < here ? min(pg_ceil(kv_len[s], page), max_pages) : 0;
            uint32_t all;
            const uint32_t inc = pg_scan(used, sm, all);
            if (tid < here) off[tid] = inc - used;
            __syncthreads();
            for (uint32_t k = tid; k < all; k += PG_BLOCK) {
                const uint32_t i = pg_find(off, here, k);
                uint32_t* at = table + (uint64_t)(base + i) * max_pages + (k - off[i]);
                const uint32_t e = *at;
                if (e < n_pages) {
                    const uint32_t to = pg_ld(P.last + e);
                    if (to) *at = to - 1;
                }
            }
            __syncthreads();
        }
    }
    pg_sync();
    for (uint32_t k = tid; k < moves; k += PG_BLOCK) pg_st(P.last + pg_ld(pairs + 2 * k + 1), 0);
    if (tid == 0) *n_pairs = moves;
}

// Page pairs[2 i + 1] copied over page pairs[2 i] in every plane, *n_pairs of them (at most max_pairs).  An item is one slice
// (span tiles of 16 bytes, no more than 8 per lane) of one pair in one plane; workgroups take items in turn, plane after
// plane.  Bound by memory: a plain copy whose addresses come out of a list.  1.2 GB in pages of 32 KiB move in 235 us
// (5.3 TB/s, a copy of one piece 6.7).  The reads stay in the caches: 32 copies of one shared page in 64 planes take 27 us
// (33 with 4 tiles a lane), twice that with reads marked as not to be kept, which move distinct pages in 230; planes side
// by side instead of one after the other take 250.
extern "C" __global__ __launch_bounds__(256) void apk_pages_copy_k(char* region, uint32_t n_planes, uint64_t plane_bytes, uint32_t n_pages,
                                                                   uint64_t page_bytes, const uint32_t* pairs, const uint32_t* n_pairs,
                                                                   uint32_t max_pairs, uint32_t slices, uint32_t span, uint32_t* fault) {
    const uint32_t n = min(*n_pairs, max_pairs), per = n * slices;  // items of a plane
    if (per == 0) return;
    const uint32_t tiles = (uint32_t)(page_bytes / 16);
    uint32_t plane = blockIdx.x / per, r = blockIdx.x % per;
    const uint32_t dp = gridDim.x / per, dr = gridDim.x % per;
    while (plane < n_planes) {
        const uint32_t i = r / slices, t0 = (r % slices) * span + threadIdx.x, t1 = min((r % slices + 1) * span, tiles);
        const uint32_t to = pairs[2 * (uint64_t)i], from = pairs[2 * (uint64_t)i + 1];
        char* const base = region + plane * plane_bytes;
        r += dr;
        plane += dp;
        if (r >= per) {
            r -= per;
            plane++;
        }
        if (to >= n_pages || from >= n_pages) {
            if (threadIdx.x == 0) atomicOr(fault, APK_FAULT_CACHE_RANGE);
            continue;
        }
        const u32x4* src = (const u32x4*)(base + from * page_bytes);
        char* dst = base + to * page_bytes;
        u32x4 v[8];
#pragma unroll
        for (int k = 0; k < 8; k++)
            v[k] = src[t0 + k * 256 < t1 ? t0 + k * 256 : 0];
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (t0 + k * 256 < t1) nt_store(v[k], dst + (uint64_t)(t0 + k * 256) * 16);
    }
}
