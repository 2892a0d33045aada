// attn_common.cuh -- what the attention kernels share: the sequences of a packed batch, the keys a
// query sees, and the split of the work.
//
// Sequence b holds the query rows cu_q[b] .. cu_q[b+1] - 1 and the keys cu_k[b] .. cu_k[b] + nk - 1 with
// nk = len_k[b] where given (a cache slot filled so far), else cu_k[b+1] - cu_k[b]. Query i of nq
// stands at position p = i + nk - nq and sees key j iff keep[j], j <= p + right and (j >= p - left or
// j < sinks); a negative left or right is no limit on that side.
#pragma once
#include "ctx_common.cuh"
#include "dn8_kernels.h"

namespace dn8 {

constexpr int ATT_FAR = 1 << 29;              // "no limit": beyond every length (checked < 2^28; sums stay in 32 bits)
constexpr float ATT_LOG2E = 1.4426950408889634f, ATT_LN2 = 0.6931471805599453f;

struct Sequence {
    int b;             // sequence, or -1: none
    int q0, nq;        // first query row, queries
    int k0, nk;        // first key row, keys
    int blk;           // which block of the sequence's rows (or keys)
};

// Rows [s, e) of a sequence inside [0, T), or an error and no rows: offsets come from device memory,
// so the kernels check them before they become addresses.
DN8_DEV int checked_len(int s, int e, int64_t T, int* err) {
    if (s >= 0 && e >= s && e <= T) return e - s;
    if (err != nullptr) atomicCAS(err, 0, ERR_SHAPE);
    return 0;
}
// Sequence b (one thread or a whole warp).
template <typename A> DN8_DEV Sequence sequence_of(const A& a, int b) {
    Sequence s;
    s.b = b;
    s.blk = 0;
    s.q0 = a.cu_q[b];
    s.nq = checked_len(s.q0, a.cu_q[b + 1], a.Tq, a.err);
    s.k0 = a.cu_k[b];
    s.nk = checked_len(s.k0, a.cu_k[b + 1], a.Tk, a.err);
    if (a.len_k != nullptr) s.nk = checked_len(0, a.len_k[b], s.nk, a.err);
    return s;
}

// Block `unit` of the batch when every sequence is cut into ceil(len mul / per) blocks, len being its
// queries (KEYS = false) or its keys, and every block into shares(queries, keys): blk then counts shares. Called
// by one whole warp.
struct OneShare {
    DN8_DEV int operator()(int, int) const { return 1; }
};
template <bool KEYS, typename A, typename S = OneShare>
DN8_DEV Sequence find_block(const A& a, int unit, int mul, int per, S shares = S()) {
    constexpr int BATCH = 4;                  // 32 sequences each, their offsets loaded together
    const int lane = threadIdx.x & 31;
    int run = 0;
    Sequence s;
    s.b = -1;
    for (int base = 0; base < a.B && s.b < 0; base += 32 * BATCH) {
        int q0[BATCH], q1[BATCH], k0[BATCH], k1[BATCH], kn[BATCH];
#pragma unroll
        for (int x = 0; x < BATCH; ++x) {
            const int b = base + 32 * x + lane;
            const bool in = b < a.B;
            q0[x] = in ? a.cu_q[b] : 0;
            q1[x] = in ? a.cu_q[b + 1] : 0;
            k0[x] = in ? a.cu_k[b] : 0;
            k1[x] = in ? a.cu_k[b + 1] : 0;
            kn[x] = in && a.len_k != nullptr ? a.len_k[b] : 0;
        }
#pragma unroll
        for (int x = 0; x < BATCH; ++x) {
            const int nq = checked_len(q0[x], q1[x], a.Tq, a.err);
            int nk = checked_len(k0[x], k1[x], a.Tk, a.err);
            if (a.len_k != nullptr) nk = checked_len(0, kn[x], nk, a.err);
            const int mine = static_cast<int>((static_cast<int64_t>(KEYS ? nk : nq) * mul + per - 1) / per) * shares(nq, nk);
            int incl = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, unit < run + incl);
            if (s.b < 0 && hit) {
                const int src = __ffs(hit) - 1;
                s.b = base + 32 * x + src;
                s.blk = unit - run - __shfl_sync(0xffffffffu, incl - mine, src);
                s.q0 = __shfl_sync(0xffffffffu, q0[x], src);
                s.nq = __shfl_sync(0xffffffffu, nq, src);
                s.k0 = __shfl_sync(0xffffffffu, k0[x], src);
                s.nk = __shfl_sync(0xffffffffu, nk, src);
            }
            run += __shfl_sync(0xffffffffu, incl, 31);
        }
    }
    return s;
}

// The sequences of a batch of up to MOST as one warp keeps them in shared memory, which asks for block after block:
// a look takes 0.1 us where find_block, which reads the offsets again, takes 1.6.
struct SequenceTable {
    static constexpr int MOST = 128;
    int4 seq[MOST];    // q0, nq, k0, nk
    int end[MOST];     // blocks of this sequence and those before it
    template <bool KEYS, typename A, typename S> DN8_DEV void fill(const A& a, int per, S shares) {
        const int lane = threadIdx.x & 31;
        int run = 0;
#pragma unroll 1
        for (int base = 0; base < a.B; base += 32) {
            const int b = base + lane;
            int incl = 0;
            if (b < a.B) {
                const Sequence s = sequence_of(a, b);
                seq[b] = make_int4(s.q0, s.nq, s.k0, s.nk);
                incl = ((KEYS ? s.nk : s.nq) + per - 1) / per * shares(s.nq, s.nk);
            }
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            if (b < a.B) end[b] = run + incl;
            run += __shfl_sync(0xffffffffu, incl, 31);
        }
        __syncwarp();
    }
    DN8_DEV Sequence find(int B, int unit) const {
        const int lane = threadIdx.x & 31;
        Sequence s;
        s.b = -1;
        for (int base = 0; base < B && s.b < 0; base += 32) {
            const unsigned hit = __ballot_sync(0xffffffffu, base + lane < B && unit < end[base + lane]);
            if (hit) s.b = base + __ffs(hit) - 1;
        }
        if (s.b >= 0) {
            const int4 v = seq[s.b];
            s.q0 = v.x;
            s.nq = v.y;
            s.k0 = v.z;
            s.nk = v.w;
            s.blk = unit - (s.b > 0 ? end[s.b - 1] : 0);
        }
        return s;
    }
};

// The same of up to 32 sequences in a warp's registers, where shared memory is full: lane b holds sequence b, its
// blocks of queries and, cut into shares, of keys.
struct SequenceLanes {
    static constexpr int MOST = 32;
    int q0, nq, k0, nk, q_end, k_end;
    template <typename A, typename S> DN8_DEV void fill(const A& a, int per, S key_shares) {
        const int lane = threadIdx.x & 31;
        q0 = nq = k0 = nk = q_end = k_end = 0;
        if (lane < a.B) {
            const Sequence s = sequence_of(a, lane);
            q0 = s.q0;
            nq = s.nq;
            k0 = s.k0;
            nk = s.nk;
            q_end = (nq + per - 1) / per;
            k_end = (nk + per - 1) / per * key_shares(nq, nk);
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, q_end, o), w = __shfl_up_sync(0xffffffffu, k_end, o);
            if (lane >= o) {
                q_end += v;
                k_end += w;
            }
        }
    }
    template <bool KEYS> DN8_DEV Sequence find(int unit) const {
        const int end = KEYS ? k_end : q_end;
        const unsigned hit = __ballot_sync(0xffffffffu, unit < end);
        Sequence s;
        s.b = __ffs(hit) - 1;                                  // (-1: none)
        const int b = max(s.b, 0);
        s.q0 = __shfl_sync(0xffffffffu, q0, b);
        s.nq = __shfl_sync(0xffffffffu, nq, b);
        s.k0 = __shfl_sync(0xffffffffu, k0, b);
        s.nk = __shfl_sync(0xffffffffu, nk, b);
        const int before = __shfl_sync(0xffffffffu, end, max(b - 1, 0));
        s.blk = unit - (b > 0 ? before : 0);
        return s;
    }
};

// Key tiles of TILE keys that queries at positions p0 .. p1 see some key of: the tiles of the first
// tokens, then those of the window. tile(t) for t = 0 .. count - 1.
struct KeyTiles {
    int base, first;   // tiles base .. base + first - 1: first tokens (base = 0 unless cut)
    int start;         // then start, start + 1, ...
    int count;
    DN8_DEV int tile(int t) const { return t < first ? base + t : start + t - first; }
    DN8_DEV void cut(int b, int e) {                           // keep tile(b) .. tile(e - 1)
        base += min(b, first);
        start += max(0, b - first);
        first = max(0, min(e, first) - b);
        count = max(0, e - b);
    }
};
// Keys sinks .. sinks + hidden_keys() - 1 of a sequence lie before every query's window (the first query stands at
// nk - nq): nobody sees them, and they may hold anything, like those behind nk or with keep = 0.
template <typename A> DN8_DEV uint32_t hidden_keys(const A& a, int nq, int nk) {
    return a.left < 0 ? 0u : static_cast<uint32_t>(max(0, nk - nq - a.left - a.sinks));
}
template <typename A> DN8_DEV bool behind_hidden(const A& a, int j, uint32_t hidden) {
    return static_cast<uint32_t>(j - a.sinks) >= hidden;
}
// Keys that one of `rows` neighbouring queries sees, at most.
template <typename A> DN8_DEV int seen_keys(const A& a, int rows, int nk) {
    if (a.left < 0 || a.right < 0) return nk;
    return min(nk, min(a.left, nk) + min(a.right, nk) + min(a.sinks, nk) + rows);
}
DN8_DEV KeyTiles key_tiles(int p0, int p1, int nk, int left, int right, int sinks, int tile) {
    const int hi = min(nk - 1, p1 + right), lo = max(0, p0 - left);
    KeyTiles k;
    k.base = k.first = k.start = k.count = 0;
    if (hi < 0) return k;
    const int s = min(sinks, hi + 1);                          // first tokens that may be seen
    k.start = lo / tile;
    if (k.start > 0) k.first = min(k.start, (s + tile - 1) / tile);
    k.count = k.first + max(0, hi / tile - k.start + 1);
    return k;
}

}  // namespace dn8
