// linrec.hip -- the gated linear recurrence over packed sequences, and its
// gradients.
//
//   h_t = a_t h_{t-1} + v_t,   o_t = q_t h_t                    a = sigmoid(g)
//   dh_t = q_t do_t + a_{t+1} dh_{t+1},   dv = dh,   dq = do h,   dg = dh h_{t-1} a (1 - a)
//
// Bound by memory: some ten operations a value, so every tensor is read and
// written once.  All tokens, whatever sequences they belong to, are cut into tiles;
// a workgroup owns a tile's tokens for a block of channels and keeps them in
// registers, a thread R tokens by V neighbouring channels.  A stretch of tokens
// maps the state before it to the state behind it by h -> A h + L, or, where a
// sequence begins in it, to L whatever came before ("cut").  Maps go from
// tokens to threads (registers), to the tile (LDS), to the tiles before it (a chain
// over the workspace); then each thread runs its tokens from the state before
// them.  Work is even whatever the sequences' lengths.
//
// The chain: a tile publishes its map, and, once it knows the state before it, the
// state behind it.  It finds that state from the nearest tile before it that
// has published one, by the maps of those between, always in the order of the
// tokens, so that reruns give the same bits whatever was published when.  A
// published word is 64 bits, {A, L}, stored and loaded by relaxed device-scope
// atomics: whoever sees A sees L, with no fence (a release fence would write back
// the L2).  A tile that has waited for long makes the missing maps itself, from the
// tensors and in the same steps (made_here), so that none depends on another's
// workgroup being started.  Where the last states take the first ones' place, a last one may so
// be stored before a tile that is late has read the first: first states of sequences that go on
// behind a tile are then read from a copy, made by the launch that empties the chain
// (keep_first).  Drawing tiles by tickets instead cost 12 us of 57 where one
// block of channels has 1565 of them (8 ns an atomic on one address).
//
// Backward, the same from the last token to the first: the message m_t = a_{t+1}
// dh_{t+1} goes through maps, cut where a sequence ends.  States come from those
// that the forward pass left before each tile (carries).
//
// Kernels measured (us by the profiler; in brackets what moving the bytes once takes at a copy's
// rate): 1 x 40001 of 1024 bf16 channels 73.8 (64); 1 x 8192 of 2048, forward 37.4 (26), backward 57
// (46); 1.25M records of 48 fp32 ones in 19200 sequences 200 (187) and 316 (327); 40504 tokens of
// 1001 fp16 ones in 48, without q, 82 to 86 (47) and 145 to 155 (79).  fp32 is bound by memory.
// With 16 bits a value a workgroup's own time shows: all its loads are at its beginning, and its
// waves wait for half of the time: the look along the chain (8 us of 74 in the first), barriers,
// LDS.  Odd rows' addresses are little of it (the last with 1000 channels 85 and 152, with 1024 77
// and 136).  First states out of a copy (see above) cost 1.7 us of 78 in the first.
#include "linrec.h"

#include <algorithm>

#include "piece.h"

// Maps are made in two places, to the same bits: nothing is fused but by fmaf.
#pragma clang fp contract(off)

namespace ssla {
namespace {

constexpr int NT = kLinRecThreads;
constexpr float kCut = -1.0f;             // in place of a map's A, which is >= 0 or NaN
constexpr int kWindow = kBehind / 4;      // tiles that a lane looks at
constexpr unsigned kUnset = 0xffffffffu;  // an A that was not published: a NaN that no map has

__device__ __forceinline__ void opaque(int& x) { asm("" : "+v"(x)); }

__device__ __forceinline__ unsigned long long word_of(float A, float L) {
    const unsigned x = __builtin_bit_cast(unsigned, A == A ? A : __builtin_nanf(""));
    return (unsigned long long)__builtin_bit_cast(unsigned, L) << 32 | x;
}
__device__ __forceinline__ float map_a(unsigned long long w) { return __builtin_bit_cast(float, (unsigned)w); }
__device__ __forceinline__ float map_l(unsigned long long w) { return __builtin_bit_cast(float, (unsigned)(w >> 32)); }

constexpr int kMaxTile = NT * 8;          // one thread along the channels, eight tokens each

// What a workgroup knows of its tile's tokens: where sequences begin (the token behind
// the tile too), and which.
struct Shared {
    unsigned mask[kMaxTile / 32 + 1];
    int some;                             // any begins
    int counts[2][NT / 64];
    __device__ __forceinline__ bool begins(int i) const { return mask[i >> 5] >> (i & 31) & 1; }
};

// First token of sequence i (the last one's end for i = n_seqs), of those in a.cu.
__device__ __forceinline__ int boundary(const LinRecArgs& a, long long i, int value) {
    return i <= a.n_seqs ? (int)min((long long)max(value, 0), a.n_tokens) : 0x7fffffff;
}
__device__ __forceinline__ int boundary(const LinRecArgs& a, long long i) {
    return i <= a.n_seqs ? boundary(a, i, a.cu[i]) : 0x7fffffff;
}

// Where a thread works.
template <int V, int R>
struct Place {
    int x, y, cb, tile, place;            // thread's column and row; block of channels; place in the chain
    bool on;                              // has channels
    int c, over;                          // first channel; those of them that the piece before has too
    int t0, t;                            // first token of the tile, of the thread
    int n;                                // tokens of the thread
    int* first;                           // [tile + 1] sequence that begins at a token
    int in;                               // sequence that the token before the thread's belongs to
    unsigned starts, ends;                // of the thread's tokens: bit r where a sequence begins, ends
    bool begun;                           // the tile's first token belongs to a sequence that began before it
    bool plain;                           // the tile is full, and no sequence begins or ends in it
    int at, next;                         // a boundary of the thread's, and the one behind it

    __device__ __forceinline__ void find(const LinRecArgs& a, Shared& sh, bool backward) {
        const int tid = threadIdx.x, nt = blockDim.x;
        // Blocks go to the eight XCDs, each with an L2 of its own, in turn: a tile's are put
        // on one, as rows that are no whole lines share lines between them.
        const int eight = blockIdx.x / (8 * a.blocks), k = blockIdx.x - eight * 8 * a.blocks,
                  wide = min(8, a.tiles - 8 * eight);
        cb = wide == 8 ? k >> 3 : k / wide;
        place = 8 * eight + k - cb * wide;
        if (a.alone) place = a.tiles - 1 - place;
        tile = backward ? a.tiles - 1 - place : place;
        // one of nt boundaries spread over all; looked at in mark, as waiting for it here would
        // put off the tile's loads (ragged fp16, kernels' us: forward 87 -> 83, backward 155 -> 146)
        if (a.cu) {
            const int step = a.n_seqs / nt + 1;
            at = a.cu[min((long long)tid * step, (long long)a.n_seqs)];
            next = a.cu[min(tid + 1, a.n_seqs)];
        }
        for (int i = tid; i <= a.tile / 32; i += nt) sh.mask[i] = 0;
        if (tid == 0) sh.some = 0;
        y = (int)((unsigned)tid * a.per_col >> 16);          // tid / a.cols
        x = tid - y * a.cols;
        const int p = cb * a.cols + x;
        on = y < a.lanes && p * V < a.channels;
        y = on ? y : 0;
        c = on ? min(p * V, a.channels - V) : 0;
        over = on ? p * V - c : 0;
        t0 = tile * a.tile;
        t = t0 + y * R;
        n = on ? (int)min((long long)R, max(0ll, a.n_tokens - t)) : 0;
    }

    __device__ __forceinline__ void set(Shared& sh, int token, int seq) {
        const int i = token - t0;
        first[i] = seq;
        atomicOr(sh.mask + (i >> 5), 1u << (i & 31));
        sh.some = 1;
    }
    // Threads of which x holds, and a barrier.  The library's asks memory for the workgroup's
    // size, and so waits for all that is on its way.
    __device__ __forceinline__ static int count(bool x, Shared& sh, int& turn) {
        int* const counts = sh.counts[turn];
        const unsigned long long wave = __ballot(x);
        if ((threadIdx.x & 63) == 0) counts[threadIdx.x >> 6] = __popcll(wave);
        __syncthreads();
        int n = 0;
        for (int i = 0; i < (int)blockDim.x >> 6; ++i) n += counts[i];
        turn ^= 1;
        return __builtin_amdgcn_readfirstlane(n);
    }
    // Marks the tokens at which sequences begin (where several do, all but the last are
    // empty), and finds the thread's.
    __device__ __forceinline__ void mark(const LinRecArgs& a, Shared& sh) {
        const int tid = threadIdx.x, nt = blockDim.x;
        const int t1 = (int)min((long long)t0 + a.tile, a.n_tokens);
        int before;                                           // sequence of the token before the tile
        if (a.cu) {
            // the first boundary at t0 or behind it is in [lo, hi]
            int step = a.n_seqs / nt + 1;
            opaque(at), opaque(next);
            at = boundary(a, (long long)tid * step, at);
            int turn = 0, k = count(at < t0, sh, turn), lo = k, hi = k;
            if (step == 1) {
                next = boundary(a, tid + 1, next);
                if (at >= t0 && at <= t1 && next != at) set(sh, at, tid);
            } else {
                lo = k ? (k - 1) * step + 1 : 0;
                hi = k ? (int)min((long long)k * step, a.n_seqs + 1ll) : 0;
                while (hi > lo) {
                    step = (hi - lo + nt - 1) / nt;
                    const long long i = lo + (long long)tid * step;
                    k = count(i < hi && boundary(a, i) < t0, sh, turn);
                    const int from = lo;
                    lo = step == 1 ? from + k : k ? from + (k - 1) * step + 1 : from;
                    hi = step == 1 ? lo : k ? (int)min((long long)hi, from + (long long)k * step) : from;
                }
                for (long long i = lo + tid; i <= a.n_seqs; i += nt) {
                    const int here = boundary(a, i);
                    if (here > t1) break;
                    if (here >= t0 && boundary(a, i + 1) != here) set(sh, here, (int)i);
                }
            }
            before = lo - 1;
        } else {
            const int len = a.seq_len, s = linrec_begun(t0, len);
            before = s - 1;
            __syncthreads();                                  // the masks are clear
            for (long long i = s + tid; i * len <= t1; i += nt) set(sh, (int)(i * len), (int)i);
        }
        __syncthreads();
        plain = !__builtin_amdgcn_readfirstlane(sh.some) && (long long)t0 + a.tile < a.n_tokens;
        if (plain) {
            in = __builtin_amdgcn_readfirstlane(before);
            begun = in >= 0 && in < a.n_seqs;
            starts = ends = 0;
            return;
        }
        const int i = y * R;
        starts = sh.mask[i >> 5] >> (i & 31) & ((1u << n) - 1);
        ends = n == 0 ? 0 : starts >> 1 | (n < R || sh.begins(i + R) || t + R >= a.n_tokens ? 1u << (n - 1) : 0);
        begun = !(sh.mask[0] & 1) && before >= 0 && before < a.n_seqs;
        unsigned m = sh.mask[i >> 5] & ((1u << (i & 31)) - 1);
        int k = i >> 5;
        while (!m && k > 0) m = sh.mask[--k];
        in = m ? first[32 * k + 31 - __builtin_clz(m)] : before;
    }
};

template <class T, int V, int R>
__device__ __forceinline__ void opaque(Piece<T, V> (&x)[R]) {
    #pragma unroll
    for (int r = 0; r < R; ++r) x[r].opaque();
}
template <class T, int V, int R>
__device__ __forceinline__ void load(Piece<T, V> (&x)[R], const void* base, long long stride, const Place<V, R>& p,
                                     bool whole, long long tokens) {
    const T* from = (const T*)base + (long long)p.t * stride + p.c;
    if (whole) {
        #pragma unroll
        for (int r = 0; r < R; ++r) {
            x[r].load(from);
            from += stride;
        }
    } else {                                                 // as many loads: nothing waits for them here
        #pragma unroll
        for (int r = 0; r < R; ++r)
            x[r].load((const T*)base + min((long long)p.t + r, tokens - 1) * stride + p.c);
    }
}
// Tokens behind the last one are read as that one; here they are zeros.
template <class T, int V, int R>
__device__ __forceinline__ void without(Piece<T, V> (&x)[R], const Place<V, R>& p, bool whole) {
    if (whole) return;
    #pragma unroll
    for (int r = 0; r < R; ++r)
        if (r >= p.n) x[r].zero();
}
// A piece; with TAIL without the channels that another thread has too.
template <bool TAIL, class T, int V>
__device__ __forceinline__ void store(T* to, const Piece<T, V>& x, int over) {
    if (!TAIL || over == 0) x.store(to);
    else x.store_from(to, over);
}
template <bool TAIL, class T, int V>
__device__ __forceinline__ void store(T* to, const float (&x)[V], int over) {
    Piece<T, V> y;
    y.set(x);
    store<TAIL>(to, y, over);
}
template <int V>
__device__ __forceinline__ void state_of(float (&h)[V], const float* pool, long long stride, int slot, int c) {
    if (pool && slot >= 0) {
        __builtin_memcpy(h, pool + slot * stride + c, sizeof(h));
    } else {
        #pragma unroll
        for (int i = 0; i < V; ++i) h[i] = 0.0f;
    }
}

// The sequences' first tokens, as one walks over the tokens: seq is the last sequence
// that begins at token t or before it.
struct Walk {
    const LinRecArgs& a;
    int t, seq;

    __device__ __forceinline__ int first(int i) const {
        return a.cu ? boundary(a, i) : i <= a.n_seqs ? i * a.seq_len : 0x7fffffff;
    }
    __device__ Walk(const LinRecArgs& args, int token) : a(args), t(token) {
        int lo = -1, hi = a.n_seqs + 1;                      // first(lo) <= t < first(hi)
        #pragma unroll 1
        while (hi - lo > 1) {
            const int mid = lo + (hi - lo) / 2;
            if (first(mid) <= t) lo = mid;
            else hi = mid;
        }
        seq = lo;
    }
    __device__ __forceinline__ void up() {
        ++t;
        #pragma unroll 1
        while (first(seq + 1) <= t) ++seq;
    }
    __device__ __forceinline__ void down() {
        --t;
        #pragma unroll 1
        while (seq >= 0 && first(seq) > t) --seq;
    }
};

// (A, L), then (x, l)
__device__ __forceinline__ void join(float& A, float& L, float x, float l) {
    L = x < 0.0f ? l : fmaf(x, L, l);
    A = x < 0.0f || A < 0.0f ? kCut : A * x;
}

// Word of a tile for one channel, in the steps of its own workgroup: what that would
// publish first.
template <class T, int R, bool BACK>
__device__ unsigned long long made_here(const LinRecArgs& a, int place, int channel) {
    const int tile = BACK ? a.tiles - 1 - place : place, t0 = tile * a.tile, per = a.lanes / 4;
    // Of the first states in a tile only the last one is left in its map, so the copy of that one
    // may stand for the others.  (Looking at a.cut for each costs registers: with 16-bit values
    // the kernel spilled.)
    const float* const from = a.firsts ? a.firsts + (long long)tile * a.channels : a.s_in;
    const long long by = a.firsts ? 0 : a.si;
    auto value = [&](const void* p, long long stride, int t) { return (float)((const T*)p)[t * stride + channel]; };
    float tA = 1.0f, tL = 0.0f;
    #pragma unroll 1
    for (int part = 0; part < 4; ++part) {
        float mA = 1.0f, mL = 0.0f;
        #pragma unroll 1
        for (int i = part * per; i < part * per + per; ++i) {
            const int y = BACK ? a.lanes - 1 - i : i, t = t0 + y * R;
            float A = 1.0f, x = 0.0f;
            bool cut = false;
            if (!BACK) {
                Walk at(a, t - 1);
                #pragma unroll 1
                for (int r = 0; r < R; ++r) {
                    const int was = at.seq;
                    at.up();
                    if (at.seq != was) {
                        const int slot = linrec_slot(a, at.seq);
                        cut = true;
                        x = a.s_in && slot >= 0 ? from[slot * by + channel] : 0.0f;
                    }
                    const float f = gate_of(value(a.g, a.gt, t + r)).a;
                    x = fmaf(f, x, value(a.v, a.vt, t + r));
                    A *= f;
                }
            } else {
                #pragma unroll 1
                for (int r = 0; r < R; ++r) A *= gate_of(t + r < a.n_tokens ? value(a.g, a.gt, t + r) : 0.0f).a;
                Walk at(a, t + R);
                #pragma unroll 1
                for (int r = R - 1; r >= 0; --r) {
                    const int was = at.seq;
                    at.down();
                    if (t + r >= a.n_tokens) continue;
                    if (at.seq != was || t + r + 1 >= a.n_tokens) {
                        const int slot = linrec_slot(a, at.seq);
                        cut = true;
                        x = a.ds_out && slot >= 0 ? a.ds_out[slot * a.dso + channel] : 0.0f;
                    }
                    const float d = a.dout ? value(a.dout, a.dot, t + r) : 0.0f;
                    const float e = a.q ? value(a.q, a.qt, t + r) * d : d;
                    x = gate_of(value(a.g, a.gt, t + r)).a * (e + x);
                }
            }
            join(mA, mL, cut ? kCut : A, x);
        }
        join(tA, tL, mA, mL);
    }
    const Walk at(a, BACK ? t0 + a.tile - 1 : t0 - 1);
    Walk next = at;
    next.up();
    const bool open = BACK ? place > 0 && next.seq == at.seq : next.seq == at.seq && at.seq >= 0 && at.seq < a.n_seqs;
    return word_of(open ? tA : kCut, tL);
}

// Maps of a thread's channels in LDS, {A, L} each; the states that take L's place.
struct alignas(8) Map {
    float A, L;
};
template <int V>
__device__ __forceinline__ void put(Map* to, const float (&A)[V], const float (&L)[V]) {
    typedef float f4 __attribute__((ext_vector_type(4)));
    if constexpr (V % 2 == 0) {
        #pragma unroll
        for (int i = 0; i < V; i += 2) *(f4*)(to + i) = f4{A[i], L[i], A[i + 1], L[i + 1]};
    } else {
        #pragma unroll
        for (int i = 0; i < V; ++i) to[i] = Map{A[i], L[i]};
    }
}
template <int V>
__device__ __forceinline__ void get(float (&x)[V], const Map* from) {
    #pragma unroll
    for (int i = 0; i < V; ++i) x[i] = from[i].L;
}

// The chain phase: a lane has a channel of the workgroup's and one of four parts of
// its threads (of the window, while it looks back); waves have sixteen channels.
struct Chain {
    int ch, part, lane;
    bool on;                              // is there such a channel
    float A[4], L[4];                     // the parts' maps
    float tA, tL;                         // the tile's

    __device__ __forceinline__ static float from(float x, int lane, int part) { return __shfl(x, (lane & 15) + 16 * part); }

    // Folds the maps in LDS, first to last or (BACK) last to first; cuts: there may be some
    // that are cut.  Without, two instructions a map for seven (of a wave's 1400 backward some
    // 300 with LDS in pairs; 1.25M records of 48 fp32 channels: 344 -> 328 us).
    template <bool BACK>
    __device__ __forceinline__ void fold(const LinRecArgs& a, const Map* maps, int row, int piece0, int v, bool cuts) {
        lane = threadIdx.x & 63;
        ch = (threadIdx.x >> 6) * 16 + (lane & 15);
        part = lane >> 4;
        on = ch < a.cols * v && (piece0 + ch / v) * v < a.channels;
        A[0] = tA = 1.0f, L[0] = tL = 0.0f;
        const Map* m = maps + (BACK ? a.lanes - 1 - part * (a.lanes / 4) : part * (a.lanes / 4)) * row + ch;
        if (on) {
            if (cuts) folded<true>(a, m, BACK ? -row : row);
            else folded<false>(a, m, BACK ? -row : row);
        }
        const float mA = A[0], mL = L[0];
        #pragma unroll
        for (int g = 0; g < 4; ++g) {
            A[g] = from(mA, lane, g), L[g] = from(mL, lane, g);
            join(tA, tL, A[g], L[g]);
        }
    }
    template <bool CUTS>
    __device__ __forceinline__ void folded(const LinRecArgs& a, const Map* m, int step) {
        float mA = 1.0f, mL = 0.0f;
        #pragma unroll 1
        for (int y = 0; y < a.lanes; y += 16) {
            Map x[4];
            #pragma unroll
            for (int j = 0; j < 4; ++j, m += step) x[j] = *m;
            #pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (CUTS) join(mA, mL, x[j].A, x[j].L);
                else mL = fmaf(x[j].A, mL, x[j].L), mA *= x[j].A;
            }
        }
        A[0] = mA, L[0] = mL;
    }
    // Puts the states before the threads, from that before the tile, into their maps' L.
    template <bool BACK>
    __device__ __forceinline__ void spread(const LinRecArgs& a, Map* maps, int row, float state, bool cuts) {
        #pragma unroll
        for (int g = 0; g < 3; ++g)
            if (g < part) state = A[g] < 0.0f ? L[g] : fmaf(A[g], state, L[g]);
        Map* m = maps + (BACK ? a.lanes - 1 - part * (a.lanes / 4) : part * (a.lanes / 4)) * row + ch;
        if (!on) return;
        if (cuts) spreading<true>(a, m, BACK ? -row : row, state);
        else spreading<false>(a, m, BACK ? -row : row, state);
    }
    template <bool CUTS>
    __device__ __forceinline__ void spreading(const LinRecArgs& a, Map* m, int step, float state) {
        #pragma unroll 1
        for (int y = 0; y < a.lanes; y += 16) {
            Map x[4];
            #pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = m[j * step];
            #pragma unroll
            for (int j = 0; j < 4; ++j, m += step) {
                m->L = state;
                const float h = fmaf(x[j].A, state, x[j].L);
                state = CUTS && x[j].A < 0.0f ? x[j].L : h;
            }
        }
    }
    // The state before place p of the chain, after publishing the tile's map; `open`: a
    // sequence goes on from the place before into this one.  `channel`: this one's.
    template <class T, int R, bool BACK>
    __device__ __forceinline__ float before(const LinRecArgs& a, int block, int p, bool open, int channel) {
        // word of this channel at place p
        unsigned long long* word = a.words + ((long long)block * (a.tiles + kBehind) + kBehind + p) * kChannels + ch;
        auto publish = [&](float x, float l) {
            if (on && part == 0 && !a.alone)
                __hip_atomic_store(word, word_of(x, l), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        };
        publish(open ? tA : kCut, tL);
        if (!open) return 0.0f;
        float state;
        if (__builtin_expect_with_probability(!look_back(word, state, a.patience), 0, 0.999999))
            state = on ? alone<T, R, BACK>(a, word, p, channel) : 0.0f;
        if (!(tA < 0.0f)) publish(kCut, fmaf(tA, state, tL));
        return state;
    }
    // The same without waiting for anyone.  What is made here is published in the tile's
    // place, unless something is by now, which may be a state.
    template <class T, int R, bool BACK>
    __device__ float alone(const LinRecArgs& a, unsigned long long* word, int p, int channel) {
        auto map = [&](int j) {
            unsigned long long* at = word - (p - j) * kChannels;
            unsigned long long w = __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if ((unsigned)w != kUnset) return w;
            const unsigned long long made = made_here<T, R, BACK>(a, j, channel);
            w = ~0ull;
            return __hip_atomic_compare_exchange_strong(at, &w, made, __ATOMIC_RELAXED, __ATOMIC_RELAXED,
                                                        __HIP_MEMORY_SCOPE_AGENT)
                       ? made
                       : w;
        };
        int j = p - 1;
        unsigned long long w = map(j);
        #pragma unroll 1
        while (!(map_a(w) < 0.0f) && j > 0) w = map(--j);    // the first place's is a state
        float h = map_l(w);
        #pragma unroll 1
        while (++j < p) {
            w = map(j);
            h = map_a(w) < 0.0f ? map_l(w) : fmaf(map_a(w), h, map_l(w));
        }
        return h;
    }
    // Looks at the nearest 4 N tiles, N a lane.  True: h is the state, from the nearest
    // published one through the maps behind it, in their order.  False: there is none
    // yet; `nearest` says whether the nearest tile has published anything.
    template <int N>
    __device__ __forceinline__ bool look(const unsigned long long* word, float& h, bool& nearest) {
        enum { kThrough, kKnown, kBlocked };                 // what a part knows: its maps, a state, nothing
        unsigned long long w[N];
        #pragma unroll
        for (int j = 0; j < N; ++j)
            w[j] = __hip_atomic_load(word - (part * N + j + 1) * kChannels, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        float x = 0.0f;
        int mode = kThrough;
        #pragma unroll
        for (int j = N - 1; j >= 0; --j) {                   // the nearest published state goes last
            if ((unsigned)w[j] == kUnset) mode = kBlocked;
            else if (map_a(w[j]) < 0.0f) mode = kKnown, x = map_l(w[j]);
            else x = fmaf(map_a(w[j]), x, map_l(w[j]));
        }
        // states from the farther parts through the nearer ones' maps
        #pragma unroll
        for (int g = 2; g >= 0; --g) {
            const float in = from(x, lane, g + 1);
            const int known = __shfl(mode, (lane & 15) + 16 * (g + 1));
            if (part == g && mode == kThrough) {
                mode = known == kKnown ? kKnown : kThrough;
                x = in;
                #pragma unroll
                for (int j = N - 1; j >= 0; --j) x = fmaf(map_a(w[j]), x, map_l(w[j]));
            }
        }
        h = from(x, lane, 0);
        mode = __shfl(mode, lane & 15);
        nearest = __all(!on || part > 0 || (unsigned)w[0] != kUnset);
        return __all(!on || mode == kKnown);
    }
    // A word a lane until the nearest tile has published something (a state, where a
    // sequence begins in it), then eight.  False: patience ran out.
    __device__ __forceinline__ bool look_back(const unsigned long long* word, float& h, unsigned patience) {
        const unsigned long long t0 = wall_clock64();
        bool nearest;
        while (!look<1>(word, h, nearest)) {
            if (nearest) {
                while (!look<kWindow>(word, h, nearest)) {
                    if (wall_clock64() - t0 > patience) return false;
                    __builtin_amdgcn_s_sleep(1);
                }
                break;
            }
            if (wall_clock64() - t0 > patience) return false;
            __builtin_amdgcn_s_sleep(1);
        }
        return true;
    }
};

// Copies the states of sequences without tokens: workgroup b of those behind the tiles.
__device__ void empty_sequences(const LinRecArgs& a, int b, const float* from, long long fs, float* to, long long ts) {
    __shared__ int which[NT];
    const int nt = blockDim.x;
    const long long seq = (long long)b * nt + threadIdx.x;
    int slot = -1;
    if (seq < a.n_seqs) {
        bool none = a.n_tokens == 0;
        if (a.cu) {
            const long long lo = max(a.cu[seq], 0), hi = max(a.cu[seq + 1], 0);
            none = min(hi, a.n_tokens) <= min(lo, a.n_tokens);
        }
        if (none) slot = linrec_slot(a, (int)seq);
    }
    which[threadIdx.x] = slot;
    __syncthreads();
    for (int i = 0; i < nt; ++i)
        if (which[i] >= 0)
            for (int c = threadIdx.x; c < a.channels; c += nt)
                to[which[i] * ts + c] = from ? from[which[i] * fs + c] : 0.0f;
}

// Four waves a SIMD with 16-bit values, whose words take half the registers; three with fp32 ones,
// which four would spill.
template <class T, int V, int R, bool TAIL>
__global__ __launch_bounds__(NT, sizeof(T) == 2 ? 4 : 3) void k_linrec(const LinRecArgs a) {
    extern __shared__ __align__(16) char smem[];
    __shared__ Shared sh;
    if (blockIdx.x >= (unsigned)(a.tiles * a.blocks)) {
        empty_sequences(a, blockIdx.x - a.tiles * a.blocks, a.s_in, a.si, a.s_out, a.so);
        return;
    }
    const int row = a.cols * V + 2;                          // a row of LDS: the workgroup's channels, and two
    Map* maps = (Map*)smem;                                  // of the threads
    Place<V, R> p;
    p.first = (int*)(maps + a.lanes * row);
    p.find(a, sh, false);
    const bool whole = p.t0 + a.tile <= a.n_tokens;
    Piece<T, V> g[R], v[R], q[R];
    load(g, a.g, a.gt, p, whole, a.n_tokens);
    load(v, a.v, a.vt, p, whole, a.n_tokens);
    if (a.q) load(q, a.q, a.qt, p, whole, a.n_tokens);
    p.mark(a, sh);

    // The thread's map.  The last state that comes in is kept: its sequence may end
    // in another thread, which may write to its slot before this one is here again; or in
    // another tile, which may have written to it already.
    float f[R][V], A[V], h[V], last[V];
    #pragma unroll
    for (int i = 0; i < V; ++i) A[i] = 1.0f, h[i] = last[i] = 0.0f;
    #pragma unroll
    for (int r = 0; r < R; ++r) {
        if (p.starts >> r & 1) {
            const int seq = p.first[p.y * R + r];
            const bool kept = a.firsts && seq == a.cut[p.tile];
            state_of(last, kept ? a.firsts : a.s_in, kept ? a.channels : a.si, kept ? p.tile : linrec_slot(a, seq), p.c);
            #pragma unroll
            for (int i = 0; i < V; ++i) h[i] = last[i];
        }
        g[r].here(), v[r].here();
        #pragma unroll
        for (int i = 0; i < V; ++i) {
            f[r][i] = gate_of(g[r].at(i)).a;
            h[i] = fmaf(f[r][i], h[i], v[r].at(i));
            A[i] *= f[r][i];
        }
    }
    Map* const own = maps + p.y * row + p.x * V;
    if (p.on) {
        float x[V];
        #pragma unroll
        for (int i = 0; i < V; ++i) x[i] = p.starts ? kCut : A[i];
        put(own, x, h);
    }
    opaque(v), opaque(q);
    opaque(p.t), opaque(p.c);
    __syncthreads();

    // the tile's map, the state before it, and those before its threads
    Chain chain;
    chain.fold<false>(a, maps, row, p.cb * a.cols, V, !p.plain);
    const int channel = min((p.cb * a.cols + chain.ch / V) * V, a.channels - V) + chain.ch % V;
    const float state = a.tiles > 1 ? chain.before<T, R, false>(a, p.cb, p.place, p.begun, channel) : 0.0f;
    chain.spread<false>(a, maps, row, state, !p.plain);
    __syncthreads();
    if (p.n == 0) return;
    get(h, own);
    if (a.carries && p.t % a.carry == 0)
        store<TAIL>(a.carries + (long long)(p.t / a.carry) * a.channels + p.c, h, p.over);
    int slot = linrec_slot(a, p.in);
    T* out = (T*)a.out + (long long)p.t * a.ot + p.c;
    #pragma unroll
    for (int r = 0; r < R; ++r) {
        if (p.starts >> r & 1) {
            slot = linrec_slot(a, p.first[p.y * R + r]);
            if (p.starts >> r == 1) {
                #pragma unroll
                for (int i = 0; i < V; ++i) h[i] = last[i];
            } else {
                state_of(h, a.s_in, a.si, slot, p.c);
            }
        }
        float o[V];
        #pragma unroll
        for (int i = 0; i < V; ++i) {
            h[i] = fmaf(f[r][i], h[i], v[r].at(i));
            o[i] = a.q ? q[r].at(i) * h[i] : h[i];
        }
        if (slot >= 0 && r < p.n) {
            store<TAIL>(out, o, p.over);
            if (a.s_out && (p.ends >> r & 1)) store<TAIL>(a.s_out + slot * a.so + p.c, h, p.over);
        } else if (a.carries && r < p.n) {        // of no sequence: zeros
            Piece<T, V> none;
            none.zero();
            store<TAIL>(out, none, p.over);
        }
        out += a.ot;
    }
}

template <class T, int V, int R, bool TAIL>
__global__ __launch_bounds__(NT, sizeof(T) == 2 ? 4 : 3) void k_linrec_backward(const LinRecArgs a) {
    extern __shared__ __align__(16) char smem[];
    __shared__ Shared sh;
    if (blockIdx.x >= (unsigned)(a.tiles * a.blocks)) {
        empty_sequences(a, blockIdx.x - a.tiles * a.blocks, a.ds_out, a.dso, a.ds_in, a.dsi);
        return;
    }
    const int row = a.cols * V + 2;
    Map* maps = (Map*)smem;
    Place<V, R> p;
    p.first = (int*)(maps + a.lanes * row);
    p.find(a, sh, true);
    const bool whole = p.t0 + a.tile <= a.n_tokens;
    Piece<T, V> g[R], v[R], q[R], d[R];
    load(g, a.g, a.gt, p, whole, a.n_tokens);
    load(v, a.v, a.vt, p, whole, a.n_tokens);
    if (a.q) load(q, a.q, a.qt, p, whole, a.n_tokens);
    if (a.dout) load(d, a.dout, a.dot, p, whole, a.n_tokens);
    // the state before the tile, of the channel that this lane has in the chain
    const int ch = (threadIdx.x >> 6) * 16 + (threadIdx.x & 15), col = (p.cb * a.cols + ch / V) * V,
              at = min(col, a.channels - V) + ch % V;
    const float carried = a.tiles > 1 ? a.carries[(long long)p.tile * a.channels + at] : 0.0f;
    p.mark(a, sh);
    without(g, p, whole);                                    // (messages come from behind them)

    // states, as the forward pass had them; w: the gates' slopes
    float f[R][V], w[R][V], A[V], h[V];
    #pragma unroll
    for (int i = 0; i < V; ++i) A[i] = 1.0f, h[i] = 0.0f;
    #pragma unroll
    for (int r = 0; r < R; ++r) {
        if (p.starts >> r & 1) state_of(h, a.s_in, a.si, linrec_slot(a, p.first[p.y * R + r]), p.c);
        g[r].here(), v[r].here();
        #pragma unroll
        for (int i = 0; i < V; ++i) {
            const Gate gate = gate_of(g[r].at(i));
            f[r][i] = gate.a, w[r][i] = gate.slope;
            h[i] = fmaf(f[r][i], h[i], v[r].at(i));
            A[i] *= f[r][i];
        }
    }
    Map* const own = maps + p.y * row + p.x * V;
    if (p.on) {
        float x[V];
        #pragma unroll
        for (int i = 0; i < V; ++i) x[i] = p.starts ? kCut : A[i];
        put(own, x, h);
    }
    opaque(v), opaque(q), opaque(d);
    __syncthreads();
    Chain chain;
    chain.fold<false>(a, maps, row, p.cb * a.cols, V, !p.plain);
    chain.spread<false>(a, maps, row, p.begun ? carried : 0.0f, !p.plain);
    __syncthreads();
    // Once more, from the state before the thread: dq is done here; what is left of a
    // token is its gate, its slope times the state before it, and what it adds to its
    // state's gradient.
    float e[R][V];
    T* dq = (T*)a.dq + (long long)p.t * a.dqt + p.c;
    int slot = linrec_slot(a, p.in);
    get(h, own);                                             // (a thread that is not on has a row, too)
    #pragma unroll
    for (int r = 0; r < R; ++r) {
        if (p.starts >> r & 1) {
            slot = linrec_slot(a, p.first[p.y * R + r]);
            state_of(h, a.s_in, a.si, slot, p.c);
        }
        float o[V];
        #pragma unroll
        for (int i = 0; i < V; ++i) {
            const float y = a.dout ? d[r].at(i) : 0.0f;
            w[r][i] *= h[i];
            h[i] = fmaf(f[r][i], h[i], v[r].at(i));
            e[r][i] = a.q ? q[r].at(i) * y : y;
            o[i] = slot < 0 ? 0.0f : y * h[i];               // of no sequence: zeros
        }
        if (a.dq && r < p.n) store<TAIL>(dq, o, p.over);
        dq += a.dqt;
    }
    __syncthreads();

    // sequence of token r
    auto slot_at = [&](int r) {
        const unsigned m = p.starts & ((2u << r) - 1);
        return linrec_slot(a, m ? p.first[p.y * R + 31 - __builtin_clz(m)] : p.in);
    };
    // the map of messages
    float m[V];
    #pragma unroll
    for (int i = 0; i < V; ++i) m[i] = 0.0f;
    #pragma unroll
    for (int r = R - 1; r >= 0; --r) {
        if (p.ends >> r & 1) state_of(m, a.ds_out, a.dso, slot_at(r), p.c);
        if (r < p.n) {
            #pragma unroll
            for (int i = 0; i < V; ++i) m[i] = f[r][i] * (e[r][i] + m[i]);
        }
    }
    if (p.on) {
        float x[V];
        #pragma unroll
        for (int i = 0; i < V; ++i) x[i] = p.ends ? kCut : A[i];
        put(own, x, m);
    }
    opaque(p.t), opaque(p.c);
    __syncthreads();
    chain.fold<true>(a, maps, row, p.cb * a.cols, V, !p.plain);
    // a sequence that goes on behind the tile
    const bool open = p.place > 0 && !sh.begins(a.tile);
    const float state = a.tiles > 1 ? chain.before<T, R, true>(a, p.cb, p.place, open, at) : 0.0f;
    chain.spread<true>(a, maps, row, state, !p.plain);
    __syncthreads();
    if (p.n == 0) return;
    get(m, own);
    slot = slot_at(R - 1);
    T* dg = (T*)a.dg + (long long)(p.t + R - 1) * a.dgt + p.c;
    T* dv = (T*)a.dv + (long long)(p.t + R - 1) * a.dvt + p.c;
    #pragma unroll
    for (int r = R - 1; r >= 0; --r) {
        if (p.ends >> r & 1) {
            slot = slot_at(r);
            state_of(m, a.ds_out, a.dso, slot, p.c);
        }
        if (r < p.n) {
            const bool none = slot < 0;
            float dh[V], z[V];
            #pragma unroll
            for (int i = 0; i < V; ++i) {
                const float x = e[r][i] + m[i];
                m[i] = f[r][i] * x;
                dh[i] = none ? 0.0f : x;
                z[i] = none ? 0.0f : x * w[r][i];
            }
            if (a.dg) store<TAIL>(dg, z, p.over);
            if (a.dv) store<TAIL>(dv, dh, p.over);
            if (a.ds_in && (p.starts >> r & 1) && !none)
                store<TAIL>(a.ds_in + slot * a.dsi + p.c, m, p.over);
        }
        dg -= a.dgt, dv -= a.dvt;
    }
}

// Short sequences, a thread a channel, token after token, kAhead of them in flight: what
// little there is to do is done before the tiles' kernel has its boundaries.
template <class T>
__global__ __launch_bounds__(64) void k_linrec_short(const LinRecArgs a) {
    constexpr int kAhead = 8;
    const int per = (a.channels - 1) / 64 + 1, seq = blockIdx.x / per, c = (blockIdx.x - seq * per) * 64 + threadIdx.x;
    const int slot = linrec_slot(a, seq);
    if (slot < 0 || c >= a.channels) return;
    const int t0 = a.cu ? boundary(a, seq) : seq * a.seq_len, t1 = a.cu ? boundary(a, seq + 1) : t0 + a.seq_len;
    float h = a.s_in ? a.s_in[slot * a.si + c] : 0.0f;
    for (int t = t0; t < t1; t += kAhead) {
        T g[kAhead], v[kAhead], q[kAhead];
        #pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const long long at = min(t + j, t1 - 1);
            g[j] = ((const T*)a.g)[at * a.gt + c];
            v[j] = ((const T*)a.v)[at * a.vt + c];
            if (a.q) q[j] = ((const T*)a.q)[at * a.qt + c];
        }
        #pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (t + j < t1) {
                if (a.carries && (t + j) % a.carry == 0) a.carries[(long long)((t + j) / a.carry) * a.channels + c] = h;
                h = fmaf(gate_of((float)g[j]).a, h, (float)v[j]);
                ((T*)a.out)[(long long)(t + j) * a.ot + c] = (T)(a.q ? (float)q[j] * h : h);
            }
    }
    if (a.s_out) a.s_out[slot * a.so + c] = h;
}

// Copies the first state of the sequence that the tile's last token belongs to, if it begins in
// the tile.
__device__ void keep_first(const LinRecArgs& a, int tile) {
    const int lane = threadIdx.x & 63, t0 = tile * a.tile;
    const long long t = min((long long)t0 + a.tile, a.n_tokens) - 1;
    auto first = [&](long long i) { return a.cu ? (long long)boundary(a, i) : i * a.seq_len; };
    int lo = -1;
    long long hi = a.n_seqs + 1ll;                           // first(lo) <= t < first(hi)
    while (hi - lo > 1) {                                    // 64 of those between at a time
        const long long step = (hi - lo + 62) / 64, i = lo + 1 + lane * step;
        const int k = __popcll(__ballot(i < hi && first(i) <= t));
        hi = min(hi, lo + 1 + k * step);
        lo = k ? (int)(lo + 1 + (k - 1) * step) : lo;
    }
    const int slot = linrec_slot(a, lo), seq = slot >= 0 && first(lo) >= t0 ? lo : -1;
    if (threadIdx.x == 0) a.cut[tile] = seq;
    if (seq < 0) return;
    #pragma unroll 4
    for (int c = threadIdx.x; c < a.channels; c += NT)
        a.firsts[(long long)tile * a.channels + c] = a.s_in[slot * a.si + c];
}

// Empties the chain: no word is published.  Workgroups behind the first `wgs`: keep_first.
__global__ __launch_bounds__(NT) void k_linrec_clear(const LinRecArgs a, long long n, int wgs) {
    if ((int)blockIdx.x >= wgs) {
        keep_first(a, blockIdx.x - wgs);
        return;
    }
    for (long long i = (long long)blockIdx.x * NT + threadIdx.x; i < n; i += (long long)wgs * NT)
        ((ulonglong2*)a.words)[i] = ulonglong2{~0ull, ~0ull};
}

size_t lds_bytes(const LinRecArgs& a) {
    return (size_t)a.lanes * (a.cols * a.vec + 2) * 8 + ((size_t)a.tile + 1) * 4;
}

// Channels of a thread: 16 bytes; its tokens.
template <class T> constexpr int kVec = 16 / sizeof(T);
// Tokens of a thread: more are more bytes in flight for the chain phase's instructions, and
// longer tiles; fewer leave room for more waves.  Kernels' us, half as many, so, twice as many:
// forward 1.25M records of 48 fp32 channels 291, 240, 338, 1 x 40001 of 1024 bf16 ones 133,
// 108, - (earlier forms; now 198 and 74; twice as many bf16 80); backward the former 435, 347,
// 473, ragged fp16 -, 160, 167.
constexpr int tokens_of(bool wide, bool backward) { return wide ? backward ? 4 : 8 : backward ? 2 : 4; }

template <class T, bool BACKWARD, int V, bool TAIL>
const void* kernel() {
    constexpr int R = tokens_of(sizeof(T) == 4, BACKWARD);
    if constexpr (BACKWARD) return (const void*)k_linrec_backward<T, V, R, TAIL>;
    else return (const void*)k_linrec<T, V, R, TAIL>;
}

template <class T, bool BACKWARD>
hipError_t launch(const LinRecArgs& a, hipStream_t st) {
    LinRecArgs args = a;
    void* pa[] = {&args};
    if (!BACKWARD && a.brief) {
        const long long wgs = (long long)a.n_seqs * ((a.channels - 1) / 64 + 1);
        return hipLaunchKernel((const void*)k_linrec_short<T>, dim3((unsigned)wgs), dim3(64), pa, 0, st);
    }
    const int nt = linrec_threads(a);
    if (a.tiles > 1) {
        long long n = (long long)linrec_words(a) / 2;
        int wgs = (int)std::min((n + 4 * NT - 1) / (4 * NT), 1024ll);              // four stores a thread
        void* pc[] = {&args, &n, &wgs};
        const hipError_t e = hipLaunchKernel((const void*)k_linrec_clear, dim3((unsigned)(wgs + (a.firsts ? a.tiles : 0))),
                                             dim3(NT), pc, 0, st);
        if (e != hipSuccess) return e;
    }
    const bool states = BACKWARD ? a.ds_in != nullptr : a.s_out && a.s_out != a.s_in;
    const long long empties = states && (a.cu || !a.n_tokens) ? ((long long)a.n_seqs + nt - 1) / nt : 0;
    const long long wgs = (long long)a.tiles * a.blocks + empties;
    if (!wgs) return hipSuccess;
    const void* f = a.vec == 1                ? kernel<T, BACKWARD, 1, false>()
                    : a.channels % a.vec == 0 ? kernel<T, BACKWARD, kVec<T>, false>()
                                              : kernel<T, BACKWARD, kVec<T>, true>();
    return hipLaunchKernel(f, dim3((unsigned)wgs), dim3(nt), pa, lds_bytes(a), st);
}

// Threads along the channels, and along the tokens.
void cut(LinRecArgs& a, int vec, int tokens) {
    a.vec = a.channels < vec ? 1 : vec;
    const int pieces = (a.channels - 1) / a.vec + 1, most = kChannels / vec;
    a.blocks = (pieces + most - 1) / most;
    a.cols = (pieces - 1) / a.blocks + 1;
    a.per_col = 65536 / a.cols + 1;
    a.lanes = 16;
    while (2 * a.lanes * a.cols <= kLinRecThreads) a.lanes *= 2;
    a.tile = a.lanes * tokens;
    a.tiles = (int)((a.n_tokens + a.tile - 1) / a.tile);
}

}  // namespace

void linrec_plan(LinRecArgs& a, int dtype, bool backward) {
    const bool wide = dtype == SSLA_F32;
    cut(a, wide ? 4 : 8, tokens_of(wide, true));
    a.carry = a.tile;
    if (backward) return;
    cut(a, wide ? 4 : 8, tokens_of(wide, false));
    // A thread a channel, without tiles, where no sequence can have more than 32 tokens (us a
    // call, so and in tiles: 1 x 17 of 96 fp32 channels 6.2 and 8.0, 1 x 32 7.3 and 7.8, 1 x 64
    // 11.0 and 7.8, 64 x 32 8.0 and 11.1, 64 x 64 12.1 and 11.0) and the card is not filled
    // (1000 x 8 of 256 bf16 channels 8.5 and 12.9, 1000 x 32 20.3 and 18.7, 4096 x 32 of 48 fp32
    // ones 17.2 and 21.6, of a single one 14.6 and 15.0).  It looks at no rows of no sequence,
    // which carries want zeros in.
    a.brief = a.n_seqs > 0 && a.n_tokens > 0 && (a.cu ? a.n_tokens : a.seq_len) <= 32 && !(a.cu && a.carries) &&
              (long long)a.n_seqs * ((a.channels - 1) / 64 + 1) <= 1 << 12;
}

hipError_t linrec_launch(const LinRecArgs& a, int dtype, hipStream_t st) {
    return dtype == SSLA_F32    ? launch<float, false>(a, st)
           : dtype == SSLA_BF16 ? launch<__bf16, false>(a, st)
                                : launch<_Float16, false>(a, st);
}
hipError_t linrec_launch_backward(const LinRecArgs& a, int dtype, hipStream_t st) {
    return dtype == SSLA_F32    ? launch<float, true>(a, st)
           : dtype == SSLA_BF16 ? launch<__bf16, true>(a, st)
                                : launch<_Float16, true>(a, st);
}

}  // namespace ssla
