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
// the L2).  Tiles are taken by tickets, so a tile waits only for ones
// that run already; the wait is bounded all the same (then states are NaN).
//
// Backward, the same from the last token to the first: the message m_t = a_{t+1}
// dh_{t+1} goes through maps, cut where a sequence ends.  States come from those
// that the forward pass left before each tile (carries).
#include "linrec.h"

namespace ssla {
namespace {

constexpr int NT = kLinRecThreads;
constexpr float kCut = -1.0f;             // in place of a map's A, which is >= 0 or NaN
constexpr int kWindow = 8;                // tiles looked at in a step
constexpr unsigned kUnset = 0xffffffffu;  // an A that was not published: a NaN that no map has

template <class T, int V>
struct Piece {
    T v[V];
};

__device__ __forceinline__ unsigned long long word_of(float A, float L) {
    const unsigned x = __builtin_bit_cast(unsigned, A == A ? A : __builtin_nanf(""));
    return (unsigned long long)__builtin_bit_cast(unsigned, L) << 32 | x;
}
__device__ __forceinline__ float map_a(unsigned long long w) { return __builtin_bit_cast(float, (unsigned)w); }
__device__ __forceinline__ float map_l(unsigned long long w) { return __builtin_bit_cast(float, (unsigned)(w >> 32)); }

// State before place p of a chain (p > 0): word j of it lies at words + j * step.
__device__ __forceinline__ float look_back(const unsigned long long* words, int p, long long step) {
    const unsigned long long t0 = wall_clock64();
    for (;;) {
        unsigned long long w[kWindow];
        #pragma unroll
        for (int j = 0; j < kWindow; ++j)
            w[j] = __hip_atomic_load(words + max(p - 1 - j, 0) * step, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        float h = 0.0f;
        bool known = false;
        #pragma unroll
        for (int j = kWindow - 1; j >= 0; --j) {             // the nearest published state goes last
            const float A = map_a(w[j]), L = map_l(w[j]);
            if ((unsigned)w[j] == kUnset) known = false;
            else if (A < 0.0f) known = true, h = L;
            else h = fmaf(A, h, L);
        }
        if (known) return h;
        if (wall_clock64() - t0 > 500000000ull) return __builtin_nanf("");      // 5 s at 100 MHz
        __builtin_amdgcn_s_sleep(1);
    }
}

// What a workgroup knows of its tile's tokens.
struct Shared {
    int ticket;
    unsigned has[NT / 32];                // threads along the tokens in whose tokens a sequence begins
    int last[NT];                         // the last of those sequences
};

// Where a thread works.
template <int V, int R>
struct Place {
    int x, y, cb, tile, place;            // thread's column and row; block of channels; place in the chain
    bool on;                              // has channels
    int c, over;                          // first channel; those of them that the piece before has too
    long long t0, t;                      // first token of the tile, of the thread
    int n;                                // tokens of the thread
    int* first;                           // [tile + 1] sequence that begins at a token, or -1
    int in;                               // sequence that the token before the thread's belongs to
    unsigned starts, ends;                // of the thread's tokens: bit r where a sequence begins, ends
    bool begun;                           // the tile's first token belongs to a sequence that began before it

    __device__ __forceinline__ void find(const LinRecArgs& a, Shared& sh, bool backward) {
        const int tid = threadIdx.x;
        cb = blockIdx.x % a.blocks;
        place = 0;
        if (a.tiles > 1) {
            if (tid == 0)
                sh.ticket = (int)__hip_atomic_fetch_add(a.tickets + cb * kTicketStep, 1u, __ATOMIC_RELAXED,
                                                        __HIP_MEMORY_SCOPE_AGENT);
            __syncthreads();
            place = __builtin_amdgcn_readfirstlane(sh.ticket);
        }
        tile = backward ? a.tiles - 1 - place : place;
        y = tid / a.cols;
        x = tid - y * a.cols;
        const int p = cb * a.cols + x;
        on = y < a.lanes && p * V < a.channels;
        c = on ? min(p * V, a.channels - V) : 0;
        over = on ? p * V - c : 0;
        t0 = (long long)tile * a.tile;
        t = t0 + y * R;
        n = on ? (int)min((long long)R, max(0ll, a.n_tokens - t)) : 0;
    }

    // Marks the tokens at which sequences begin.
    __device__ __forceinline__ void mark(const LinRecArgs& a, Shared& sh) {
        const int tid = threadIdx.x;
        const long long t1 = min(t0 + a.tile, a.n_tokens);
        int before;                                           // sequence of the token before the tile
        if (a.cu) {
            for (int i = tid; i <= a.tile; i += NT) first[i] = -1;
            if (tid < NT / 32) sh.has[tid] = 0;
            // the first boundary at t0 or behind it, from NT at a time (and at least one barrier)
            int lo = 0, hi = a.n_seqs + 1;
            while (hi - lo > 0) {
                const int step = (hi - lo + NT - 1) / NT;
                const long long i = lo + (long long)tid * step;
                const int k = __syncthreads_count(i < hi && max(a.cu[i], 0) < t0);
                if (step == 1) {
                    lo += k;
                    break;
                }
                hi = k == 0 ? lo : (int)min((long long)hi, lo + (long long)k * step);
                lo = k == 0 ? lo : lo + (k - 1) * step + 1;
            }
            before = lo - 1;
            for (long long i = lo + tid; i <= a.n_seqs; i += NT) {
                const long long at = min((long long)max(a.cu[i], 0), a.n_tokens);
                if (at > t1) break;
                if (at >= t0) atomicMax(first + (at - t0), (int)i);
            }
        } else {
            const unsigned len = (unsigned)a.seq_len;
            for (int i = tid; i <= a.tile; i += NT) {
                const unsigned at = (unsigned)(t0 + i), s = at / len;
                first[i] = at == s * len ? (int)s : -1;
            }
            if (tid < NT / 32) sh.has[tid] = 0;
            before = t0 ? (int)((unsigned)(t0 - 1) / len) : -1;
        }
        __syncthreads();
        starts = ends = 0;
        int last = -1;
        if (y < a.lanes) {
            int next = first[y * R];
            #pragma unroll
            for (int r = 0; r < R; ++r) {
                if (next >= 0) starts |= 1u << r, last = next;
                next = first[y * R + r + 1];
                if (next >= 0 || t + r + 1 >= a.n_tokens) ends |= 1u << r;
            }
            if (x == 0 && last >= 0) {
                sh.last[y] = last;
                atomicOr(sh.has + (y >> 5), 1u << (y & 31));
            }
        }
        begun = first[0] < 0 && before >= 0 && before < a.n_seqs;
        __syncthreads();
        in = before;
        unsigned m = sh.has[y >> 5] & ((1u << (y & 31)) - 1);
        for (int k = y >> 5;; m = sh.has[--k]) {
            if (m) {
                in = sh.last[32 * k + 31 - __builtin_clz(m)];
                break;
            }
            if (k == 0) break;
        }
    }
};

template <class T, int V, int R>
__device__ __forceinline__ void load(Piece<T, V> (&x)[R], const void* base, long long stride, const Place<V, R>& p) {
    const T* from = (const T*)base + p.t * stride + p.c;
    #pragma unroll
    for (int r = 0; r < R; ++r)
        if (r < p.n) __builtin_memcpy(&x[r], from + r * stride, sizeof(x[r]));
}
// A piece without the channels that another thread has too.
template <class T, int V>
__device__ __forceinline__ void store(T* to, const Piece<T, V>& x, int over) {
    if (over == 0) {
        __builtin_memcpy(to, &x, sizeof(x));
    } else {
        #pragma unroll
        for (int i = 1; i < V; ++i)
            if (i >= over) to[i] = x.v[i];
    }
}
template <int V>
__device__ __forceinline__ void read_state(float (&h)[V], const float* pool, long long stride, int slot, int c) {
    if (pool && slot >= 0) {
        __builtin_memcpy(h, pool + slot * stride + c, sizeof(h));
    } else {
        #pragma unroll
        for (int i = 0; i < V; ++i) h[i] = 0.0f;
    }
}

// Copies the states of sequences without tokens: workgroup b of those behind the tiles.
__device__ void empty_sequences(const LinRecArgs& a, int b, const float* from, long long fs, float* to, long long ts) {
    __shared__ int which[NT];
    const long long seq = (long long)b * NT + threadIdx.x;
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
    for (int i = 0; i < NT; ++i)
        if (which[i] >= 0)
            for (int c = threadIdx.x; c < a.channels; c += NT)
                to[which[i] * ts + c] = from ? from[which[i] * fs + c] : 0.0f;
}

template <class T, int V, int R>
__global__ __launch_bounds__(NT) void k_linrec(const LinRecArgs a) {
    extern __shared__ __align__(16) char smem[];
    __shared__ Shared sh;
    if (blockIdx.x >= (unsigned)(a.tiles * a.blocks)) {
        empty_sequences(a, blockIdx.x - a.tiles * a.blocks, a.s_in, a.si, a.s_out, a.so);
        return;
    }
    const int cb = a.cols * V;                               // channels of a workgroup, and of a row of LDS
    float* sA = (float*)smem;                                // [lanes][cb]
    float* sL = sA + a.lanes * cb;
    Place<V, R> p;
    p.first = (int*)(sL + a.lanes * cb);
    p.find(a, sh, false);

    Piece<T, V> g[R] = {}, v[R] = {}, q[R] = {};
    load(g, a.g, a.gt, p);
    load(v, a.v, a.vt, p);
    if (a.q) load(q, a.q, a.qt, p);
    p.mark(a, sh);

    // Token r with state h behind it.
    auto finish = [&](int r, const float (&h)[V], int slot) {
        if (slot < 0 && !a.carries) return;                  // of no sequence: stays, zero with carries
        Piece<T, V> y;
        #pragma unroll
        for (int i = 0; i < V; ++i) y.v[i] = (T)(slot < 0 ? 0.0f : a.q ? (float)q[r].v[i] * h[i] : h[i]);
        store((T*)a.out + (p.t + r) * a.ot + p.c, y, p.over);
        if (a.s_out && slot >= 0 && (p.ends >> r & 1)) {
            Piece<float, V> s;
            #pragma unroll
            for (int i = 0; i < V; ++i) s.v[i] = h[i];
            store(a.s_out + slot * a.so + p.c, s, p.over);
        }
    };

    // the thread's map; tokens from its first beginning of a sequence on are done here
    float c[R][V], A[V], h[V];
    #pragma unroll
    for (int i = 0; i < V; ++i) A[i] = 1.0f, h[i] = 0.0f;
    bool cut = false;
    int slot = -1;
    #pragma unroll
    for (int r = 0; r < R; ++r) {
        if (r < p.n && (p.starts >> r & 1)) {
            cut = true;
            slot = linrec_slot(a, p.first[p.y * R + r]);
            read_state(h, a.s_in, a.si, slot, p.c);
        }
        #pragma unroll
        for (int i = 0; i < V; ++i) {
            c[r][i] = gate_of((float)g[r].v[i]);
            h[i] = through(c[r][i], h[i]) + (float)v[r].v[i];
            A[i] = through(c[r][i], A[i]);
        }
        if (cut && r < p.n) finish(r, h, slot);
    }
    if (p.on) {
        #pragma unroll
        for (int i = 0; i < V; ++i) {
            sA[p.y * cb + p.x * V + i] = cut ? kCut : A[i];
            sL[p.y * cb + p.x * V + i] = h[i];
        }
    }
    __syncthreads();

    // a thread a channel: the tile's map, the state before it, and those before its threads
    const int k = threadIdx.x;
    if (k < cb && (p.cb * a.cols + k / V) * V < a.channels) {
        float state = 0.0f;
        if (a.tiles > 1) {
            float tA = 1.0f, tL = 0.0f;
            for (int y = 0; y < a.lanes; ++y) {
                const float yA = sA[y * cb + k], yL = sL[y * cb + k];
                tL = yA < 0.0f ? yL : fmaf(yA, tL, yL);
                tA = yA < 0.0f || tA < 0.0f ? kCut : tA * yA;
            }
            const long long step = (long long)a.blocks * cb;
            unsigned long long* words = a.words + p.cb * cb + k;
            auto publish = [&](float A, float L) {
                __hip_atomic_store(words + p.place * step, word_of(A, L), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            };
            publish(p.begun ? tA : kCut, tL);
            if (p.begun) {
                state = look_back(words, p.place, step);
                if (!(tA < 0.0f)) publish(kCut, fmaf(tA, state, tL));
                if (a.carries) {
                    const int col = (p.cb * a.cols + k / V) * V, at = min(col, a.channels - V) + k % V;
                    if (at >= col) a.carries[(long long)p.tile * a.channels + at] = state;
                }
            }
        }
        for (int y = 0; y < a.lanes; ++y) {
            const float yA = sA[y * cb + k], yL = sL[y * cb + k];
            sL[y * cb + k] = state;
            state = yA < 0.0f ? yL : fmaf(yA, state, yL);
        }
    }
    __syncthreads();
    if (p.n == 0 || (p.starts & 1)) return;
    #pragma unroll
    for (int i = 0; i < V; ++i) h[i] = sL[p.y * cb + p.x * V + i];
    slot = linrec_slot(a, p.in);
    #pragma unroll
    for (int r = 0; r < R; ++r) {
        if (r >= p.n || (p.starts >> r & 1)) break;
        #pragma unroll
        for (int i = 0; i < V; ++i) h[i] = through(c[r][i], h[i]) + (float)v[r].v[i];
        finish(r, h, slot);
    }
}

template <class T, int V, int R>
__global__ __launch_bounds__(NT) void k_linrec_backward(const LinRecArgs a) {
    extern __shared__ __align__(16) char smem[];
    __shared__ Shared sh;
    if (blockIdx.x >= (unsigned)(a.tiles * a.blocks)) {
        empty_sequences(a, blockIdx.x - a.tiles * a.blocks, a.ds_out, a.dso, a.ds_in, a.dsi);
        return;
    }
    const int cb = a.cols * V;
    float* sA = (float*)smem;
    float* sL = sA + a.lanes * cb;
    Place<V, R> p;
    p.first = (int*)(sL + a.lanes * cb);
    p.find(a, sh, true);

    Piece<T, V> g[R] = {}, v[R] = {}, q[R] = {}, d[R] = {};
    load(g, a.g, a.gt, p);
    load(v, a.v, a.vt, p);
    if (a.q) load(q, a.q, a.qt, p);
    if (a.dout) load(d, a.dout, a.dot, p);
    p.mark(a, sh);

    // states, as the forward pass had them: hs[r] before token r, hs[R] behind the last
    float c[R][V], A[V], h[V], hs[R + 1][V];
    #pragma unroll
    for (int i = 0; i < V; ++i) A[i] = 1.0f, h[i] = 0.0f;
    bool cut = false;
    #pragma unroll
    for (int r = 0; r < R; ++r) {
        if (r < p.n && (p.starts >> r & 1)) {
            cut = true;
            read_state(h, a.s_in, a.si, linrec_slot(a, p.first[p.y * R + r]), p.c);
        }
        #pragma unroll
        for (int i = 0; i < V; ++i) {
            c[r][i] = gate_of((float)g[r].v[i]);
            hs[r][i] = h[i];
            h[i] = through(c[r][i], h[i]) + (float)v[r].v[i];
            A[i] = through(c[r][i], A[i]);
        }
    }
    if (p.on) {
        #pragma unroll
        for (int i = 0; i < V; ++i) {
            sA[p.y * cb + p.x * V + i] = cut ? kCut : A[i];
            sL[p.y * cb + p.x * V + i] = h[i];
        }
    }
    __syncthreads();
    const int k = threadIdx.x;
    const int col = (p.cb * a.cols + k / V) * V, at = min(col, a.channels - V) + k % V;
    const bool chain = k < cb && col < a.channels;
    if (chain) {
        float state = p.begun && a.tiles > 1 ? a.carries[(long long)p.tile * a.channels + at] : 0.0f;
        for (int y = 0; y < a.lanes; ++y) {
            const float yA = sA[y * cb + k], yL = sL[y * cb + k];
            sL[y * cb + k] = state;
            state = yA < 0.0f ? yL : fmaf(yA, state, yL);
        }
    }
    __syncthreads();
    #pragma unroll
    for (int i = 0; i < V; ++i) hs[R][i] = h[i];
    if (p.on) {
        #pragma unroll
        for (int i = 0; i < V; ++i) h[i] = sL[p.y * cb + p.x * V + i];
        bool before = true;                                  // of the thread's first beginning
        #pragma unroll
        for (int r = 0; r < R; ++r) {
            if (p.starts >> r & 1) before = false;
            #pragma unroll
            for (int i = 0; i < V; ++i)
                if (before) {
                    hs[r][i] = h[i];
                    h[i] = through(c[r][i], h[i]) + (float)v[r].v[i];
                }
        }
        #pragma unroll
        for (int i = 0; i < V; ++i)
            if (before) hs[R][i] = h[i];
    }
    __syncthreads();

    // Token r with the gradient of its state.
    auto finish = [&](int r, const float (&dh)[V], int slot) {
        Piece<T, V> y;
        const long long t = p.t + r;
        if (a.dv) {
            #pragma unroll
            for (int i = 0; i < V; ++i) y.v[i] = (T)(slot < 0 ? 0.0f : dh[i]);
            store((T*)a.dv + t * a.dvt + p.c, y, p.over);
        }
        if (a.dg) {
            #pragma unroll
            for (int i = 0; i < V; ++i) y.v[i] = (T)(slot < 0 ? 0.0f : dh[i] * hs[r][i] * slope_of(c[r][i]));
            store((T*)a.dg + t * a.dgt + p.c, y, p.over);
        }
        if (a.dq) {
            #pragma unroll
            for (int i = 0; i < V; ++i) {
                const float behind = through(c[r][i], hs[r][i]) + (float)v[r].v[i];
                y.v[i] = (T)(slot < 0 ? 0.0f : (float)d[r].v[i] * behind);
            }
            store((T*)a.dq + t * a.dqt + p.c, y, p.over);
        }
        if (a.ds_in && slot >= 0 && (p.starts >> r & 1)) {
            Piece<float, V> s;
            #pragma unroll
            for (int i = 0; i < V; ++i) s.v[i] = through(c[r][i], dh[i]);
            store(a.ds_in + slot * a.dsi + p.c, s, p.over);
        }
    };
    // sequence of token r
    auto seq_of = [&](int r) {
        const unsigned m = p.starts & ((2u << r) - 1);
        return linrec_slot(a, m ? p.first[p.y * R + 31 - __builtin_clz(m)] : p.in);
    };

    // the map of messages; tokens up to the last end of a sequence are done here
    float m[V];
    #pragma unroll
    for (int i = 0; i < V; ++i) A[i] = 1.0f, m[i] = 0.0f;
    cut = false;
    #pragma unroll
    for (int r = R - 1; r >= 0; --r) {
        if (r < p.n && (p.ends >> r & 1)) {
            cut = true;
            read_state(m, a.ds_out, a.dso, seq_of(r), p.c);
        }
        float dh[V];
        #pragma unroll
        for (int i = 0; i < V; ++i) {
            const float e = a.q ? (float)q[r].v[i] * (float)d[r].v[i] : (float)d[r].v[i];
            dh[i] = e + m[i];
        }
        if (cut && r < p.n) finish(r, dh, seq_of(r));
        #pragma unroll
        for (int i = 0; i < V; ++i) {
            m[i] = r < p.n ? through(c[r][i], dh[i]) : 0.0f;
            A[i] = r < p.n ? through(c[r][i], A[i]) : A[i];
        }
    }
    if (p.on) {
        #pragma unroll
        for (int i = 0; i < V; ++i) {
            sA[p.y * cb + p.x * V + i] = cut ? kCut : A[i];
            sL[p.y * cb + p.x * V + i] = m[i];
        }
    }
    __syncthreads();
    if (chain) {
        float state = 0.0f;
        if (a.tiles > 1) {
            float tA = 1.0f, tL = 0.0f;
            for (int y = a.lanes - 1; y >= 0; --y) {
                const float yA = sA[y * cb + k], yL = sL[y * cb + k];
                tL = yA < 0.0f ? yL : fmaf(yA, tL, yL);
                tA = yA < 0.0f || tA < 0.0f ? kCut : tA * yA;
            }
            // a sequence that goes on behind the tile
            const bool open = p.place > 0 && p.first[a.tile] < 0;
            const long long step = (long long)a.blocks * cb;
            unsigned long long* words = a.words + p.cb * cb + k;
            auto publish = [&](float A, float L) {
                __hip_atomic_store(words + p.place * step, word_of(A, L), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            };
            publish(open ? tA : kCut, tL);
            if (open) {
                state = look_back(words, p.place, step);
                if (!(tA < 0.0f)) publish(kCut, fmaf(tA, state, tL));
            }
        }
        for (int y = a.lanes - 1; y >= 0; --y) {
            const float yA = sA[y * cb + k], yL = sL[y * cb + k];
            sL[y * cb + k] = state;
            state = yA < 0.0f ? yL : fmaf(yA, state, yL);
        }
    }
    __syncthreads();
    if (p.n == 0 || (p.ends >> (p.n - 1) & 1)) return;
    #pragma unroll
    for (int i = 0; i < V; ++i) m[i] = sL[p.y * cb + p.x * V + i];
    const int slot = seq_of(R - 1);
    bool behind = true;                                      // behind the last end
    #pragma unroll
    for (int r = R - 1; r >= 0; --r) {
        if (p.ends >> r & 1) behind = false;
        if (!behind || r >= p.n) continue;
        float dh[V];
        #pragma unroll
        for (int i = 0; i < V; ++i) {
            const float e = a.q ? (float)q[r].v[i] * (float)d[r].v[i] : (float)d[r].v[i];
            dh[i] = e + m[i];
            m[i] = through(c[r][i], dh[i]);
        }
        finish(r, dh, slot);
    }
}

// Empties the chain: no word is published, no ticket taken.
__global__ __launch_bounds__(NT) void k_linrec_clear(unsigned long long* words, long long n, unsigned* tickets, int nt) {
    const long long i = (long long)blockIdx.x * NT + threadIdx.x;
    if (i < n) words[i] = ~0ull;
    if (i < nt) tickets[i] = 0;
}

size_t lds_bytes(const LinRecArgs& a) {
    return (size_t)a.lanes * a.cols * a.vec * 8 + ((size_t)a.tile + 1) * 4;
}

template <int V> constexpr int kTokens = V == 8 ? 4 : 8;     // of a thread

template <class T>
hipError_t launch(const LinRecArgs& a, bool backward, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    LinRecArgs args = a;
    if (a.tiles > 1) {
        long long n = (long long)linrec_words(a);
        int nt = a.blocks * kTicketStep;
        void* pc[] = {&args.words, &n, &args.tickets, &nt};
        const long long most = n > nt ? n : nt;
        const hipError_t e = hipLaunchKernel((const void*)k_linrec_clear, dim3((unsigned)((most + NT - 1) / NT)), dim3(NT),
                                             pc, 0, st);
        if (e != hipSuccess) return e;
    }
    const bool states = backward ? a.ds_in != nullptr : a.s_out && a.s_out != a.s_in;
    const long long empties = states && (a.cu || !a.n_tokens) ? ((long long)a.n_seqs + NT - 1) / NT : 0;
    const long long wgs = (long long)a.tiles * a.blocks + empties;
    if (!wgs) return hipSuccess;
    void* pa[] = {&args};
    const void* f = backward ? a.vec > 1 ? (const void*)k_linrec_backward<T, V, kTokens<V>>
                                         : (const void*)k_linrec_backward<T, 1, kTokens<1>>
                    : a.vec > 1 ? (const void*)k_linrec<T, V, kTokens<V>>
                                : (const void*)k_linrec<T, 1, kTokens<1>>;
    return hipLaunchKernel(f, dim3((unsigned)wgs), dim3(NT), pa, lds_bytes(a), st);
}

}  // namespace

void linrec_plan(LinRecArgs& a, int dtype) {
    a.vec = dtype == SSLA_F32 ? 4 : 8;
    const int tokens = a.vec == 8 ? kTokens<8> : kTokens<4>;
    static_assert(kTokens<4> == kTokens<1>);
    if (a.channels < a.vec) a.vec = 1;
    const int pieces = (a.channels - 1) / a.vec + 1;
    a.blocks = (pieces + 15) / 16;
    a.cols = (pieces - 1) / a.blocks + 1;
    a.lanes = kLinRecThreads / a.cols;
    a.tile = a.lanes * (a.vec == 1 ? kTokens<1> : tokens);
    a.tiles = (int)((a.n_tokens + a.tile - 1) / a.tile);
}

hipError_t linrec_launch(const LinRecArgs& a, int dtype, hipStream_t st) {
    return dtype == SSLA_F32    ? launch<float>(a, false, st)
           : dtype == SSLA_BF16 ? launch<__bf16>(a, false, st)
                                : launch<_Float16>(a, false, st);
}
hipError_t linrec_launch_backward(const LinRecArgs& a, int dtype, hipStream_t st) {
    return dtype == SSLA_F32    ? launch<float>(a, true, st)
           : dtype == SSLA_BF16 ? launch<__bf16>(a, true, st)
                                : launch<_Float16>(a, true, st);
}

}  // namespace ssla
