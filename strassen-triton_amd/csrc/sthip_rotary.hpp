// Rotary positions: the pairs (a, b) of a head's first `rot` elements turned by position * frequency and scaled by `gain`.
//
// Cosines and sines are computed where they are used, from the angle in 64 bits, so that far positions lose nothing and no
// table is read; a thread keeps those of its pairs for all the heads it turns, which makes them cheap.  Bound by memory: MI355X,
// 8192 tokens, 40 heads of 128 bf16 31.4 us = 5.3 TB/s (38.8 before the next head's pieces were fetched ahead); 8 tokens 4.1 us.
// One width of pieces serves the pairs and what is copied: 20 turned elements of 80 in fp32 make pieces of 8 bytes, 3003 tokens, 24
// heads 14.4 us = 3.2 TB/s.
#pragma once
#include "sthip_rows.hpp"

namespace sthip {

struct RotaryParams {
    const void* q; const void* k; void* qo; void* ko;
    int64_t qs[3], ks[3], qos[3], kos[3];   // batch, token, head strides in elements
    const double* freq;                     // rot / 2 radians a position
    const void* pos;                        // positions: null, 32-bit or 64-bit
    int64_t pos_bs, pos_ts, first;          // strides; null: first + token
    int pos64;
    int tokens, rows;                       // rows = batch * tokens
    int heads_q, heads;                     // heads = q's + k's
    int rot, interleaved;
    int groups;                             // head groups: thread (row, group, item) takes heads group, group + groups, ...
    int items, turn_items;                  // chunks of a head, those with pairs first
    float gain, sign;                       // sign = -1: the rotation back
    int64_t first_block;                    // of this launch: one launch holds less than 2^32 threads
};

// cos and sin of the angle: the quarter turns are taken off in 64 bits, the rest (at most pi / 4) goes through the Taylor series
// up to x^9 and x^10, whose first left-out terms are 2e-9 and 1e-10.
__device__ __forceinline__ void turn_of(double angle, float& c, float& s) {
    const double n = __builtin_rint(angle * 0.63661977236758134308);
    const float x = (float)__builtin_fma(n, -6.123233995736766e-17, __builtin_fma(n, -1.5707963267948966, angle));
    const int quarter = (int)(n - 4.0 * __builtin_floor(n * 0.25));
    const float y = x * x;
    const float sx = x + x * y * (-1.f / 6 + y * (1.f / 120 + y * (-1.f / 5040 + y * (1.f / 362880))));
    const float cx = 1.f + y * (-0.5f + y * (1.f / 24 + y * (-1.f / 720 + y * (1.f / 40320 + y * (-1.f / 3628800)))));
    const float a = quarter & 1 ? sx : cx, b = quarter & 1 ? cx : sx;
    c = quarter == 1 || quarter == 2 ? -a : a;
    s = quarter >= 2 ? -b : b;
}

// V elements (of 16 bytes or less) as they are loaded and stored at once.
template <class T, int V> struct Piece {
    float v[V];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (V * sizeof(T) == 16) { Chunk<T> c; c.load(p, V);
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = c.v[e];
        } else if constexpr (V * sizeof(T) == 8 && sizeof(T) == 2) {
            const f32x4 f = load4<T>(p, 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = f[e];
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = to_f32<T>(p + e);
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (V * sizeof(T) == 16) { Chunk<T> c;
#pragma unroll
            for (int e = 0; e < V; ++e) c.v[e] = v[e];
            c.store(p, V);
        } else if constexpr (V * sizeof(T) == 8 && sizeof(T) == 2) store4<T>(p, f32x4{v[0], v[1], v[2], v[3]}, 4);
        else {
#pragma unroll
            for (int e = 0; e < V; ++e) from_f32(p + e, v[e]);
        }
    }
};

// V pairs a thread, in two pieces of V elements; V divides the pairs and what is copied.
template <class T, int V>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryParams p) {
    const int64_t t = (p.first_block + blockIdx.x) * 256 + threadIdx.x;
    const int item = (int)(t % p.items);
    const int64_t rest = t / p.items;
    const int group = (int)(rest % p.groups);
    const int64_t row = rest / p.groups;
    if (row >= p.rows) return;
    const int64_t b = row / p.tokens, tok = row - b * p.tokens;
    const bool turns = item < p.turn_items;
    // places of the thread's two pieces in the head
    int first, second;
    if (!turns) first = second = p.rot + (item - p.turn_items) * V;
    else if (p.interleaved) { first = item * 2 * V; second = first + V; }
    else { first = item * V; second = first + p.rot / 2; }
    auto place = [&](int head, bool isout) -> int64_t {
        const bool isq = head < p.heads_q;
        const int64_t* st = isout ? (isq ? p.qos : p.kos) : (isq ? p.qs : p.ks);
        return b * st[0] + tok * st[1] + (isq ? head : head - p.heads_q) * st[2];
    };
    // the first head's pieces are on their way while the angles are computed, each later one's while the one before is turned
    Piece<T, V> nu, nw;
    auto fetch = [&](int head) {
        if (head >= p.heads) return;
        const T* in = reinterpret_cast<const T*>(head < p.heads_q ? p.q : p.k) + place(head, false);
        nu.load(in + first);
        if (turns) nw.load(in + second);
    };
    fetch(group);
    float c[V], s[V];
    if (turns) {
        double pos;
        if (!p.pos) pos = (double)(p.first + tok);
        else if (p.pos64) pos = (double)reinterpret_cast<const int64_t*>(p.pos)[b * p.pos_bs + tok * p.pos_ts];
        else pos = (double)reinterpret_cast<const int32_t*>(p.pos)[b * p.pos_bs + tok * p.pos_ts];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            turn_of(pos * p.freq[item * V + e], c[e], s[e]);
            c[e] *= p.gain;
            s[e] *= p.gain * p.sign;
        }
    }
    for (int head = group; head < p.heads; head += p.groups) {
        T* out = reinterpret_cast<T*>(head < p.heads_q ? p.qo : p.ko) + place(head, true);
        const Piece<T, V> u = nu, w = nw;
        Piece<T, V> x, y;
        fetch(head + p.groups);
        if (!turns) { u.store(out + first); continue; }
        if (p.interleaved) {
            if constexpr (V == 1) {
                x.v[0] = u.v[0] * c[0] - w.v[0] * s[0];
                y.v[0] = u.v[0] * s[0] + w.v[0] * c[0];
            } else {
                // piece u holds the first half of the pairs, piece w the others
#pragma unroll
                for (int e = 0; e < V / 2; ++e) {
                    x.v[2 * e] = u.v[2 * e] * c[e] - u.v[2 * e + 1] * s[e];
                    x.v[2 * e + 1] = u.v[2 * e] * s[e] + u.v[2 * e + 1] * c[e];
                    y.v[2 * e] = w.v[2 * e] * c[V / 2 + e] - w.v[2 * e + 1] * s[V / 2 + e];
                    y.v[2 * e + 1] = w.v[2 * e] * s[V / 2 + e] + w.v[2 * e + 1] * c[V / 2 + e];
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                x.v[e] = u.v[e] * c[e] - w.v[e] * s[e];
                y.v[e] = u.v[e] * s[e] + w.v[e] * c[e];
            }
        }
        x.store(out + first);
        y.store(out + second);
    }
}

}  // namespace sthip
