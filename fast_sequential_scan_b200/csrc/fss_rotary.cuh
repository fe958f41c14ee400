// Rotary positions: the first R channels of every head are taken as R / 2 pairs (x, y), and the pair j of a token at
// position p is turned by p * turns[j] turns:
//
//     x' = m (x cos - y sin) ,   y' = m (x sin + y cos)
//
// turns[j] is a 64-bit fraction of a full turn, so that the product with the position, taken modulo 2^64, is the exact
// fraction of a turn for every position (positions in fp32 would leave an angle of 100,000 radians a sixteenth of a
// degree off).  The angle's upper 32 bits go through sincospif.  The gradient is the same rotation backwards.
//
// Bound by memory: queries and keys read and written once.  The sines of a token are made once, in shared memory, for
// all its heads.
#pragma once

#include "fss_common.cuh"

namespace fss {
namespace rotary {

constexpr int kThreads = 256, kMaxPairs = 512;

template <typename T> struct Side {      // queries or keys: [B, T, heads, D]
    const T *in;
    int64_t sb, st, sh;
    T *out;                              // contiguous
    int heads;
};

template <typename T> struct Params {
    int64_t B, T_;
    int D, R;
    Side<T> side[2];
    const int64_t *positions;            // position of (b, t): positions[b * psb + t * pst]
    int64_t psb, pst;
    const int64_t *turns;
    float magnitude;
    int tokens;                          // of a CTA
    int splits;                          // CTAs that share a token group's heads
};

// V: channels of an access.  kInterleaved: neighbouring channels make a pair, else channels j and j + R / 2.
template <typename T, int V, bool kInterleaved, bool kInverse> __global__ void __launch_bounds__(kThreads) rotate(Params<T> p) {
    extern __shared__ float2 turned[];      // [tokens][R / 2]: cos, sin
    const int pairs = p.R / 2;
    const int64_t all = p.B * p.T_, first = (int64_t)(blockIdx.x / p.splits) * p.tokens;
    const int split = blockIdx.x % p.splits;
    const int tokens = (int)min((int64_t)p.tokens, all - first);
    for (int i = threadIdx.x; i < tokens * pairs; i += kThreads) {
        const int64_t at = first + i / pairs;
        const int64_t position = p.positions[at / p.T_ * p.psb + at % p.T_ * p.pst];
        const uint64_t phase = (uint64_t)position * (uint64_t)p.turns[i % pairs];
        // the upper 32 bits as a signed fraction of half a turn
        float s, c;
        sincospif((float)(int32_t)(phase >> 32) * 0x1p-31f, &s, &c);
        turned[i] = make_float2(c * p.magnitude, (kInverse ? -s : s) * p.magnitude);
    }
    __syncthreads();
    // items: fragments of the turned channels (two for "half"), then of the channels that pass through
    const int per_turn = kInterleaved ? p.R / V : pairs / V, rest = (p.D - p.R) / V, per_head = per_turn + rest;
    const int heads = p.side[0].heads + p.side[1].heads;
    const int per_token = heads * per_head, items = tokens * per_token;
    for (int i = split * kThreads + threadIdx.x; i < items; i += p.splits * kThreads) {
        const int tok = i / per_token, j = i % per_token % per_head;
        int h = i % per_token / per_head;
        const Side<T> &x = p.side[h >= p.side[0].heads];
        if (h >= p.side[0].heads) h -= p.side[0].heads;
        const int64_t at = first + tok;
        const T *in = x.in + at / p.T_ * x.sb + at % p.T_ * x.st + (int64_t)h * x.sh;
        T *out = x.out + (at * x.heads + h) * p.D;
        float a[V], b[V];
        if (j >= per_turn) {
            const int d = p.R + (j - per_turn) * V;
            Frag<T, V>::load(in + d, a);
            Frag<T, V>::store(out + d, a);
        } else if (kInterleaved) {
            const float2 *cs = turned + tok * pairs + j * (V / 2);
            Frag<T, V>::load(in + j * V, a);
#pragma unroll
            for (int e = 0; e < V; e += 2) {
                const float2 z = cs[e / 2];
                b[e] = a[e] * z.x - a[(e + 1) % V] * z.y;
                b[(e + 1) % V] = a[e] * z.y + a[(e + 1) % V] * z.x;
            }
            Frag<T, V>::store(out + j * V, b);
        } else {
            const float2 *cs = turned + tok * pairs + j * V;
            Frag<T, V>::load(in + j * V, a);
            Frag<T, V>::load(in + pairs + j * V, b);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float2 z = cs[e];
                const float x0 = a[e] * z.x - b[e] * z.y;
                b[e] = a[e] * z.y + b[e] * z.x;
                a[e] = x0;
            }
            Frag<T, V>::store(out + j * V, a);
            Frag<T, V>::store(out + pairs + j * V, b);
        }
    }
}

// Interleaved pairs of single channels (odd strides): the pair itself is the item.
template <typename T, bool kInverse> __global__ void __launch_bounds__(kThreads) rotate_pairs(Params<T> p) {
    extern __shared__ float2 turned[];
    const int pairs = p.R / 2;
    const int64_t all = p.B * p.T_, first = (int64_t)(blockIdx.x / p.splits) * p.tokens;
    const int split = blockIdx.x % p.splits;
    const int tokens = (int)min((int64_t)p.tokens, all - first);
    for (int i = threadIdx.x; i < tokens * pairs; i += kThreads) {
        const int64_t at = first + i / pairs;
        const int64_t position = p.positions[at / p.T_ * p.psb + at % p.T_ * p.pst];
        const uint64_t phase = (uint64_t)position * (uint64_t)p.turns[i % pairs];
        float s, c;
        sincospif((float)(int32_t)(phase >> 32) * 0x1p-31f, &s, &c);
        turned[i] = make_float2(c * p.magnitude, (kInverse ? -s : s) * p.magnitude);
    }
    __syncthreads();
    const int rest = p.D - p.R, per_head = pairs + rest, heads = p.side[0].heads + p.side[1].heads;
    const int per_token = heads * per_head, items = tokens * per_token;
    for (int i = split * kThreads + threadIdx.x; i < items; i += p.splits * kThreads) {
        const int tok = i / per_token, j = i % per_token % per_head;
        int h = i % per_token / per_head;
        const Side<T> &x = p.side[h >= p.side[0].heads];
        if (h >= p.side[0].heads) h -= p.side[0].heads;
        const int64_t at = first + tok;
        const T *in = x.in + at / p.T_ * x.sb + at % p.T_ * x.st + (int64_t)h * x.sh;
        T *out = x.out + (at * x.heads + h) * p.D;
        if (j >= pairs) {
            out[p.R + j - pairs] = in[p.R + j - pairs];
        } else {
            const float2 z = turned[tok * pairs + j];
            const float a = (float)in[2 * j], b = (float)in[2 * j + 1];
            out[2 * j] = (T)(a * z.x - b * z.y);
            out[2 * j + 1] = (T)(a * z.y + b * z.x);
        }
    }
}

}  // namespace rotary
}  // namespace fss
