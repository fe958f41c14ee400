// Linear attention on the tensor cores, 64 tokens ("a chunk") at a time.  With G the sums of the log decays inside a
// chunk, for every sequence and head
//
//     o_i  = e^{G_i} S^T q_i + sum_{j <= i} e^{G_i - G_j} (q_i . k_j) v_j ,      S' = e^{G_last} S + sum_j (e^{G_last - G_j} k_j) v_j^T
//
// which are four products of matrices a chunk, all with value channels or queries on the tensor cores' 128 lanes:
//
//     scores  A = Q K^T            [64 queries (of 128 lanes) x 64 keys]
//     O1^T = S^T Q^T               [value channels x 64 queries], S^T from tensor memory
//     O2^T = V^T P^T               P = decayed, masked scores, through shared memory
//     dS^T = V^T K'                [value channels x key channels], K' = decayed keys
//
// The state itself stays in fp32 registers (a thread: one value channel, half of the key channels).
//
// Precision.  A tensor core takes bf16 operands.  A value is handed over as one bf16 (relative error 2^-9), or as the sum of
// three, which is all 24 bits of an fp32 value; products of pieces whose orders sum to more than two are below 2^-24 and left
// out.  K' is always three pieces, because the last state is an fp32 result.  Scores and state take one piece for
// outputs of bf16: each of the two parts of an output has then been rounded once more than the output itself, which
// together is about as much as the output's own rounding.  They take three where outputs are fp32 (kState = 3), and
// so do fp32 inputs (kInput = 3).
//
// All exponents are differences G_i - G_j in base 2 with their whole part kept as an integer, exact to 2^-24 whatever lies
// between; an empty state (-inf) is a step of -2^20.
#pragma once

#include "fss_linattn.cuh"
#include "fss_umma.cuh"

namespace fss {
namespace linattn {
namespace mma {

constexpr int kChunk = 64, kThreads = 256, kPanel = kChunk * 128;      // kPanel: bytes of 64 tokens x 64 channels
constexpr int kValues = 128;                                           // value channels of a CTA

// kLoad: how the tokens come into shared memory
enum Load { kTma = 0, kPlain = 1 };

template <int KD, int kInput, int kState, bool kOut> struct Plan {
    static constexpr int kPanels = KD / 64;
    static constexpr int kKeyPiece = kPanels * kPanel, kValuePiece = 2 * kPanel;
    // Q first: its product reads 128 rows, of which the upper half lies behind its panels
    static constexpr int kQ = 0, kK = kQ + (kOut ? kInput * kKeyPiece : 0), kV = kK + 3 * kKeyPiece, kP = kV + kInput * kValuePiece;
    static constexpr int kEnd = kP + (kOut ? kState * kPanel : 0);
    static constexpr int kShared = kEnd + 1024;      // (the base is moved up to a multiple of 1,024)
    // tensor memory
    static constexpr int kO1 = 0, kScores = 64, kAdded = kOut ? 128 : 0;
    static constexpr int kColumns = !kOut ? 128 : kState == 1 ? 256 : 512;
    // the state's column of key channels 16 s .. 16 s + 15 of a piece.  One piece lies over the columns that its own
    // threads have read the state's increment from: each half of the threads has a half of the key channels
    static __device__ __forceinline__ int state_column(int piece, int s) {
        if (kState == 1) return kAdded + s / (KD / 32) * (KD / 2) + s % (KD / 32) * 8;
        return 256 + piece * 64 + s * 8;
    }
};

struct Maps { CUtensorMap q, k, v; };

// What a chunk's decays come to, by row.
struct Decays {
    float enter[kChunk];      // e^{G_i} times the outputs' scale
    float leave[kChunk];      // e^{G_last - G_j} times the scale of k v^T; 0 for rows that are not there
    int whole[kChunk];        // floor of G in base 2
    float part[kChunk];       // and the rest
    float all;                // e^{G_last}
};

// One warp: the decays of visits s0 .. s0 + 63, two for each lane; returns the chunk's sum in base 2.
__device__ __forceinline__ double chunk_decays(Decays *d, const Problem &p, int64_t b, int64_t h, int64_t s0, int64_t len, int lane) {
    constexpr double kLog2e = 1.4426950408889634, kEmpty = -1048576.0;
    double g[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int64_t s = s0 + 2 * lane + i;
        g[i] = s < len ? (double)p.log_decay(b, h, s, len) * kLog2e : 0.0;
        if (g[i] < kEmpty) g[i] = kEmpty;      // (a NaN stays one)
    }
    double sum = g[0] + g[1];
#pragma unroll
    for (int w = 1; w < 32; w <<= 1) {
        const double x = __shfl_up_sync(0xffffffffu, sum, w);
        if (lane >= w) sum += x;
    }
    const double last = __shfl_sync(0xffffffffu, sum, 31);
    const double G[2] = {sum - g[1], sum};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int visit = 2 * lane + i, row = p.reverse ? kChunk - 1 - visit : visit;
        const bool there = s0 + visit < len;
        const double whole = floor(G[i]);
        d->whole[row] = (int)whole;
        d->part[row] = (float)(G[i] - whole);
        d->enter[row] = exp2f((float)G[i]) * p.out_scale;
        d->leave[row] = there ? exp2f((float)(last - G[i])) * p.in_scale : 0.f;
    }
    if (lane == 0) d->all = exp2f((float)last);
    return last;
}

// x as the sum of `n` bf16 values, pairs packed
template <int n> __device__ __forceinline__ void pieces(float x, float y, uint32_t (&w)[n]) {
#pragma unroll
    for (int i = 0; i < n; ++i) {
        w[i] = umma::pack(x, y);
        if (i + 1 < n) {
            x -= umma::low(w[i]);
            y -= umma::high(w[i]);
        }
    }
}

__device__ __forceinline__ uint32_t unit_address(uint32_t base, int row, int channel) {      // of 8 channels, in the swizzle
    return base + channel / 64 * kPanel + row * 128 + ((channel % 64 / 8) ^ (row & 7)) * 16;
}
__device__ __forceinline__ void store_shared16(uint32_t at, const uint32_t (&w)[4]) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
}
__device__ __forceinline__ void load_shared16(uint32_t at, uint32_t (&w)[4]) {
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
}

// The chunk's rows of one tensor by ordinary loads, in `n` pieces; zeros for channels and rows that are not there.
template <typename T, int n> __device__ __forceinline__ void load_rows(uint32_t base, int piece, const T *x, int64_t stride, int first, int last, int D,
                                                                       int padded, bool vec) {
    for (int i = threadIdx.x; i < kChunk * padded / 8; i += kThreads) {
        const int row = i / (padded / 8), c = i % (padded / 8) * 8;
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = 0.f;
        if (row >= first && row < last && c < D) {
            const T *at = x + row * stride + c;
            if (vec && c + 8 <= D) {
                constexpr int V = VecWidth<T>::value;
#pragma unroll
                for (int j = 0; j < 8; j += V) {
                    float y[V];
                    Frag<T, V>::load(at + j, y);
#pragma unroll
                    for (int e = 0; e < V; ++e) f[j + e] = y[e];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (c + j < D) f[j] = (float)at[j];
            }
        }
        uint32_t w[n][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t y[n];
            pieces<n>(f[2 * j], f[2 * j + 1], y);
#pragma unroll
            for (int m = 0; m < n; ++m) w[m][j] = y[m];
        }
#pragma unroll
        for (int m = 0; m < n; ++m) store_shared16(unit_address(base + m * piece, row, c), w[m]);
    }
}

template <typename T, typename TO, int KD, int kLoad, int kInput, int kState, bool kOut>
__global__ void __launch_bounds__(kThreads, kOut && kState > 1 ? 1 : kInput > 1 ? 1 : 2)
    chunked(Problem p, const __grid_constant__ Maps maps, Heads<const T> q, Heads<const T> k, Heads<const T> v, Heads<TO> o, int v_tiles, int flags,
            int32_t *status) {
    using L = Plan<KD, kInput, kState, kOut>;
    extern __shared__ char raw[];
    __shared__ Decays decays[2];
    __shared__ __align__(8) uint64_t barriers[3];
    __shared__ uint32_t tmem_slot;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, half = warp / 4;
    const uint32_t base = (umma::shared_address(raw) + 1023u) & ~1023u;
    const uint32_t loaded = umma::shared_address(&barriers[0]), scored = umma::shared_address(&barriers[1]), added = umma::shared_address(&barriers[2]);
    int64_t id = blockIdx.x;
    const int vt = id % v_tiles;
    id /= v_tiles;
    const int seg = id % p.nseg;
    id /= p.nseg;
    const int64_t h = id % p.H, b = id / p.H, len = p.length(b);
    const int Dv = min(p.Dv - vt * kValues, kValues);      // of this CTA
    const bool vec = flags & 1, packed = sizeof(TO) == 2 && (flags & 2);
    const int64_t begin = seg * p.seg_len, end = min((int64_t)p.T, begin + p.seg_len), stop = min(end, len);
    const int v_panels = Dv > 64 ? 2 : 1;
    const T *k_rows = k.row(b, 0, h), *q_rows = kOut ? q.row(b, 0, h) : nullptr, *v_rows = v.row(b, 0, h) + vt * kValues;
    const int k_head = (int)(h / k.group), q_head = kOut ? (int)(h / q.group) : 0, v_head = (int)(h / v.group);
    TO *out = kOut ? o.row(b, 0, h) + vt * kValues : nullptr;
    bool gave_up = false;

    if (warp == 0) umma::tmem_alloc<L::kColumns>(umma::shared_address(&tmem_slot));
    if (threadIdx.x == 32) {
        for (int i = 0; i < 3; ++i) umma::barrier_init(umma::shared_address(&barriers[i]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // channels that no load writes
    if (kLoad == kTma && v_panels == 1)
        for (int i = threadIdx.x; i < kPanel / 16; i += kThreads) {
            const uint32_t zero[4] = {0, 0, 0, 0};
            store_shared16(base + L::kV + kPanel + i * 16, zero);
        }

    // the state that enters: lane = value channel, this half's key channels
    constexpr int kMine = KD / 2;
    const int dv = (warp % 4) * 32 + lane, key0 = half * kMine;
    float state[kMine];
    {
        const float *from = nullptr;
        int64_t sk = p.Dv, sv = 1;
        if (p.nseg > 1) {
            if (kOut) from = p.seg_state + ((b * p.H + h) * p.nseg + seg) * (int64_t)p.Dk * p.Dv;
        } else if (p.state_in) {
            from = p.state_in + (b * p.H + h) * (int64_t)p.Dk * p.Dv;
            sk = p.sk;
            sv = p.sv;
        }
#pragma unroll
        for (int i = 0; i < kMine; ++i) state[i] = from && dv < Dv && key0 + i < p.Dk ? from[(key0 + i) * sk + (vt * kValues + dv) * sv] : 0.f;
    }
    umma::fence_async_shared();
    umma::before_sync();
    __syncthreads();
    umma::after_sync();
    const uint32_t tmem = tmem_slot, lanes = (uint32_t)(warp % 4) * 32 << 16;

    const auto write_state = [&] {      // as the operand of the next chunk's outputs
#pragma unroll
        for (int i = 0; i < kMine; i += 16) {
            uint32_t w[kState][8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                uint32_t y[kState];
                pieces<kState>(state[i + 2 * j], state[i + 2 * j + 1], y);
#pragma unroll
                for (int m = 0; m < kState; ++m) w[m][j] = y[m];
            }
#pragma unroll
            for (int m = 0; m < kState; ++m) umma::tmem_store8(tmem + lanes + L::state_column(m, (key0 + i) / 16), w[m]);
        }
        umma::tmem_wait_stores();
    };
    const auto first_token = [&](int64_t s0) { return p.reverse ? len - s0 - kChunk : s0; };
    const auto load = [&](int64_t s0) {
        const int64_t t0 = first_token(s0);
        if (kLoad == kTma) {
            if (threadIdx.x == 64) {
                umma::barrier_expect(loaded, (uint32_t)(((kOut ? 2 : 1) * L::kPanels + v_panels) * kPanel));
                for (int c = 0; c < L::kPanels; ++c) {
                    umma::tma_load(base + L::kK + c * kPanel, &maps.k, c * 64, k_head, (int)t0, (int)b, loaded);
                    if (kOut) umma::tma_load(base + L::kQ + c * kPanel, &maps.q, c * 64, q_head, (int)t0, (int)b, loaded);
                }
                for (int c = 0; c < v_panels; ++c)
                    umma::tma_load(base + L::kV + c * kPanel, &maps.v, vt * kValues + c * 64, v_head, (int)t0, (int)b, loaded);
            }
        } else {
            const int there = (int)min((int64_t)kChunk, stop - s0), first = p.reverse ? kChunk - there : 0, last = p.reverse ? kChunk : there;
            load_rows<T, kInput>(base + L::kK, L::kKeyPiece, k_rows + t0 * k.st, k.st, first, last, p.Dk, KD, vec);
            if (kOut) load_rows<T, kInput>(base + L::kQ, L::kKeyPiece, q_rows + t0 * q.st, q.st, first, last, p.Dk, KD, vec);
            load_rows<T, kInput>(base + L::kV, L::kValuePiece, v_rows + t0 * v.st, v.st, first, last, Dv, kValues, vec);
        }
    };

    double total = 0.0;      // warp 3: the logarithm of the decay of all chunks
    if (begin < stop) {
        load(begin);
        if (warp == 3) total += chunk_decays(&decays[0], p, b, h, begin, len, lane);
        if (kOut) write_state();
    }
    umma::fence_async_shared();
    umma::before_sync();
    __syncthreads();
    umma::after_sync();

    // operands (steps and pieces are added to the address field, in units of 16 bytes)
    const uint64_t queries = umma::operand(base + L::kQ, 16), keys = umma::operand(base + L::kK, 16), values = umma::operand(base + L::kV, kPanel),
                   scores = umma::operand(base + L::kP, 16), decayed = umma::operand(base + L::kK, kPanel);
    uint32_t parity = 0, lost = 2;      // lost: the phase whose copies did not come
    for (int64_t s0 = begin; s0 < stop; s0 += kChunk, parity ^= 1) {
        const Decays &d = decays[parity];
        const int there = (int)min((int64_t)kChunk, stop - s0);      // tokens of the chunk
        const int64_t t0 = first_token(s0);
        if (kLoad == kTma) {
            const bool before = gave_up;
            umma::barrier_wait(loaded, parity, gave_up);
            if (gave_up && !before) lost = parity;
            if (there < kChunk) {
                // Rows behind the sequence hold anything.  Scores and keys of such rows are replaced by zeros below; values
                // meet those zeros in a product, so they have to be numbers.
                for (int i = threadIdx.x; i < v_panels * kChunk * 8; i += kThreads) {
                    const int row = i / 8 % kChunk;
                    const uint32_t zero[4] = {0, 0, 0, 0};
                    if ((p.reverse ? kChunk - 1 - row : row) >= there) store_shared16(base + L::kV + i / (8 * kChunk) * kPanel + row * 128 + i % 8 * 16, zero);
                }
            }
        }
        if (kOut && threadIdx.x == 64) {
            constexpr uint32_t what = umma::product(128, kChunk, false, false);
            bool more = false;
            // (small pieces first: what a sum in fp32 loses goes by its size)
#pragma unroll
            for (int a = kInput - 1; a >= 0; --a)
#pragma unroll
                for (int c = kInput - 1; c >= 0; --c)
#pragma unroll
                    for (int s = 0; s < (a + c < 3 ? KD / 16 : 0); ++s, more = true)
                        umma::multiply(tmem + L::kScores, queries + ((a * L::kKeyPiece + s / 4 * kPanel + s % 4 * 32) >> 4),
                                       keys + ((c * L::kKeyPiece + s / 4 * kPanel + s % 4 * 32) >> 4), what, more);
            more = false;
#pragma unroll
            for (int a = kState - 1; a >= 0; --a)
#pragma unroll
                for (int c = kInput - 1; c >= 0; --c)
#pragma unroll
                    for (int s = 0; s < (a + c < 3 ? KD / 16 : 0); ++s, more = true)
                        umma::multiply_tmem(tmem + L::kO1, tmem + L::state_column(a, s),
                                            queries + ((c * L::kKeyPiece + s / 4 * kPanel + s % 4 * 32) >> 4), what, more);
            umma::tell_when_done(scored);
        }
        // decayed keys: a unit of 8 channels of a row at a time, over the keys themselves once the scores are made
        constexpr int kUnits = kChunk * KD / 8 / kThreads;
        uint32_t unit[kUnits][kInput][4];
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            const int at = threadIdx.x + i * kThreads, row = at / (KD / 8), c = at % (KD / 8) * 8;
#pragma unroll
            for (int m = 0; m < kInput; ++m) load_shared16(unit_address(base + L::kK + m * L::kKeyPiece, row, c), unit[i][m]);
        }
        if (kOut) umma::barrier_wait(scored, parity, gave_up);
        umma::after_sync();
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            const int at = threadIdx.x + i * kThreads, row = at / (KD / 8), c = at % (KD / 8) * 8;
            const float f = d.leave[row];
            const bool here = (p.reverse ? kChunk - 1 - row : row) < there;
            uint32_t w[3][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float x = umma::low(unit[i][0][j]), y = umma::high(unit[i][0][j]);
                if (kInput == 3) {      // (exact: the pieces do not overlap)
                    x = (umma::low(unit[i][kInput - 1][j]) + umma::low(unit[i][kInput / 2][j])) + x;
                    y = (umma::high(unit[i][kInput - 1][j]) + umma::high(unit[i][kInput / 2][j])) + y;
                }
                uint32_t z[3];
                pieces<3>(here ? x * f : 0.f, here ? y * f : 0.f, z);
#pragma unroll
                for (int m = 0; m < 3; ++m) w[m][j] = z[m];
            }
#pragma unroll
            for (int m = 0; m < 3; ++m) store_shared16(unit_address(base + L::kK + m * L::kKeyPiece, row, c), w[m]);
        }
        if (kOut && warp % 4 < 2) {
            // scores: this thread's query, half of the keys
            const int i = warp % 4 * 32 + lane;
            const int whole = d.whole[i], visit = p.reverse ? kChunk - 1 - i : i;
            const float part = d.part[i], scale = p.in_scale * p.out_scale;
#pragma unroll
            for (int j0 = 0; j0 < 32; j0 += 16) {
                uint32_t r[16];
                umma::tmem_load16(tmem + lanes + L::kScores + half * 32 + j0, r);
                umma::tmem_wait_loads();
#pragma unroll
                for (int e = 0; e < 16; e += 8) {
                    uint32_t w[kState][4];
#pragma unroll
                    for (int f = 0; f < 8; f += 2) {
                        float x[2];
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const int j = half * 32 + j0 + e + f + u, other = p.reverse ? kChunk - 1 - j : j;
                            const int power = min(max(whole - d.whole[j], -127), 128);
                            const float decay = umma::exp2_fast(part - d.part[j]) * __int_as_float((power + 127) << 23);
                            x[u] = other <= visit && visit < there ? __uint_as_float(r[e + f + u]) * (decay * scale) : 0.f;
                        }
                        uint32_t y[kState];
                        pieces<kState>(x[0], x[1], y);
#pragma unroll
                        for (int m = 0; m < kState; ++m) w[m][f / 2] = y[m];
                    }
#pragma unroll
                    for (int m = 0; m < kState; ++m) store_shared16(unit_address(base + L::kP + m * kPanel, i, half * 32 + j0 + e), w[m]);
                }
            }
        }
        if (warp == 3 && s0 + kChunk < stop) total += chunk_decays(&decays[parity ^ 1], p, b, h, s0 + kChunk, len, lane);
        umma::fence_async_shared();
        umma::before_sync();
        __syncthreads();
        umma::after_sync();
        if (threadIdx.x == 64) {
            bool more = false;
            if (kOut) {
                constexpr uint32_t what = umma::product(kValues, kChunk, true, false);
#pragma unroll
                for (int a = kInput - 1; a >= 0; --a)
#pragma unroll
                    for (int c = kState - 1; c >= 0; --c)
#pragma unroll
                        for (int s = 0; s < (a + c < 3 ? kChunk / 16 : 0); ++s, more = true)
                            umma::multiply(tmem + L::kScores, values + ((a * L::kValuePiece + s * 2048) >> 4),
                                           scores + ((c * kPanel + s * 32) >> 4), what, more);
            }
            more = false;
            constexpr uint32_t what = umma::product(kValues, KD, true, true);
#pragma unroll
            for (int a = kInput - 1; a >= 0; --a)
#pragma unroll
                for (int c = 2; c >= 0; --c)
#pragma unroll
                    for (int s = 0; s < (a + c < 3 ? kChunk / 16 : 0); ++s, more = true)
                        umma::multiply(tmem + L::kAdded, values + ((a * L::kValuePiece + s * 2048) >> 4),
                                       decayed + ((c * L::kKeyPiece + s * 2048) >> 4), what, more);
            umma::tell_when_done(added);
        }
        umma::barrier_wait(added, parity, gave_up);
        umma::after_sync();
        if (s0 + kChunk < stop && !(kLoad == kTma && gave_up)) load(s0 + kChunk);
        const float all = d.all;
#pragma unroll
        for (int i = 0; i < kMine; i += 16) {
            uint32_t r[16];
            umma::tmem_load16(tmem + lanes + L::kAdded + key0 + i, r);
            umma::tmem_wait_loads();
#pragma unroll
            for (int j = 0; j < 16; ++j) state[i + j] = fmaf(all, state[i + j], __uint_as_float(r[j]));
        }
        if (kOut) {
            if (s0 + kChunk < stop) write_state();
            // outputs: lane = value channel, this half's 32 tokens
            TO *to = out + (t0 + half * 32) * o.st + (packed ? dv & ~1 : dv);
#pragma unroll
            for (int i0 = 0; i0 < 32; i0 += 16) {
                uint32_t r1[16], r2[16];
                umma::tmem_load16(tmem + lanes + L::kO1 + half * 32 + i0, r1);
                umma::tmem_load16(tmem + lanes + L::kScores + half * 32 + i0, r2);
                umma::tmem_wait_loads();
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                    const int row = half * 32 + i0 + e;
                    float x = fmaf(d.enter[row], __uint_as_float(r1[e]), __uint_as_float(r2[e]));
                    float y = fmaf(d.enter[row + 1], __uint_as_float(r1[e + 1]), __uint_as_float(r2[e + 1]));
                    const auto here = [&](int r) { return (p.reverse ? kChunk - 1 - r : r) < there; };
                    if (packed) {
                        // neighbouring lanes swap a token each, and store two channels of one
                        const float z = __shfl_xor_sync(0xffffffffu, lane % 2 ? x : y, 1);
                        const uint32_t w = lane % 2 ? umma::pack(z, y) : umma::pack(x, z);
                        const int mine = row + lane % 2;
                        if (here(mine) && dv < Dv) *reinterpret_cast<uint32_t *>(to + (i0 + e + lane % 2) * o.st) = w;
                    } else if (dv < Dv) {
                        if (here(row)) to[(i0 + e) * o.st] = (TO)x;
                        if (here(row + 1)) to[(i0 + e + 1) * o.st] = (TO)y;
                    }
                }
            }
        }
        umma::fence_async_shared();
        umma::before_sync();
        __syncthreads();
        umma::after_sync();
    }
    if (gave_up) report_status(status, FSS_STATUS_TMA_TIMEOUT);
    if (lost < 2) {      // copies that are still on their way: another two seconds before the CTA leaves its shared memory
        bool again = false;
        umma::barrier_wait(loaded, lost, again);
    }
    if (kOut) {
        const int64_t z0 = max(begin, len);
        for (int64_t i = threadIdx.x; i < (end - z0) * Dv; i += kThreads) out[(z0 + i / Dv) * o.st + i % Dv] = (TO)0.f;
    }
    if (!kOut || (p.nseg == 1 && p.state_out)) {
        float *to = kOut ? p.state_out + (b * p.H + h) * (int64_t)p.Dk * p.Dv : p.seg_state + ((b * p.H + h) * p.nseg + seg) * (int64_t)p.Dk * p.Dv;
        const int64_t sk = kOut ? p.sk : p.Dv, sv = kOut ? p.sv : 1;
        const float last = kOut && p.reverse && len > 0 ? expf(p.g[b * p.gsb + h * p.gsh]) : 1.f;
        if (!kOut && vt == 0 && threadIdx.x == 96) p.seg_decay[(b * p.H + h) * p.nseg + seg] = (float)exp2(total);
#pragma unroll
        for (int i = 0; i < kMine; ++i)
            if (dv < Dv && key0 + i < p.Dk) to[(key0 + i) * sk + (vt * kValues + dv) * sv] = state[i] * last;
    }
    umma::before_sync();
    __syncthreads();
    if (warp == 0) umma::tmem_free<L::kColumns>(tmem);
}

}  // namespace mma
}  // namespace linattn
}  // namespace fss
