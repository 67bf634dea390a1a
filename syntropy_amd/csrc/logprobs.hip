// Log probabilities of given tokens, entropy and most probable tokens of each row of logits x [rows][vocab]:
//   m = max x, d_i = (x_i - m) scale, s = sum exp d_i, e = sum exp(d_i) d_i;  log p_i = d_i - log s;
//   H = log s - e / s;  rank = the number of logits above the token's;
//   the `top` first tokens by (logit descending, index ascending).
// A row with nothing visible (all -infinity) has log probabilities of -infinity and the entropy 0; a NaN or
// +infinity in it makes them NaN (their exponential is one).  A NaN orders above everything.
//
// One pass, bound by reading the logits once.  A wavefront takes steps of 64 lanes x 16 values; each lane
// keeps its own running m, s and e and rescales them where its maximum grows, so that no lane waits for
// another until the end.  For the greatest ones the pass keeps each lane's maximum over every few steps (a
// group, at most 32 of them) in LDS and nothing more: the top-th of the 256 lanes' maxima is a bound that
// only a few values besides those maxima reach, and the lanes that reach it read their groups that do again.
// (Looking at each step's values as they come costs more than the sums: the bound is low at first, and a
// step of 1024 values nearly always holds one above it.)  Those values as keys (ordered value, then the
// index from below; all different) are gathered in LDS in any order, and each finds its place by counting
// the greater ones: a few dozen, in less time and code than a sort across lanes.  Where equal values fill the
// LDS, the `top` greatest of it stay and raise the bound.
//
// Few long rows are split over workgroups, whose parts a second launch joins.
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"

namespace syn {

namespace {

constexpr int LP_VALUES = 16;              // a lane's values a step
constexpr int LP_STEP = 64 * LP_VALUES;
constexpr int lp_groups(int waves) { return waves > 4 ? 16 : 32; }
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

// A whole number that orders as the value does (-0 as +0, every NaN above +infinity), and the value again.
SYN_DEV uint32_t lp_order(float v) {
    if (v != v) return 0xFFFFFFFFu;
    const uint32_t b = f2u(v + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
SYN_DEV float lp_value(uint32_t k) { return u2f(k >> 31 ? k ^ 0x80000000u : ~k); }
// (an index is below 2^31 - 256, so a key is never 0: that is none)
SYN_DEV uint64_t lp_key(float v, int i) { return (uint64_t)lp_order(v) << 32 | (0x7FFFFFFFu - (uint32_t)i); }
SYN_DEV int lp_index(uint64_t k) { return (int)(0x7FFFFFFFu - (uint32_t)k); }

// The greatest number that at least n of a wavefront's values (four a lane) reach, but for its last 14 bits
// (which let a few more values pass).  Two bits a turn: a turn is the wait for the counts.
SYN_DEV uint32_t reached_by(const uint32_t (&v)[4], int n) {
    uint32_t r = 0;
#pragma unroll 1
    for (int at = 30; at >= 14; at -= 2) {
        int c[3] = {0, 0, 0};
#pragma unroll
        for (uint32_t b = 1; b < 4; ++b)
#pragma unroll
            for (int j = 0; j < 4; ++j) c[b - 1] += __builtin_popcountll(__builtin_amdgcn_ballot_w64(v[j] >= (r | b << at)));
        r |= (c[2] >= n ? 3u : c[1] >= n ? 2u : c[0] >= n ? 1u : 0u) << at;
    }
    return r;
}

constexpr int LP_ROOM = 512;
// The greatest keys so far of a workgroup of W wavefronts, in LDS.
template <int W>
struct Greatest {
    uint64_t keys[LP_ROOM];                // in any order
    uint64_t sorted[LOGPROB_MAX_TOP];      // of sort()
    uint32_t most[64 * W];                 // the lanes' greatest
    int count;                             // of keys, and of those that found no room
    int more[W];
    uint32_t reached;                      // of bound()

    // (every thread) a number that at least `top` keys reach, from the lanes' greatest values' orders: of 256
    // values, each of W / 4 lanes.  One wavefront counts; all of them would be in each other's way.
    SYN_DEV uint32_t bound(uint32_t mine, int top) {
        most[threadIdx.x] = mine;
        if (threadIdx.x == 0) count = 0;
        __syncthreads();
        if (threadIdx.x < 64) {
            uint32_t of[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                of[j] = 0;
#pragma unroll
                for (int w = j; w < W; w += 4) {
                    const uint32_t v = most[64 * w + threadIdx.x];
                    of[j] = v > of[j] ? v : of[j];
                }
            }
            const uint32_t r = reached_by(of, top);
            if (threadIdx.x == 0) reached = r;
        }
        __syncthreads();
        return reached;
    }
    // (every thread; a barrier before and after) the `top` greatest in order; returns how many there are
    SYN_DEV int sort(int top) {
        const int n = count < LP_ROOM ? count : LP_ROOM;
        for (int j = threadIdx.x; j < n; j += 64 * W) {
            const uint64_t k = keys[j];
            int rank = 0;
#pragma unroll 4
            for (int i = 0; i < n; ++i) rank += keys[i] > k ? 1 : 0;
            if (rank < top) sorted[rank] = k;
        }
        return n < top ? n : top;
    }
    // true where it found no room
    SYN_DEV bool put(uint64_t k) {
        const int at = atomicAdd(&count, 1);
        if (at < LP_ROOM) keys[at] = k;
        return at >= LP_ROOM;
    }
    // (every thread, after put) whether any thread has more to put; where there is no room left, the bound is
    // raised to the top-th of what there is, and only the greatest stay
    SYN_DEV bool round(bool mine, int top, uint64_t& bound) {
        const bool any = __builtin_amdgcn_ballot_w64(mine) != 0;
        if ((threadIdx.x & 63) == 0) more[threadIdx.x >> 6] = any;
        __syncthreads();
        bool go = false;
        for (int w = 0; w < W; ++w) go |= more[w] != 0;
        const bool full = count >= LP_ROOM;
        if (go || full) __syncthreads();  // uniform: everyone has read what the next round writes
        if (full) {
            sort(top);
            __syncthreads();
            const uint64_t b = sorted[top - 1];
            bound = b > bound ? b : bound;
            if ((int)threadIdx.x < top) keys[threadIdx.x] = sorted[threadIdx.x];
            if (threadIdx.x == 0) count = top;
            __syncthreads();
        }
        return go;
    }
};
static_assert(LP_ROOM > LOGPROB_MAX_TOP, "room behind those that stay");

// A running softmax: the greatest value m; with t_i = (x_i - m) c, c = scale log2(e), the sum of 2^t_i and that
// of 2^t_i t_i.  (A t below -150 has the power 0, and one of -300 stands for it in the second sum, for
// -infinity times 0 is a NaN.)
constexpr float LP_LEAST = -300.0f;
struct Soft {
    float m = -__builtin_inff(), s = 0.0f, e = 0.0f;
    // to the maximum n >= m (a lane that has seen nothing but -infinity and NaN keeps its sums, 0 or NaN)
    SYN_DEV void rebase(float n, float c) {
        const float t = m == -__builtin_inff() ? 0.0f : fmaxf((m - n) * c, LP_LEAST);
        const float f = __builtin_amdgcn_exp2f(t);
        e = f * __builtin_fmaf(t, s, e);
        s = f * s;
        m = n;
    }
    SYN_DEV void add(Soft o, float c) {
        const float n = fmaxf(m, o.m);
        rebase(n, c);
        o.rebase(n, c);
        s += o.s;
        e += o.e;
    }
    SYN_DEV float base() const { return m == -__builtin_inff() ? 0.0f : m; }
};
SYN_DEV float max_of_lanes(float v) {
    for (int d = 1; d < 64; d *= 2) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}
SYN_DEV Soft soft_of_lanes(Soft v, float c) {
    v.rebase(max_of_lanes(v.m), c);
    for (int d = 1; d < 64; d *= 2) {
        v.s += __shfl_xor(v.s, d);
        v.e += __shfl_xor(v.e, d);
    }
    return v;
}

template <int TY>
struct Values {
    static constexpr int WORDS = TY == T_F32 ? 16 : 8, PER = TY == T_F32 ? 4 : 8;  // values a 16-byte piece
    uint32_t w[WORDS];

    // value i of lane l in the step from `first` on: index first + 64 PER (i / PER) + PER l + i % PER
    static SYN_DEV int index(int first, int i) {
        return first + 64 * PER * (i / PER) + PER * (int)(threadIdx.x & 63) + i % PER;
    }
    // The step's values, -infinity past the row's end; `first` may be another in every lane.  (The row's last
    // step one value a load, each at an index that is there: a branch around each would wait for the one
    // before.)
    SYN_DEV void load(const uint8_t* row, int first, int vocab) {
        if (__builtin_amdgcn_ballot_w64(first + LP_STEP > vocab) == 0) {  // uniform
#pragma unroll
            for (int p = 0; p < LP_VALUES / PER; ++p)  // (pieces at any value's address)
                __builtin_memcpy(w + 4 * p, row + (int64_t)index(first, PER * p) * (16 / PER), 16);
            return;
        }
        uint32_t v[LP_VALUES];
#pragma unroll
        for (int i = 0; i < LP_VALUES; ++i) {
            const int id = index(first, i), in = id < vocab ? id : vocab - 1;
            if constexpr (TY == T_F32)
                v[i] = ((const uint32_t*)row)[in];
            else
                v[i] = ((const uint16_t*)row)[in];
        }
#pragma unroll
        for (int i = 0; i < LP_VALUES; ++i) {
            constexpr uint32_t NONE = TY == T_F32 ? 0xFF800000u : TY == T_F16 ? 0xFC00u : 0xFF80u;
            v[i] = index(first, i) < vocab ? v[i] : NONE;
        }
#pragma unroll
        for (int j = 0; j < WORDS; ++j) w[j] = TY == T_F32 ? v[j] : v[2 * j % LP_VALUES] | v[(2 * j + 1) % LP_VALUES] << 16;
    }
    SYN_DEV float at(int i) const {
        if constexpr (TY == T_F32) return u2f(w[i]);
        const uint32_t h = w[i / 2];
        if constexpr (TY == T_F16) return f16_to_f32(i & 1 ? h >> 16 : h);
        return u2f(i & 1 ? h & 0xFFFF0000u : h << 16);
    }
};

template <int TY>
SYN_DEV float lp_load(const uint8_t* row, int64_t i) {
    if constexpr (TY == T_F32) return ((const float*)row)[i];
    const uint32_t h = ((const uint16_t*)row)[i];
    return TY == T_F16 ? f16_to_f32(h) : u2f(h << 16);
}

SYN_DEV int64_t lp_token(const LogprobArgs& g, uint64_t row) {
    return g.wide ? ((const int64_t*)g.tokens)[row] : ((const int32_t*)g.tokens)[row];
}

// A part's results: m, s, e and the rank's count; its `top` greatest keys lie behind all parts.
struct Part {
    float m, s, e;
    uint32_t above;
};

// The row's results from its softmax, count and sorted keys, by one wavefront.
SYN_DEV void lp_write(const LogprobArgs& g, uint64_t row, const Soft& v, uint32_t above, float xt, int64_t t,
                      const uint64_t* sorted) {
    const int lane = threadIdx.x & 63;
    const bool none = v.s == 0.0f;
    const float ls = logf(v.s), base = v.base();
    if (lane == 0) {
        const bool known = t >= 0 && t < g.vocab;
        g.logprob[row] = t < 0 ? 0.0f : !known ? __builtin_nanf("") : none ? -__builtin_inff() : (xt - base) * g.scale - ls;
        g.rank[row] = known ? (int)above : -1;
        g.entropy[row] = none ? 0.0f : ls - v.e / v.s * LN2;
    }
    if (lane < g.top) {
        const uint64_t k = sorted[lane];
        g.top_ids[row * g.top + lane] = lp_index(k);
        g.top_logprobs[row * g.top + lane] = none ? -__builtin_inff() : (lp_value((uint32_t)(k >> 32)) - base) * g.scale - ls;
    }
}

}  // namespace

template <int TY, int TOP, int W>
__global__ __launch_bounds__(64 * W) void k_logprobs(LogprobArgs g, int parts, int part_steps, int group_steps) {
    const uint64_t row = blockIdx.x / (uint32_t)parts;
    const int part = (int)(blockIdx.x % (uint32_t)parts);
    const uint8_t* x = (const uint8_t*)g.x + row * g.ldx * (TY == T_F32 ? 4 : 2);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    __shared__ uint32_t groups[TOP ? W : 1][TOP ? lp_groups(W) : 1][64];
    __shared__ typename std::conditional<TOP != 0, Greatest<W>, int>::type best;
    __shared__ Part sums[W];
    const int steps = (g.vocab + LP_STEP - 1) / LP_STEP;
    const int last = (part + 1) * part_steps < steps ? (part + 1) * part_steps : steps;
    const int step0 = part * part_steps + wave;
    int step = step0;

    using V = Values<TY>;
    V cur, nxt;
    if (step < last) cur.load(x, step * LP_STEP, g.vocab);
    const int64_t t = lp_token(g, row);
    const bool known = t >= 0 && t < g.vocab;
    const float xt = known ? lp_load<TY>(x, t) : __builtin_nanf("");  // (nothing is above a NaN)

    const float c = g.scale * LOG2E;
    Soft v;
    uint32_t above = 0;
    float most = -__builtin_inff(), group = most;  // the lane's greatest value, and that of its group
    int in_group = 0, n_groups = 0;
    while (step < last) {  // uniform
        step += W;
        if (step < last) nxt.load(x, step * LP_STEP, g.vocab);
        float mx = cur.at(0);
#pragma unroll
        for (int i = 1; i < LP_VALUES; ++i) mx = fmaxf(mx, cur.at(i));
        const float n = fmaxf(v.m, mx);
        if (__builtin_amdgcn_ballot_w64(n > v.m) != 0) v.rebase(n, c);
        const float base = v.base();
#pragma unroll
        for (int i = 0; i < LP_VALUES; ++i) {
            const float xi = cur.at(i), t2 = (xi - base) * c, p = __builtin_amdgcn_exp2f(t2);
            v.s += p;
            v.e = __builtin_fmaf(p, fmaxf(t2, LP_LEAST), v.e);
            above += (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(xi > xt));
        }
        if constexpr (TOP) {
            group = fmaxf(group, mx);
            if (++in_group == group_steps || step >= last) {
                most = fmaxf(most, group);
                // (once a NaN or +infinity is in the sum, every group may hold a NaN)
                groups[wave][n_groups++][lane] = v.s != v.s ? 0xFFFFFFFFu : lp_order(group);
                group = -__builtin_inff();
                in_group = 0;
            }
        }
        cur = nxt;
    }
    if constexpr (TOP) {
        const uint32_t b = best.bound(lp_order(most), g.top);
        uint64_t bound = b ? ((uint64_t)b << 32) - 1 : 0;  // all of that value are above it
        uint32_t mine = 0;  // the lane's groups that reach it
        for (int i = 0; i < n_groups; ++i) mine |= groups[wave][i][lane] >= b ? 1u << i : 0u;
        uint32_t may = 0;  // the lane's values of `cur` that may pass (a NaN may)
        int at = 0, in = 0;
        bool go = true;
#pragma unroll 1
        while (go) {  // uniform
            if (may == 0 && mine != 0) {  // the lane's next step
                const int gi = __builtin_ctz(mine), st = step0 + (gi * group_steps + in) * W;
                at = st * LP_STEP;
                // (equal values: a group behind the bound's index holds nothing before it)
                if (st < last &&
                    ((uint64_t)groups[wave][gi][lane] << 32 | (0x7FFFFFFFu - (uint32_t)V::index(at, 0))) > bound) {
                    const float bv = lp_value((uint32_t)((bound + 1) >> 32));
                    cur.load(x, at, g.vocab);
#pragma unroll
                    for (int i = 0; i < LP_VALUES; ++i) may |= !(cur.at(i) < bv) ? 1u << i : 0u;
                }
                if (++in == group_steps) in = 0, mine &= mine - 1;
            }
#pragma unroll 1
            for (; may != 0; may &= may - 1) {  // each lane its own
                const int i = __builtin_ctz(may), id = V::index(at, i);
                if (id >= g.vocab) continue;
                const uint64_t key = lp_key(lp_load<TY>(x, id), id);  // (a choice of the registers by lane costs more)
                if (key > bound && best.put(key)) break;
            }
            go = best.round(may != 0 || mine != 0, g.top, bound);
        }
        const int n = best.sort(g.top);
        if ((int)threadIdx.x >= n && (int)threadIdx.x < g.top) best.sorted[threadIdx.x] = 0;
    }
    v = soft_of_lanes(v, c);
    if (lane == 0) sums[wave] = Part{v.m, v.s, v.e, above};
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < W; ++w) {
        const Part o = sums[w];
        Soft ov;
        ov.m = o.m;
        ov.s = o.s;
        ov.e = o.e;
        v.add(ov, c);
        above += o.above;
    }
    const uint64_t* sorted = nullptr;
    if constexpr (TOP) sorted = best.sorted;
    if (parts == 1) {
        lp_write(g, row, v, above, xt, t, sorted);
    } else {
        if (lane == 0) ((Part*)g.ws)[row * parts + part] = Part{v.m, v.s, v.e, above};
        uint64_t* keys = (uint64_t*)(g.ws + (uint64_t)g.rows * parts * sizeof(Part));
        if (TOP && lane < g.top) keys[(row * parts + part) * g.top + lane] = sorted[lane];
    }
}

// The parts of a row.
template <int TY, int TOP>
__global__ __launch_bounds__(TOP ? 256 : 64) void k_logprobs_join(LogprobArgs g, int parts) {
    const uint64_t row = blockIdx.x;
    const int lane = threadIdx.x & 63;
    __shared__ typename std::conditional<TOP != 0, Greatest<4>, int>::type best;
    const Part* from = (const Part*)g.ws + row * parts;
    const int64_t t = lp_token(g, row);
    const float xt = t >= 0 && t < g.vocab ? lp_load<TY>((const uint8_t*)g.x + row * g.ldx * (TY == T_F32 ? 4 : 2), t) : 0.0f;
    const float c = g.scale * LOG2E;
    Soft v;
    uint32_t above = 0;
    if (lane < parts) {  // (at most 64)
        const Part o = from[lane];
        v.m = o.m;
        v.s = o.s;
        v.e = o.e;
        above = o.above;
    }
    const uint64_t* sorted = nullptr;
    if constexpr (TOP) {
        const uint64_t* keys = (const uint64_t*)(g.ws + (uint64_t)g.rows * parts * sizeof(Part)) + row * parts * g.top;
        const int n = parts * g.top;
        uint64_t k = (int)threadIdx.x < n ? keys[threadIdx.x] : 0, mx = k;
        for (int i = threadIdx.x + 256; i < n; i += 256) mx = keys[i] > mx ? keys[i] : mx;
        const uint32_t b = best.bound((uint32_t)(mx >> 32), g.top);
        uint64_t bound = b ? ((uint64_t)b << 32) - 1 : 0;
        bool go = true;
        int i = threadIdx.x;
#pragma unroll 1
        while (go) {  // uniform
            if (i < n && !(k > bound && best.put(k))) {
                i += 256;
                k = i < n ? keys[i] : 0;
            }
            go = best.round(i < n, g.top, bound);
        }
        best.sort(g.top);  // (at least `top` of them: the vocabulary has as many)
        __syncthreads();
        if (threadIdx.x >= 64) return;
        sorted = best.sorted;
    }
    v = soft_of_lanes(v, c);
    for (int d = 1; d < 64; d *= 2) above += __shfl_xor(above, d);
    lp_write(g, row, v, above, xt, t, sorted);
}

// How a call runs: wavefronts a workgroup, parts of a row.  A workgroup of 16 wavefronts takes a whole row where
// the rows are few and not long, or nearly fill the chip: one launch (64 rows of 32064, 64 greatest, 14.9 us
// against 17.2 in parts; 256 rows of 128256 BF16 24.6 against 28.6, 145 F32 21.4 against 25.4; but 24 rows of
// 128256 22.1 against 16.8, 145 of 250000 BF16 31.0 against 27.3).  Other few
// and long rows are in parts, so that about 1024 workgroups of four keep reads in flight.
struct LpPlan {
    int waves, parts, part_steps, group_steps;
};
static LpPlan lp_plan(int rows, int vocab) {
    const int steps = (vocab + LP_STEP - 1) / LP_STEP;
    LpPlan p{4, 1, 0, 0};
    if (rows <= 256 && steps > 4 && (steps <= 64 || rows > 160 || (rows > 110 && steps <= 160))) {
        p.waves = 16;
    } else if (steps > 32) {
        const int most = (steps + 3) / 4 < 64 ? (steps + 3) / 4 : 64;
        p.parts = 1024 / rows < most ? 1024 / rows : most;
        p.parts = p.parts < 1 ? 1 : p.parts;
    }
    p.part_steps = (steps + p.parts - 1) / p.parts;
    const int wave_steps = (p.part_steps + p.waves - 1) / p.waves;
    p.group_steps = (wave_steps + lp_groups(p.waves) - 1) / lp_groups(p.waves);
    return p;
}

uint64_t logprob_ws_bytes(int rows, int vocab, int top) {
    if (rows == 0) return 0;
    const int p = lp_plan(rows, vocab).parts;
    return p > 1 ? align_up((uint64_t)rows * p * (sizeof(Part) + 8 * (uint64_t)top), 256) : 0;
}

template <int TY, int W>
static void logprobs_of(const LogprobArgs& a, const LpPlan& p, hipStream_t stream) {
    const dim3 grid((uint32_t)a.rows * (uint32_t)p.parts);
    if (a.top)
        hipLaunchKernelGGL((k_logprobs<TY, 1, W>), grid, dim3(64 * W), 0, stream, a, p.parts, p.part_steps, p.group_steps);
    else
        hipLaunchKernelGGL((k_logprobs<TY, 0, W>), grid, dim3(64 * W), 0, stream, a, p.parts, p.part_steps, p.group_steps);
}
template <int TY>
static void logprobs_as(const LogprobArgs& a, hipStream_t stream) {
    const LpPlan p = lp_plan(a.rows, a.vocab);
    p.waves == 16 ? logprobs_of<TY, 16>(a, p, stream) : logprobs_of<TY, 4>(a, p, stream);
    if (p.parts > 1 && a.top)
        hipLaunchKernelGGL((k_logprobs_join<TY, 1>), dim3(a.rows), dim3(256), 0, stream, a, p.parts);
    else if (p.parts > 1)
        hipLaunchKernelGGL((k_logprobs_join<TY, 0>), dim3(a.rows), dim3(64), 0, stream, a, p.parts);
}

void launch_logprobs(const LogprobArgs& a, hipStream_t stream) {
    if (a.xtype == T_F32)
        logprobs_as<T_F32>(a, stream);
    else if (a.xtype == T_F16)
        logprobs_as<T_F16>(a, stream);
    else
        logprobs_as<T_BF16>(a, stream);
}

}  // namespace syn
