// Log probabilities of given tokens, entropy and most probable tokens of each row of logits x [rows][vocab]:
//   z = x scale, m = max z, s = sum exp(z - m), e = sum exp(z - m) (z - m);  log p_i = (z_i - m) - log s;
//   H = log s - e / s;  rank = the number of logits above the token's;
//   the `top` first tokens by (logit descending, index ascending).
// A row with nothing visible (all -infinity) has log probabilities of -infinity and the entropy 0; a NaN or
// +infinity in it makes them NaN (their exponential is one).  A NaN orders above everything.
//
// One pass, bound by reading the logits once.  A wavefront takes steps of 64 lanes x 16 values; each lane
// keeps its own running m, s and e and rescales them where its maximum grows, so that no lane waits for
// another until the end.  The greatest ones are keys (ordered value, then the index from below), which are
// all different: a wavefront holds its 64 greatest, a lane each in order, and their top-th is a bound that
// almost no later value passes; a step is looked at closer only where a lane's maximum does.  What passes is
// gathered in LDS and sorted in 64 at a time (bitonic, across lanes without LDS).  The bound of the first
// step is the top-th of the lanes' maxima, and the wavefronts of a workgroup share the best bound.
//
// Few rows: a row is split over workgroups, whose parts a second launch joins.
#include "common.hpp"
#include "kernels.hpp"

namespace syn {

namespace {

constexpr int LP_WAVES = 4;
constexpr int LP_VALUES = 16;              // a lane's values a step
constexpr int LP_STEP = 64 * LP_VALUES;
constexpr float LOG2E = 1.44269504088896340736f;

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

// Lane l's word from lane l ^ D.
template <int D>
SYN_DEV uint32_t lane_xor(uint32_t v) {
    if constexpr (D == 1) return dpp_u32<DPP_XOR1>(v);
    if constexpr (D == 2) return dpp_u32<DPP_XOR2>(v);
    if constexpr (D == 4) return dpp_u32<0x1B>(dpp_u32<DPP_HALF_MIRROR>(v));  // 7 - l, then l ^ 3
    if constexpr (D == 8) return dpp_u32<0x128>(v);                           // rotated by 8 in a row of 16
    if constexpr (D == 16) {
        const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);  // rows 0, 0, 2, 2 and 1, 1, 3, 3
        return threadIdx.x & 16 ? s[0] : s[1];
    }
    if constexpr (D == 32) {
        const auto s = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return threadIdx.x & 32 ? s[0] : s[1];
    }
}
template <int D>
SYN_DEV uint64_t lane_xor64(uint64_t v) {
    return (uint64_t)lane_xor<D>((uint32_t)(v >> 32)) << 32 | lane_xor<D>((uint32_t)v);
}
// One exchange of a bitonic network: the greater of the pair to the lower lane where `down`, else to the upper.
template <int D>
SYN_DEV void exchange(uint64_t& k, bool down) {
    const uint64_t o = lane_xor64<D>(k);
    const bool lower = (threadIdx.x & D) == 0;
    k = (o > k) == (lower == down) ? o : k;
}
// 64 lanes' keys that rise to a lane and fall from it (or the other way): in descending order.
SYN_DEV void merge64(uint64_t& k) {
    exchange<32>(k, true);
    exchange<16>(k, true);
    exchange<8>(k, true);
    exchange<4>(k, true);
    exchange<2>(k, true);
    exchange<1>(k, true);
}
SYN_DEV void sort64(uint64_t& k) {
    const int l = threadIdx.x & 63;
    exchange<1>(k, (l & 2) == 0);
    exchange<2>(k, (l & 4) == 0);
    exchange<1>(k, (l & 4) == 0);
    exchange<4>(k, (l & 8) == 0);
    exchange<2>(k, (l & 8) == 0);
    exchange<1>(k, (l & 8) == 0);
    exchange<8>(k, (l & 16) == 0);
    exchange<4>(k, (l & 16) == 0);
    exchange<2>(k, (l & 16) == 0);
    exchange<1>(k, (l & 16) == 0);
    exchange<16>(k, (l & 32) == 0);
    exchange<8>(k, (l & 32) == 0);
    exchange<4>(k, (l & 32) == 0);
    exchange<2>(k, (l & 32) == 0);
    exchange<1>(k, (l & 32) == 0);
    merge64(k);
}
SYN_DEV uint64_t lane_key(uint64_t k, int lane) {  // uniform
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(k >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)k, lane);
}

// A wavefront's greatest keys so far.
struct Greatest {
    uint64_t list = 0;   // lane l: the l-th greatest
    uint64_t bound = 0;  // only a key above it can be among the `top` greatest
    int waiting = 0;     // keys in buf
    uint64_t* buf;       // LDS, 128 of this wavefront
    int top;

    SYN_DEV void take() {  // the first 64 of buf into the list
        const int l = threadIdx.x & 63;
        wave_lds_sync();
        uint64_t k = l < waiting ? buf[l] : 0;
        const uint64_t rest = buf[64 + l];
        wave_lds_sync();
        buf[l] = rest;
        waiting = waiting > 64 ? waiting - 64 : 0;
        // against the list in reverse, so that the pairs' greater ones are the 64 greatest
        sort64(k);
        const uint64_t rev = lane_xor64<32>(lane_xor64<16>(lane_xor64<8>(lane_xor64<4>(lane_xor64<2>(lane_xor64<1>(k))))));
        list = rev > list ? rev : list;
        merge64(list);
        const uint64_t b = lane_key(list, top - 1);
        bound = b > bound ? b : bound;
    }
    SYN_DEV void push(uint64_t k, bool pass) {
        const uint64_t m = __builtin_amdgcn_ballot_w64(pass);
        if (m == 0) return;  // uniform
        const int at = waiting + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
        if (pass) buf[at] = k;
        waiting += __builtin_popcountll(m);
        if (waiting >= 64) take();
    }
    SYN_DEV void finish() {
        while (waiting > 0) take();
    }
};

// A running softmax: the greatest, the sum of exponentials, the sum of exponentials times their arguments.
struct Soft {
    float m = -__builtin_inff(), s = 0.0f, e = 0.0f;
    // to the maximum n >= m (a lane that has seen nothing but -infinity and NaN keeps its sums, 0 or NaN)
    SYN_DEV void rebase(float n) {
        const float d = m == -__builtin_inff() ? 0.0f : fmaxf(m - n, -200.0f);  // (from -104 on the factor is 0)
        const float f = __builtin_amdgcn_exp2f(d * LOG2E);
        e = f * __builtin_fmaf(d, s, e);
        s = f * s;
        m = n;
    }
    SYN_DEV void add(Soft o) {
        const float n = fmaxf(m, o.m);
        rebase(n);
        o.rebase(n);
        s += o.s;
        e += o.e;
    }
    SYN_DEV float base() const { return m == -__builtin_inff() ? 0.0f : m; }
};
SYN_DEV Soft soft_of_lanes(Soft v) {
    for (int d = 1; d < 64; d *= 2) {
        Soft o;
        o.m = __shfl_xor(v.m, d);
        o.s = __shfl_xor(v.s, d);
        o.e = __shfl_xor(v.e, d);
        v.add(o);
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
    SYN_DEV void load(const uint8_t* row, int first, int vocab) {
        constexpr int ES = TY == T_F32 ? 4 : 2;
        if (first + LP_STEP <= vocab) {  // uniform; pieces at any value's address
#pragma unroll
            for (int p = 0; p < LP_VALUES / PER; ++p)
                __builtin_memcpy(w + 4 * p, row + (int64_t)index(first, PER * p) * ES, 16);
        } else {
#pragma unroll
            for (int j = 0; j < WORDS; ++j) {
                if constexpr (TY == T_F32) {
                    const int i = index(first, j);
                    w[j] = i < vocab ? ((const uint32_t*)row)[i] : 0xFF800000u;
                } else {
                    constexpr uint32_t NONE = TY == T_F16 ? 0xFC00u : 0xFF80u;
                    const int i = index(first, 2 * j);
                    const uint32_t lo = i < vocab ? ((const uint16_t*)row)[i] : NONE;
                    const uint32_t hi = i + 1 < vocab ? ((const uint16_t*)row)[i + 1] : NONE;
                    w[j] = lo | hi << 16;
                }
            }
        }
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

// A part's results: m, s, e and the rank's count, then its `top` greatest keys.
struct Part {
    float m, s, e;
    uint32_t above;
};
SYN_HD inline uint64_t part_bytes(int top) { return sizeof(Part) + 8 * (uint64_t)top; }

// The row's results from its softmax, count and list (lane l the l-th greatest), by one wavefront.
SYN_DEV void lp_write(const LogprobArgs& g, uint64_t row, const Soft& v, uint32_t above, float xt, int64_t t, uint64_t list) {
    const int lane = threadIdx.x & 63;
    const bool none = v.s == 0.0f;
    const float ls = logf(v.s), base = v.base();
    if (lane == 0) {
        const bool known = t >= 0 && t < g.vocab;
        g.logprob[row] = t < 0 ? 0.0f : !known ? __builtin_nanf("") : none ? -__builtin_inff() : (xt * g.scale - base) - ls;
        g.rank[row] = known ? (int)above : -1;
        g.entropy[row] = none ? 0.0f : ls - v.e / v.s;
    }
    if (lane < g.top) {
        g.top_ids[row * g.top + lane] = lp_index(list);
        g.top_logprobs[row * g.top + lane] =
            none ? -__builtin_inff() : (lp_value((uint32_t)(list >> 32)) * g.scale - base) - ls;
    }
}

}  // namespace

template <int TY, int TOP>
__global__ __launch_bounds__(64 * LP_WAVES) void k_logprobs(LogprobArgs g, int parts, int part_steps) {
    const uint64_t row = blockIdx.x / (uint32_t)parts;
    const int part = (int)(blockIdx.x % (uint32_t)parts);
    const uint8_t* x = (const uint8_t*)g.x + row * g.ldx * (TY == T_F32 ? 4 : 2);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    __shared__ uint64_t buf[TOP ? LP_WAVES : 1][TOP ? 128 : 1];
    __shared__ unsigned long long shared_bound;
    __shared__ Part sums[LP_WAVES];
    const int steps = (g.vocab + LP_STEP - 1) / LP_STEP;
    const int last = (part + 1) * part_steps < steps ? (part + 1) * part_steps : steps;
    int step = part * part_steps + wave;

    using V = Values<TY>;
    V cur, nxt;
    if (step < last) cur.load(x, step * LP_STEP, g.vocab);
    const int64_t t = lp_token(g, row);
    const bool known = t >= 0 && t < g.vocab;
    const float xt = known ? lp_load<TY>(x, t) : __builtin_nanf("");  // (nothing is above a NaN)
    if (TOP) {
        if (threadIdx.x == 0) shared_bound = 0;
        __syncthreads();
    }

    Soft v;
    uint32_t above = 0;
    Greatest best;
    best.buf = buf[TOP ? wave : 0];
    best.top = g.top;
    bool first = true;
    while (step < last) {  // uniform
        const int at = step * LP_STEP;
        step += LP_WAVES;
        if (step < last) nxt.load(x, step * LP_STEP, g.vocab);
        float mx = cur.at(0);
#pragma unroll
        for (int i = 1; i < LP_VALUES; ++i) mx = fmaxf(mx, cur.at(i));
        const float n = fmaxf(v.m, mx * g.scale);
        if (__builtin_amdgcn_ballot_w64(n > v.m) != 0) v.rebase(n);
        const float base = v.base();
#pragma unroll
        for (int i = 0; i < LP_VALUES; ++i) {
            const float xi = cur.at(i), d = xi * g.scale - base, p = __builtin_amdgcn_exp2f(d * LOG2E);
            v.s += p;
            v.e = __builtin_fmaf(p, fmaxf(d, -200.0f), v.e);  // (p is 0 from -104 on: nothing, not 0 times -infinity)
            above += (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(xi > xt));
        }
        if constexpr (TOP) {
            if (first) {  // the bound from the lanes' greatest
                uint64_t k = 0;
#pragma unroll
                for (int i = 0; i < LP_VALUES; ++i) {
                    const int id = V::index(at, i);
                    const uint64_t o = id < g.vocab ? lp_key(cur.at(i), id) : 0;
                    k = o > k ? o : k;
                }
                sort64(k);
                const uint64_t b = lane_key(k, g.top - 1);
                best.bound = b ? b - 1 : 0;  // (that one passes too)
                first = false;
            }
            const uint64_t sb = *(volatile unsigned long long*)&shared_bound;
            best.bound = sb > best.bound ? sb : best.bound;
            const float bv = lp_value((uint32_t)(best.bound >> 32));
            // (the bound below a first key may be its neighbour's in value: not above, but equal)
            if (__builtin_amdgcn_ballot_w64(!(mx < bv) || v.s != v.s) != 0) {
#pragma unroll
                for (int i = 0; i < LP_VALUES; ++i) {
                    const int id = V::index(at, i);
                    const uint64_t k = id < g.vocab ? lp_key(cur.at(i), id) : 0;
                    best.push(k, k > best.bound);
                }
                if (lane == 0) atomicMax(&shared_bound, (unsigned long long)best.bound);
            }
        }
        cur = nxt;
    }
    v = soft_of_lanes(v);
    if (lane == 0) sums[wave] = Part{v.m, v.s, v.e, above};
    if constexpr (TOP) {
        best.finish();
        buf[wave][lane] = best.list;
    }
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < LP_WAVES; ++w) {
        const Part o = sums[w];
        Soft ov;
        ov.m = o.m;
        ov.s = o.s;
        ov.e = o.e;
        v.add(ov);
        above += o.above;
        if constexpr (TOP) {
            const uint64_t rev = buf[w][63 - lane];
            best.list = rev > best.list ? rev : best.list;
            merge64(best.list);
        }
    }
    if (parts == 1) {
        lp_write(g, row, v, above, xt, t, best.list);
    } else {
        uint8_t* to = g.ws + ((uint64_t)row * parts + part) * part_bytes(g.top);
        if (lane == 0) *(Part*)to = Part{v.m, v.s, v.e, above};
        if (lane < g.top) ((uint64_t*)(to + sizeof(Part)))[lane] = best.list;
    }
}

// The parts of a row, by one wavefront.
template <int TY>
__global__ __launch_bounds__(64) void k_logprobs_join(LogprobArgs g, int parts) {
    const uint64_t row = blockIdx.x;
    const int lane = threadIdx.x;
    __shared__ uint64_t buf[128];
    const uint8_t* from = g.ws + row * parts * part_bytes(g.top);
    const int64_t t = lp_token(g, row);
    const float xt = t >= 0 && t < g.vocab ? lp_load<TY>((const uint8_t*)g.x + row * g.ldx * (TY == T_F32 ? 4 : 2), t) : 0.0f;
    Soft v;
    uint32_t above = 0;
    for (int p = lane; p < parts; p += 64) {
        const Part o = *(const Part*)(from + p * part_bytes(g.top));
        Soft ov;
        ov.m = o.m;
        ov.s = o.s;
        ov.e = o.e;
        v.add(ov);
        above += o.above;
    }
    v = soft_of_lanes(v);
    for (int d = 1; d < 64; d *= 2) above += __shfl_xor(above, d);
    Greatest best;
    best.buf = buf;
    best.top = g.top;
    if (g.top) {
        const int n = parts * g.top;
        auto key = [&](int i) -> uint64_t {
            return i < n ? ((const uint64_t*)(from + (uint64_t)(i / g.top) * part_bytes(g.top) + sizeof(Part)))[i % g.top] : 0;
        };
        uint64_t k = 0;
        for (int i = lane; i < n; i += 64) {
            const uint64_t o = key(i);
            k = o > k ? o : k;
        }
        sort64(k);
        const uint64_t b = lane_key(k, g.top - 1);
        best.bound = b ? b - 1 : 0;
        for (int i = 0; i < n; i += 64) {
            const uint64_t o = key(i + lane);
            best.push(o, o > best.bound);
        }
        best.finish();
    }
    lp_write(g, row, v, above, xt, t, best.list);
}

// Parts a row: enough workgroups to keep reads in flight on every CU, each of at least a step a wavefront.
static int lp_parts(int rows, int vocab) {
    const int steps = (vocab + LP_STEP - 1) / LP_STEP;
    const int most = (steps + LP_WAVES - 1) / LP_WAVES;
    int p = 512 / rows;
    p = p < most ? p : most;
    p = p < 64 ? p : 64;
    return p < 1 ? 1 : p;
}
static int lp_part_steps(int parts, int vocab) { return ((vocab + LP_STEP - 1) / LP_STEP + parts - 1) / parts; }

uint64_t logprob_ws_bytes(int rows, int vocab, int top) {
    if (rows == 0) return 0;
    const int p = lp_parts(rows, vocab);
    return p > 1 ? align_up((uint64_t)rows * p * part_bytes(top), 256) : 0;
}

template <int TY>
static void logprobs_as(const LogprobArgs& a, hipStream_t stream) {
    const int parts = lp_parts(a.rows, a.vocab), ps = lp_part_steps(parts, a.vocab);
    const dim3 grid((uint32_t)a.rows * (uint32_t)parts);
    if (a.top)
        hipLaunchKernelGGL((k_logprobs<TY, 1>), grid, dim3(64 * LP_WAVES), 0, stream, a, parts, ps);
    else
        hipLaunchKernelGGL((k_logprobs<TY, 0>), grid, dim3(64 * LP_WAVES), 0, stream, a, parts, ps);
    if (parts > 1) hipLaunchKernelGGL(k_logprobs_join<TY>, dim3(a.rows), dim3(64), 0, stream, a, parts);
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
