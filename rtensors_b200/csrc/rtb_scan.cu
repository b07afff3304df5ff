// Gated linear recurrence along one axis, f32 / f64:
//
//   h_s = a_s h_{s-1} + b_s        b = x, or (1 - a) x in the coupled form;   h_{-1} = h0 or 0
//
// and its gradient.  A step is the affine map h -> a h + b; maps compose associatively,
// (A2, B2) o (A1, B1) = (A2 A1, A2 B1 + B2), so the axis is cut into chunks whose maps are formed in
// parallel, and only the carry between chunks is sequential.  The backward pass is the same recurrence
// run the other way, g_s = dy_s + a_{s+1} g_{s+1}, with an epilogue (dx = g, da = g h_{s-1}), so one
// kernel body serves both: `s` below is always the PROCESSING index; the host folds the direction into
// signed strides.
//
// Every element is read once and written once.  A tile (chunk of the axis x lanes) stays in registers from its
// load to its store; in between the CTA learns the carry into its chunk.  Chunks of one lane group form a
// chain: a tile publishes its own map, waits until some predecessor within kWindow chunks has published its
// END STATE and the ones in between their maps, and folds those in axis order.  The fold from any end state
// gives the bits of the fold from the start, so results do not depend on timing.  Tiles are
// handed out by a ticket in chunk order: a tile only ever waits for tiles whose CTAs are already running.
// Waits are bounded; a wait that runs out makes the carry NaN.
//
// A product of gates that leaves the type's range inside one chunk (at most a few thousand steps) makes the
// carry's share inf or NaN where step-by-step evaluation might not; gates in [-1, 1] cannot.
#include <algorithm>
#include <vector>

#include "rtb_internal.h"
#include "rtb_ckpt8.cuh"

namespace rtb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kWindow = 32;              // predecessors a tile looks at, one flag per lane of a warp
constexpr int kMaxLaneDims = 6;
constexpr unsigned kSpinLimit = 1u << 22;  // polls of about a microsecond
constexpr size_t kWsHeader = 65536;        // completion counters in front of the workspace (rtb_context.cpp)
enum : unsigned { kFlagNone = 0, kFlagMap = 1, kFlagState = 2 };

__device__ __forceinline__ float fma_(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ double fma_(double a, double b, double c) { return fma(a, b, c); }
__device__ __forceinline__ float nan_of(float) { return __int_as_float(0x7fffffff); }
__device__ __forceinline__ double nan_of(double) { return __longlong_as_double(0x7fffffffffffffffll); }

template <typename T, int V> struct alignas(sizeof(T) * V) Pack {
    T e[V];
};
template <typename T, int V> __device__ __forceinline__ Pack<T, V> ld(const T *p) { return *reinterpret_cast<const Pack<T, V> *>(p); }
template <typename T, int V> __device__ __forceinline__ void st(T *p, const Pack<T, V> &v) { *reinterpret_cast<Pack<T, V> *>(p) = v; }
// published tile states are read past L1
template <typename T, int V> __device__ __forceinline__ Pack<T, V> ld_cg(const T *p) {
    Pack<T, V> v;
    if constexpr (sizeof(v) == 16) {
        uint4 q = __ldcg(reinterpret_cast<const uint4 *>(p));
        memcpy(&v, &q, 16);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v.e[j] = __ldcg(p + j);
    }
    return v;
}
__device__ __forceinline__ unsigned ld_acquire(const unsigned *p) {
    unsigned v;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ void st_release(unsigned *p, unsigned v) {
    asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}

// The dims other than the axis, merged as far as every operand allows, outermost first.  A lane is one
// sequence; its element s sits at base + s * step in each operand.
struct LaneDims {
    int nd;
    uint64_t n[kMaxLaneDims];
    int64_t so[kMaxLaneDims], sg[kMaxLaneDims], sb[kMaxLaneDims], sx[kMaxLaneDims];
};

template <typename T> struct ScanArgs {
    LaneDims dims;
    uint64_t lanes, steps;
    int64_t to, tg, tb, tx;  // signed steps along the axis in processing order (elements)
    int64_t o0;              // flat position of processing index 0 in the dense outputs
    const T *g;              // gate, at processing index 0
    const T *b;              // forward: x; backward: the upstream
    const T *x;              // backward, coupled: x
    const T *h0;             // dense over the lanes, or null
    const T *h;              // backward: dense states (flat)
    const int8_t *codes;     // or their 8-bit checkpoint
    const T *mags;
    T *out;                  // forward: h; backward: dx (may be null)
    T *dg;                   // backward: gradient of the gate, dense (may be null)
    T *dh0;                  // backward (may be null)
    // chunk chain (chunks > 1)
    uint64_t groups, chunks;
    unsigned long long *ticket;
    unsigned *flags;         // [group][chunk]
    T *maps;                 // [group][chunk][2][width]
    T *states;               // [group][chunk][width]
};

struct LaneAt {
    int64_t o, g, b, x;
};

__device__ __forceinline__ LaneAt locate(const LaneDims &d, uint64_t lane) {
    LaneAt at{0, 0, 0, 0};
    // 32-bit division wherever the index allows: the 64-bit one costs about a hundred instructions
#pragma unroll
    for (int k = kMaxLaneDims - 1; k >= 0; --k) {
        if (k >= d.nd) continue;
        uint64_t q, r;
        if (k == 0) {
            q = 0, r = lane;
        } else if (((lane | d.n[k]) >> 32) == 0) {
            q = (uint32_t)lane / (uint32_t)d.n[k];
            r = (uint32_t)lane - (uint32_t)q * (uint32_t)d.n[k];
        } else {
            q = lane / d.n[k], r = lane - q * d.n[k];
        }
        at.o += (int64_t)r * d.so[k];
        at.g += (int64_t)r * d.sg[k];
        at.b += (int64_t)r * d.sb[k];
        at.x += (int64_t)r * d.sx[k];
        lane = q;
    }
    return at;
}

// Warp-wide: publishes (A, H), the map of tile `chunk` of the chain, learns the state in front of it and
// publishes the state behind it.  `first` is the state in front of chunk 0.
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> chain_carry(const ScanArgs<T> &p, uint64_t group, uint64_t chunk, int lane, const Pack<T, V> &A,
                                                  const Pack<T, V> &H, const Pack<T, V> &first) {
    constexpr int W = 32 * V;
    const uint64_t at = group * p.chunks + chunk;
    const bool last = chunk + 1 == p.chunks;
    Pack<T, V> carry = first;
    if (chunk > 0) {
        if (!last) {
            st<T, V>(p.maps + (at * 2) * W + lane * V, A);
            st<T, V>(p.maps + (at * 2 + 1) * W + lane * V, H);
            __threadfence();
            __syncwarp();
            if (lane == 0) st_release(p.flags + at, kFlagMap);
        }
        // lane i watches predecessor chunk - 1 - i
        const bool mine = (uint64_t)lane < chunk;
        const unsigned *flag = p.flags + at - 1 - lane;
        unsigned seen = kFlagNone;
        int dist = -1;
        for (unsigned poll = 0; poll < kSpinLimit; ++poll) {
            if (mine && seen != kFlagState) seen = ld_acquire(flag);
            const unsigned st_mask = __ballot_sync(0xffffffffu, seen == kFlagState);
            const unsigned map_mask = __ballot_sync(0xffffffffu, seen != kFlagNone);
            if (st_mask) {
                const int d = __ffs(st_mask) - 1;                  // the nearest end state
                const unsigned nearer = d ? (1u << d) - 1u : 0u;
                if ((map_mask & nearer) == nearer) {
                    dist = d;
                    break;
                }
            }
        }
        __syncwarp();
        if (dist < 0) {
#pragma unroll
            for (int j = 0; j < V; ++j) carry.e[j] = nan_of(T());
        } else {
            const uint64_t from = at - 1 - dist;
            carry = ld_cg<T, V>(p.states + from * W + lane * V);
            // fold the maps in between in axis order, a batch of loads ahead of each batch of folds
            constexpr int kBatch = 4;
            for (int d = 0; d < dist; d += kBatch) {
                Pack<T, V> a[kBatch], h[kBatch];
#pragma unroll
                for (int k = 0; k < kBatch; ++k)
                    if (d + k < dist) {
                        a[k] = ld_cg<T, V>(p.maps + ((from + 1 + d + k) * 2) * W + lane * V);
                        h[k] = ld_cg<T, V>(p.maps + ((from + 1 + d + k) * 2 + 1) * W + lane * V);
                    }
#pragma unroll
                for (int k = 0; k < kBatch; ++k)
                    if (d + k < dist) {
#pragma unroll
                        for (int j = 0; j < V; ++j) carry.e[j] = fma_(a[k].e[j], carry.e[j], h[k].e[j]);
                    }
            }
        }
    }
    if (!last) {
        Pack<T, V> end;
#pragma unroll
        for (int j = 0; j < V; ++j) end.e[j] = fma_(A.e[j], carry.e[j], H.e[j]);
        st<T, V>(p.states + at * W + lane * V, end);
        __threadfence();
        __syncwarp();
        if (lane == 0) st_release(p.flags + at, kFlagState);
    }
    return carry;
}

__global__ void __launch_bounds__(kThreads) scan_clear_kernel(unsigned long long *ticket, unsigned *flags, size_t n) {
    grid_dep_sync();
    if (blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0;
    for (size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (size_t)gridDim.x * kThreads) flags[i] = kFlagNone;
}

// The tile this CTA works on; `slot` is shared memory.
template <typename T> __device__ __forceinline__ uint64_t take_tile(const ScanArgs<T> &p, unsigned long long *slot) {
    if (p.chunks == 1) return blockIdx.x;
    if (threadIdx.x == 0) *slot = atomicAdd(p.ticket, 1ull);
    __syncthreads();
    return *slot;
}

enum Mode { kForward = 0, kBackDense = 1, kBackCodes = 2 };

// A kept state, from the dense tensor or from its 8-bit checkpoint.
template <typename T, int V, int MODE> __device__ __forceinline__ Pack<T, V> kept(const ScanArgs<T> &p, int64_t flat) {
    if constexpr (MODE == kBackDense) return ld<T, V>(p.h + flat);
    Pack<T, V> v;
    if constexpr (MODE == kBackCodes) {
        const Pack<int8_t, V> c = ld<int8_t, V>(p.codes + flat);
        const Ckpt8Scale<T> scale(p.mags[flat >> kCkpt8Shift]);   // V divides the block: one magnitude
#pragma unroll
        for (int j = 0; j < V; ++j) v.e[j] = scale.restore(c.e[j]);
    }
    return v;
}

// ---- lanes contiguous in memory: a warp covers 32 * V lanes and R steps of the axis, a CTA kWarps * R steps ---------
// GVEC: the gate's lanes are contiguous too; otherwise the V lanes of a thread share one gate value (V = 1: any stride).
template <typename T, int V, int R, int MODE, bool COUPLED, bool GVEC>
__global__ void __launch_bounds__(kThreads) scan_lanes_kernel(const __grid_constant__ ScanArgs<T> p) {
    constexpr int W = 32 * V;
    __shared__ alignas(16) T sA[kWarps][W], sH[kWarps][W];
    __shared__ alignas(16) T sC[W];
    __shared__ unsigned long long slot;
    using P = Pack<T, V>;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    grid_dep_sync();
    const uint64_t tile = take_tile(p, &slot);
    const uint64_t chunk = p.chunks == 1 ? 0 : tile / p.groups, group = p.chunks == 1 ? tile : tile - chunk * p.groups;
    const uint64_t first_lane = group * W + (uint64_t)lane * V;
    const bool active = first_lane < p.lanes;
    const LaneAt at = locate(p.dims, active ? first_lane : 0);
    const int64_t s0 = (int64_t)(chunk * kWarps + warp) * R;
    const int64_t steps = (int64_t)p.steps;

    auto gate_at = [&](int64_t s) {
        P v;
        if constexpr (GVEC) return ld<T, V>(p.g + at.g + s * p.tg);
        const T one = p.g[at.g + s * p.tg];
#pragma unroll
        for (int j = 0; j < V; ++j) v.e[j] = one;
        return v;
    };
    P a[R], b[R], hp[MODE == kForward ? 1 : R], x[MODE != kForward && COUPLED ? R : 1], alast;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int64_t s = s0 + r;
#pragma unroll
        for (int j = 0; j < V; ++j) a[r].e[j] = (T)1, b[r].e[j] = (T)0;
        if (active && s < steps) {
            if constexpr (MODE == kForward) {
                a[r] = gate_at(s);
            } else if (s > 0) {
                a[r] = gate_at(s - 1);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) a[r].e[j] = (T)0;
            }
            b[r] = ld<T, V>(p.b + at.b + s * p.tb);
        }
    }
    if constexpr (MODE != kForward) {
#pragma unroll
        for (int j = 0; j < V; ++j) alast.e[j] = (T)0;
        if (active) {
            if (s0 + R - 1 < steps && (COUPLED || (p.dh0 && s0 + R == steps))) alast = gate_at(s0 + R - 1);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int64_t s = s0 + r;
                if (s >= steps) continue;
                if (p.dg) {
                    if (s + 1 < steps) {
                        hp[r] = kept<T, V, MODE>(p, p.o0 + at.o + (s + 1) * p.to);
                    } else {
#pragma unroll
                        for (int j = 0; j < V; ++j) hp[r].e[j] = p.h0 ? p.h0[first_lane + j] : (T)0;
                    }
                    if constexpr (COUPLED) x[r] = ld<T, V>(p.x + at.x + s * p.tx);
                }
            }
        }
    }
    if constexpr (MODE == kForward && COUPLED) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int j = 0; j < V; ++j) b[r].e[j] = ((T)1 - a[r].e[j]) * b[r].e[j];
    }
    // the thread's own map over its R steps
    P A = a[0], H = b[0];
#pragma unroll
    for (int r = 1; r < R; ++r)
#pragma unroll
        for (int j = 0; j < V; ++j) {
            A.e[j] = a[r].e[j] * A.e[j];
            H.e[j] = fma_(a[r].e[j], H.e[j], b[r].e[j]);
        }
    st<T, V>(&sA[warp][lane * V], A);
    st<T, V>(&sH[warp][lane * V], H);
    __syncthreads();
    if (warp == 0) {
        P first;
#pragma unroll
        for (int j = 0; j < V; ++j) first.e[j] = MODE == kForward && p.h0 && active ? p.h0[first_lane + j] : (T)0;
        if (p.chunks > 1) {
            for (int w = 1; w < kWarps; ++w) {
                const P wa = ld<T, V>(&sA[w][lane * V]), wh = ld<T, V>(&sH[w][lane * V]);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    A.e[j] = wa.e[j] * A.e[j];
                    H.e[j] = fma_(wa.e[j], H.e[j], wh.e[j]);
                }
            }
            first = chain_carry<T, V>(p, group, chunk, lane, A, H, first);
        }
        st<T, V>(&sC[lane * V], first);
    }
    __syncthreads();
    if (!active) return;
    P c = ld<T, V>(&sC[lane * V]);
    for (int w = 0; w < warp; ++w) {
        const P wa = ld<T, V>(&sA[w][lane * V]), wh = ld<T, V>(&sH[w][lane * V]);
#pragma unroll
        for (int j = 0; j < V; ++j) c.e[j] = fma_(wa.e[j], c.e[j], wh.e[j]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int64_t s = s0 + r;
        if (s >= steps) break;
#pragma unroll
        for (int j = 0; j < V; ++j) c.e[j] = fma_(a[r].e[j], c.e[j], b[r].e[j]);
        const int64_t o = p.o0 + at.o + s * p.to;
        if constexpr (MODE == kForward) {
            st<T, V>(p.out + o, c);
        } else {
            const P &now = r + 1 < R ? a[r + 1] : alast;   // the gate of step s
            if (p.out) {
                P d = c;
                if constexpr (COUPLED) {
                    // behind the last step of the axis a[r + 1] is the padding's 1, so alast's rule is applied here too
                    const P gate = (r + 1 < R && s + 1 == steps) ? gate_at(s) : now;
#pragma unroll
                    for (int j = 0; j < V; ++j) d.e[j] = ((T)1 - gate.e[j]) * c.e[j];
                }
                st<T, V>(p.out + o, d);
            }
            if (p.dg) {
                P d;
#pragma unroll
                for (int j = 0; j < V; ++j) d.e[j] = c.e[j] * (COUPLED ? hp[r].e[j] - x[COUPLED ? r : 0].e[j] : hp[r].e[j]);
                st<T, V>(p.dg + o, d);
            }
            if (p.dh0 && s + 1 == steps) {
                const P gate = r + 1 < R ? gate_at(s) : now;
#pragma unroll
                for (int j = 0; j < V; ++j) p.dh0[first_lane + j] = gate.e[j] * c.e[j];
            }
        }
    }
}

// ---- the axis itself contiguous: a warp covers runs of 32 * V consecutive steps of one lane -------------------------
// Within a run thread l holds V consecutive steps; their maps are scanned across the warp by shuffles.
// VEC: all operands have unit stride (either sign) along the axis and 16-byte aligned runs.
template <typename T> __device__ __forceinline__ T shfl_up(T v, int d) { return __shfl_up_sync(0xffffffffu, v, d); }
template <typename T> __device__ __forceinline__ T shfl_down1(T v) { return __shfl_down_sync(0xffffffffu, v, 1); }
template <typename T> __device__ __forceinline__ T shfl_at(T v, int l) { return __shfl_sync(0xffffffffu, v, l); }

template <typename T, int V, int K, int MODE, bool COUPLED, bool VEC> struct RowTile {
    using P = Pack<T, V>;
    P a[K], b[K], g[MODE == kForward ? 1 : K], hp[MODE == kForward ? 1 : K], x[MODE != kForward && COUPLED ? K : 1];
    T exA[K], exH[K];   // map of the steps of this tile in front of the thread's own
    T A, H;             // map of the whole tile (the same in all threads)

    // V steps from s on of an operand with signed step t
    static __device__ __forceinline__ P run(const T *base, int64_t s, int64_t t, int64_t steps, T pad) {
        P v;
        if (VEC) {   // steps is a multiple of V: whole runs only
            if (s < steps) {
                if (t > 0) return ld<T, V>(base + s);
                const P w = ld<T, V>(base - s - (V - 1));
#pragma unroll
                for (int j = 0; j < V; ++j) v.e[j] = w.e[V - 1 - j];
                return v;
            }
#pragma unroll
            for (int j = 0; j < V; ++j) v.e[j] = pad;
            return v;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) v.e[j] = s + j < steps ? base[(s + j) * t] : pad;
        return v;
    }
    static __device__ __forceinline__ void put(T *base, int64_t s, int64_t t, int64_t steps, const P &v) {
        if (VEC) {
            if (s >= steps) return;
            if (t > 0) {
                st<T, V>(base + s, v);
                return;
            }
            P w;
#pragma unroll
            for (int j = 0; j < V; ++j) w.e[j] = v.e[V - 1 - j];
            st<T, V>(base - s - (V - 1), w);
            return;
        }
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (s + j < steps) base[(s + j) * t] = v.e[j];
    }

    __device__ __forceinline__ void load(const ScanArgs<T> &p, const LaneAt &at, uint64_t lane_no, int64_t s0, int lane) {
        const int64_t steps = (int64_t)p.steps;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int64_t s = s0 + (int64_t)(k * 32 + lane) * V;
            const P gv = run(p.g + at.g, s, p.tg, steps, (T)1);
            b[k] = run(p.b + at.b, s, p.tb, steps, (T)0);
            if constexpr (MODE == kForward) {
                a[k] = gv;
            } else {
                g[k] = gv;
                T before = shfl_up(gv.e[V - 1], 1);   // the gate of the step in front of the run
                if (lane == 0) before = s > 0 && s - 1 < steps ? p.g[at.g + (s - 1) * p.tg] : (T)0;
                a[k].e[0] = before;
#pragma unroll
                for (int j = 1; j < V; ++j) a[k].e[j] = gv.e[j - 1];
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (s + j >= steps) a[k].e[j] = (T)1;
                if (p.dg) {
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const int64_t next = s + j + 1;
                        hp[k].e[j] = (T)0;
                        if (next < steps) hp[k].e[j] = kept<T, 1, MODE>(p, p.o0 + at.o + next * p.to).e[0];
                        else if (next == steps && p.h0) hp[k].e[j] = p.h0[lane_no];
                    }
                    if constexpr (COUPLED) x[k] = run(p.x + at.x, s, p.tx, steps, (T)0);
                }
            }
        }
    }
    __device__ __forceinline__ void compose(int lane) {
        A = (T)1, H = (T)0;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if constexpr (MODE == kForward && COUPLED) {
#pragma unroll
                for (int j = 0; j < V; ++j) b[k].e[j] = ((T)1 - a[k].e[j]) * b[k].e[j];
            }
            T la = a[k].e[0], lh = b[k].e[0];
#pragma unroll
            for (int j = 1; j < V; ++j) {
                la = a[k].e[j] * la;
                lh = fma_(a[k].e[j], lh, b[k].e[j]);
            }
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const T pa = shfl_up(la, d), ph = shfl_up(lh, d);
                if (lane >= d) {
                    lh = fma_(la, ph, lh);
                    la = la * pa;
                }
            }
            T ea = shfl_up(la, 1), eh = shfl_up(lh, 1);
            if (lane == 0) ea = (T)1, eh = (T)0;
            exA[k] = ea * A;
            exH[k] = fma_(ea, H, eh);
            const T ta = shfl_at(la, 31), th = shfl_at(lh, 31);
            H = fma_(ta, H, th);
            A = ta * A;
        }
    }
    __device__ __forceinline__ void finish(const ScanArgs<T> &p, const LaneAt &at, uint64_t lane_no, int64_t s0, int lane, T carry) {
        const int64_t steps = (int64_t)p.steps;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int64_t s = s0 + (int64_t)(k * 32 + lane) * V;
            T c = fma_(exA[k], carry, exH[k]);
            P h;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                c = fma_(a[k].e[j], c, b[k].e[j]);
                h.e[j] = c;
            }
            if constexpr (MODE == kForward) {
                put(p.out + p.o0 + at.o, s, p.to, steps, h);
            } else {
                if (p.out) {
                    P d = h;
                    if constexpr (COUPLED) {
#pragma unroll
                        for (int j = 0; j < V; ++j) d.e[j] = ((T)1 - g[k].e[j]) * h.e[j];
                    }
                    put(p.out + p.o0 + at.o, s, p.to, steps, d);
                }
                if (p.dg) {
                    P d;
#pragma unroll
                    for (int j = 0; j < V; ++j) d.e[j] = h.e[j] * (COUPLED ? hp[k].e[j] - x[COUPLED ? k : 0].e[j] : hp[k].e[j]);
                    put(p.dg + p.o0 + at.o, s, p.to, steps, d);
                }
                if (p.dh0) {
#pragma unroll
                    for (int j = 0; j < V; ++j)
                        if (s + j + 1 == steps) p.dh0[lane_no] = g[k].e[j] * h.e[j];
                }
            }
        }
    }
};

// One CTA per (lane, chunk of kWarps * K * 32 * V steps); chunks of a lane form a chain of width 32 (thread 0's slot counts).
template <typename T, int V, int K, int MODE, bool COUPLED, bool VEC>
__global__ void __launch_bounds__(kThreads) scan_axis_kernel(const __grid_constant__ ScanArgs<T> p) {
    __shared__ T sA[kWarps], sH[kWarps], sC;
    __shared__ unsigned long long slot;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    grid_dep_sync();
    const uint64_t tile = take_tile(p, &slot);
    const uint64_t chunk = p.chunks == 1 ? 0 : tile / p.groups, seq = p.chunks == 1 ? tile : tile - chunk * p.groups;
    const LaneAt at = locate(p.dims, seq);
    const int64_t s0 = (int64_t)(chunk * kWarps + warp) * (K * 32 * V);
    RowTile<T, V, K, MODE, COUPLED, VEC> t;
    t.load(p, at, seq, s0, lane);
    t.compose(lane);
    if (lane == 0) sA[warp] = t.A, sH[warp] = t.H;
    __syncthreads();
    if (warp == 0) {
        Pack<T, 1> A{{t.A}}, H{{t.H}}, first{{MODE == kForward && p.h0 ? p.h0[seq] : (T)0}};
        if (p.chunks > 1) {
            for (int w = 1; w < kWarps; ++w) {
                A.e[0] = sA[w] * A.e[0];
                H.e[0] = fma_(sA[w], H.e[0], sH[w]);
            }
            first = chain_carry<T, 1>(p, seq, chunk, lane, A, H, first);
        }
        if (lane == 0) sC = first.e[0];
    }
    __syncthreads();
    T c = sC;
    for (int w = 0; w < warp; ++w) c = fma_(sA[w], c, sH[w]);
    t.finish(p, at, seq, s0, lane, c);
}

// Many lanes: one warp walks its lane from end to end, the carry stays in a register.
template <typename T, int V, int K, int MODE, bool COUPLED, bool VEC>
__global__ void __launch_bounds__(kThreads) scan_axis_warp_kernel(const __grid_constant__ ScanArgs<T> p) {
    const int lane = threadIdx.x & 31;
    grid_dep_sync();
    const uint64_t seq = (uint64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (seq >= p.lanes) return;
    const LaneAt at = locate(p.dims, seq);
    T carry = MODE == kForward && p.h0 ? p.h0[seq] : (T)0;
    for (int64_t s0 = 0; s0 < (int64_t)p.steps; s0 += K * 32 * V) {
        RowTile<T, V, K, MODE, COUPLED, VEC> t;
        t.load(p, at, seq, s0, lane);
        t.compose(lane);
        t.finish(p, at, seq, s0, lane, carry);
        carry = fma_(t.A, carry, t.H);
    }
}

// ---- one step in place: state = a state + b over any view ------------------------------------------------
template <typename T, int V, bool COUPLED, bool GVEC>
__global__ void __launch_bounds__(kThreads) step_kernel(LaneDims dims, uint64_t lanes, T *state, const T *g, const T *x) {
    grid_dep_sync();
    const uint64_t i = ((uint64_t)blockIdx.x * kThreads + threadIdx.x) * V;
    if (i >= lanes) return;
    const LaneAt at = locate(dims, i);
    Pack<T, V> h = ld<T, V>(state + at.o), a, b = ld<T, V>(x + at.b);
    if constexpr (GVEC) {
        a = ld<T, V>(g + at.g);
    } else {
        const T one = g[at.g];
#pragma unroll
        for (int j = 0; j < V; ++j) a.e[j] = one;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) h.e[j] = fma_(a.e[j], h.e[j], COUPLED ? ((T)1 - a.e[j]) * b.e[j] : b.e[j]);
    st<T, V>(state + at.o, h);
}

// ---- host ------------------------------------------------------------------------------------------------
// Merges the dims of `shape` other than `axis` (axis >= rank: all of them).  -> false when more than kMaxLaneDims remain.
bool lane_dims(size_t rank, const size_t *shape, size_t axis, const ptrdiff_t *so, const ptrdiff_t *sg, const ptrdiff_t *sb,
               const ptrdiff_t *sx, LaneDims *out) {
    out->nd = 0;
    std::vector<uint64_t> n;
    std::vector<int64_t> s[4];
    const ptrdiff_t *in[4] = {so, sg, sb, sx};
    for (size_t k = 0; k < rank; ++k) {
        if (k == axis || shape[k] == 1) continue;
        bool merge = !n.empty();
        for (int q = 0; q < 4 && merge; ++q)
            if (in[q] && s[q].back() != (int64_t)in[q][k] * (int64_t)shape[k]) merge = false;
        if (merge) {
            n.back() *= shape[k];
            for (int q = 0; q < 4; ++q) s[q].back() = in[q] ? (int64_t)in[q][k] : 0;
        } else {
            n.push_back(shape[k]);
            for (int q = 0; q < 4; ++q) s[q].push_back(in[q] ? (int64_t)in[q][k] : 0);
        }
    }
    if (n.empty()) {
        n.push_back(1);
        for (int q = 0; q < 4; ++q) s[q].push_back(0);
    }
    if (n.size() > (size_t)kMaxLaneDims) return false;
    out->nd = (int)n.size();
    for (int k = 0; k < out->nd; ++k) {
        out->n[k] = n[k];
        out->so[k] = s[0][k], out->sg[k] = s[1][k], out->sb[k] = s[2][k], out->sx[k] = s[3][k];
    }
    return true;
}

template <typename T> bool aligned16(const T *p) { return ((uintptr_t)p & 15u) == 0; }

// every stride except the innermost lane's is a multiple of V elements
template <int V> bool strides_whole(const LaneDims &d, const int64_t *s, int64_t step) {
    if (step % V) return false;
    for (int k = 0; k + 1 < d.nd; ++k)
        if (s[k] % V) return false;
    return true;
}

template <typename T> int chain_workspace(Ctx *ctx, ScanArgs<T> *p, size_t width) {
    const size_t tiles = (size_t)(p->groups * p->chunks);
    const size_t flag_bytes = (tiles * sizeof(unsigned) + 255) & ~size_t(255);
    const size_t state_bytes = tiles * width * sizeof(T);
    void *ws = nullptr;
    int rc = workspace(ctx, 256 + flag_bytes + 3 * state_bytes, &ws);
    if (rc) return rc;
    char *at = (char *)ws + kWsHeader;
    p->ticket = (unsigned long long *)at;
    p->flags = (unsigned *)(at + 256);
    p->states = (T *)(at + 256 + flag_bytes);
    p->maps = (T *)(at + 256 + flag_bytes + state_bytes);
    const unsigned grid = (unsigned)std::min<size_t>((tiles + kThreads - 1) / kThreads, (size_t)ctx->sm_count);
    launch_dep(ctx, grid, kThreads, scan_clear_kernel, p->ticket, p->flags, tiles);
    return check_launch(ctx, "scan_clear_kernel");
}

constexpr uint64_t kMaxGrid = 0x7fffffffull;

template <typename T, int V, int R, int MODE, bool COUPLED, bool GVEC> int run_lanes(Ctx *ctx, ScanArgs<T> &p) {
    constexpr uint64_t W = 32 * V, S = (uint64_t)kWarps * R;
    p.groups = (p.lanes + W - 1) / W;
    p.chunks = (p.steps + S - 1) / S;
    if (p.groups > kMaxGrid / p.chunks) return fail(RTB_ERR_TOO_LARGE, "gated scan: %zu x %zu tiles are beyond one launch", (size_t)p.groups, (size_t)p.chunks);
    if (p.chunks > 1)
        if (int rc = chain_workspace(ctx, &p, W)) return rc;
    launch_dep(ctx, (unsigned)(p.groups * p.chunks), kThreads, scan_lanes_kernel<T, V, R, MODE, COUPLED, GVEC>, p);
    return check_launch(ctx, "scan_lanes_kernel");
}

template <typename T, int MODE, bool COUPLED> int pick_lanes(Ctx *ctx, ScanArgs<T> &p) {
    constexpr int V = 16 / sizeof(T);
    constexpr int R = MODE == kForward ? 8 : 4;
    const LaneDims &d = p.dims;
    const int in = d.nd - 1;
    const bool gvec = d.sg[in] == 1;
    // the V lanes of a thread are neighbours in every operand (or share the gate), at 16-byte aligned places
    bool vec = d.n[in] % V == 0 && d.so[in] == 1 && d.sb[in] == 1 && strides_whole<V>(d, d.so, p.to) && strides_whole<V>(d, d.sb, p.tb) &&
               aligned16(p.b) && p.o0 % V == 0 && (gvec || d.sg[in] == 0);
    if (gvec) vec = vec && strides_whole<V>(d, d.sg, p.tg) && aligned16(p.g);
    if (p.x) vec = vec && d.sx[in] == 1 && strides_whole<V>(d, d.sx, p.tx) && aligned16(p.x);
    for (const T *q : {(const T *)p.out, (const T *)p.dg, p.h}) vec = vec && aligned16(q);
    if (MODE == kBackCodes) vec = vec && aligned16((const T *)p.codes);
    if (vec && gvec) return run_lanes<T, V, R, MODE, COUPLED, true>(ctx, p);
    if (vec) return run_lanes<T, V, R, MODE, COUPLED, false>(ctx, p);
    return run_lanes<T, 1, 8, MODE, COUPLED, false>(ctx, p);
}

template <typename T, int MODE, bool COUPLED, bool VEC> int run_axis(Ctx *ctx, ScanArgs<T> &p) {
    constexpr int V = 16 / sizeof(T), K = 4;
    // A warp per lane streams well once a few thousand warps are there; fewer lanes are cut along the axis.
    constexpr uint64_t S = (uint64_t)kWarps * K * 32 * V;
    if (p.lanes >= (uint64_t)ctx->sm_count * 16 || p.steps <= K * 32 * V) {
        const uint64_t grid = (p.lanes + kWarps - 1) / kWarps;
        if (grid > kMaxGrid) return fail(RTB_ERR_TOO_LARGE, "gated scan: %zu sequences are beyond one launch", (size_t)p.lanes);
        p.groups = p.chunks = 1;
        launch_dep(ctx, (unsigned)grid, kThreads, scan_axis_warp_kernel<T, V, K, MODE, COUPLED, VEC>, p);
        return check_launch(ctx, "scan_axis_warp_kernel");
    }
    p.groups = p.lanes;
    p.chunks = (p.steps + S - 1) / S;
    if (p.groups > kMaxGrid / p.chunks) return fail(RTB_ERR_TOO_LARGE, "gated scan: %zu x %zu tiles are beyond one launch", (size_t)p.groups, (size_t)p.chunks);
    if (p.chunks > 1)
        if (int rc = chain_workspace(ctx, &p, 32)) return rc;
    launch_dep(ctx, (unsigned)(p.groups * p.chunks), kThreads, scan_axis_kernel<T, V, K, MODE, COUPLED, VEC>, p);
    return check_launch(ctx, "scan_axis_kernel");
}

template <typename T, int MODE, bool COUPLED> int pick_axis(Ctx *ctx, ScanArgs<T> &p) {
    constexpr int V = 16 / sizeof(T);
    auto unit = [](int64_t s) { return s == 1 || s == -1; };
    auto rows = [&](const int64_t *s) {
        for (int k = 0; k < p.dims.nd; ++k)
            if (s[k] % V) return false;
        return true;
    };
    // a reversed operand's pointer stands on its last element
    auto whole = [&](const T *q, int64_t s) { return aligned16(s > 0 ? q : q - (V - 1)); };
    bool vec = p.steps % V == 0 && unit(p.tg) && unit(p.tb) && unit(p.to) && rows(p.dims.sg) && rows(p.dims.sb) && rows(p.dims.so) &&
               whole(p.g, p.tg) && whole(p.b, p.tb);
    if (p.x) vec = vec && unit(p.tx) && rows(p.dims.sx) && whole(p.x, p.tx);
    for (const T *q : {(const T *)p.out, (const T *)p.dg}) vec = vec && aligned16(q);
    return vec ? run_axis<T, MODE, COUPLED, true>(ctx, p) : run_axis<T, MODE, COUPLED, false>(ctx, p);
}

template <typename T, int MODE> int pick(Ctx *ctx, ScanArgs<T> &p, bool along_axis, bool coupled) {
    if (along_axis) return coupled ? pick_axis<T, MODE, true>(ctx, p) : pick_axis<T, MODE, false>(ctx, p);
    return coupled ? pick_lanes<T, MODE, true>(ctx, p) : pick_lanes<T, MODE, false>(ctx, p);
}

// A temporary block of the context allocator, given back when the scope ends (stream order keeps it alive).
struct Temp {
    rtb_ctx *c;
    void *p = nullptr;
    explicit Temp(rtb_ctx *ctx) : c(ctx) {}
    ~Temp() {
        if (p) rtb_free(c, p);
    }
};

struct View {
    const void *p;
    const ptrdiff_t *strides;
    size_t offset;
};

// An operand is read in place when its lanes (or, along the axis, its steps) are neighbours in memory; a broadcast
// one as well.  Any other view (a transposed one, a negative step) is first copied row-major: one more
// pass, where reading it in place would fetch a 32-byte sector per element.
int in_place_or_copy(rtb_ctx *c, int dtype, size_t rank, const size_t *shape, size_t inner_dim, bool must_copy, size_t total,
                     const std::vector<ptrdiff_t> &dense, View *v, Temp *tmp) {
    const ptrdiff_t s = inner_dim < rank ? v->strides[inner_dim] : 1;
    if (!must_copy && (s == 0 || s == 1)) return RTB_OK;
    int rc = rtb_alloc(c, total * dtype_size(dtype), &tmp->p);
    if (rc) return rc;
    rc = rtb_copy_view(c, dtype, v->p, rank, shape, v->strides, v->offset, tmp->p);
    if (rc) return rc;
    v->p = tmp->p, v->strides = dense.data(), v->offset = 0;
    return RTB_OK;
}

int check_scan(rtb_ctx *c, int dtype, int flags, size_t rank, const size_t *shape, size_t axis) {
    if (!c) return fail(RTB_ERR_INVALID, "null ctx");
    if (dtype != RTB_F32 && dtype != RTB_F64) return fail(RTB_ERR_DTYPE, "the gated scan is defined for f32 and f64 only");
    if (flags & ~(RTB_SCAN_REVERSE | RTB_SCAN_COUPLED)) return fail(RTB_ERR_INVALID, "unknown scan flags %d", flags);
    if (rank > RTB_MAX_RANK) return fail(RTB_ERR_DIM, "rank %zu exceeds %d", rank, RTB_MAX_RANK);
    if (rank && !shape) return fail(RTB_ERR_INVALID, "null shape");
    if (axis >= rank) return fail(RTB_ERR_DIM, "axis %zu out of range for rank %zu", axis, rank);
    return RTB_OK;
}

struct ScanCall {
    bool back;
    View gate, b, x;
    const void *h0, *h, *codes, *mags;
    void *out, *dg, *dh0;
};

template <typename T> int run_scan(rtb_ctx *c, Ctx *ctx, int dtype, int flags, ScanCall call, size_t rank, const size_t *shape, size_t axis,
                                   size_t total) {
    std::vector<ptrdiff_t> dense(rank);
    rtb_meta_contiguous_strides(rank, shape, dense.data());
    const bool coupled = flags & RTB_SCAN_COUPLED, need_x = call.back && coupled && call.dg;
    // the innermost dim with more than one element decides: the axis itself, or a lane dim
    size_t inner = rank;
    for (size_t k = rank; k-- > 0;)
        if (shape[k] != 1) {
            inner = k;
            break;
        }
    const bool along_axis = inner >= rank || inner == axis;
    ScanArgs<T> p{};
    Temp tg(c), tb(c), tx(c);
    int rc;
    for (int pass = 0;; ++pass) {
        const bool copy = pass == 1;   // too many lane dims: dense copies have two at most
        if ((rc = in_place_or_copy(c, dtype, rank, shape, inner, copy && !tg.p, total, dense, &call.gate, &tg))) return rc;
        if ((rc = in_place_or_copy(c, dtype, rank, shape, inner, copy && !tb.p, total, dense, &call.b, &tb))) return rc;
        if (need_x && (rc = in_place_or_copy(c, dtype, rank, shape, inner, copy && !tx.p, total, dense, &call.x, &tx))) return rc;
        if (lane_dims(rank, shape, axis, dense.data(), call.gate.strides, call.b.strides, need_x ? call.x.strides : nullptr, &p.dims)) break;
    }
    const int64_t steps = (int64_t)shape[axis];
    const bool down = ((flags & RTB_SCAN_REVERSE) != 0) != call.back;   // processing order runs towards lower indices
    auto place = [&](const View &v, int64_t *step) {
        const int64_t s = (int64_t)v.strides[axis];
        *step = down ? -s : s;
        return (const T *)v.p + (int64_t)v.offset + (down ? (steps - 1) * s : 0);
    };
    p.steps = (uint64_t)steps;
    p.lanes = total / shape[axis];
    p.g = place(call.gate, &p.tg);
    p.b = place(call.b, &p.tb);
    if (need_x) p.x = place(call.x, &p.tx);
    p.to = down ? -(int64_t)dense[axis] : (int64_t)dense[axis];
    p.o0 = down ? (steps - 1) * (int64_t)dense[axis] : 0;
    p.h0 = (const T *)call.h0, p.h = (const T *)call.h;
    p.codes = (const int8_t *)call.codes, p.mags = (const T *)call.mags;
    p.out = (T *)call.out, p.dg = (T *)call.dg, p.dh0 = (T *)call.dh0;
    std::lock_guard<std::mutex> lock(ctx->ws_mu);
    if (!call.back) return pick<T, kForward>(ctx, p, along_axis, coupled);
    if (call.codes) return pick<T, kBackCodes>(ctx, p, along_axis, coupled);
    return pick<T, kBackDense>(ctx, p, along_axis, coupled);
}

template <typename T, bool COUPLED> int run_step(Ctx *ctx, const LaneDims &d, uint64_t lanes, T *state, const T *g, const T *x) {
    constexpr int V = 16 / sizeof(T);
    const int in = d.nd - 1;
    const bool gvec = d.sg[in] == 1;
    bool vec = d.n[in] % V == 0 && d.so[in] == 1 && d.sb[in] == 1 && (gvec || d.sg[in] == 0) && strides_whole<V>(d, d.so, 0) &&
               strides_whole<V>(d, d.sb, 0) && aligned16(state) && aligned16(x);
    if (gvec) vec = vec && strides_whole<V>(d, d.sg, 0) && aligned16(g);
    const uint64_t per = (uint64_t)kThreads * (vec ? V : 1), grid = (lanes + per - 1) / per;
    if (grid > kMaxGrid) return fail(RTB_ERR_TOO_LARGE, "gated step: %zu elements are beyond one launch", (size_t)lanes);
    if (vec && gvec) launch_dep(ctx, (unsigned)grid, kThreads, step_kernel<T, V, COUPLED, true>, d, lanes, state, g, x);
    else if (vec) launch_dep(ctx, (unsigned)grid, kThreads, step_kernel<T, V, COUPLED, false>, d, lanes, state, g, x);
    else launch_dep(ctx, (unsigned)grid, kThreads, step_kernel<T, 1, COUPLED, false>, d, lanes, state, g, x);
    return check_launch(ctx, "step_kernel");
}

template <typename T> int step_any(Ctx *ctx, int flags, T *state, const ptrdiff_t *ss, const T *g, const ptrdiff_t *sg, const T *x,
                                   const ptrdiff_t *sx, size_t rank, const size_t *shape) {
    LaneDims d;
    uint64_t lanes = 1;
    for (size_t k = 0; k < rank; ++k) lanes *= shape[k];
    if (lane_dims(rank, shape, rank, ss, sg, sx, nullptr, &d))
        return flags & RTB_SCAN_COUPLED ? run_step<T, true>(ctx, d, lanes, state, g, x) : run_step<T, false>(ctx, d, lanes, state, g, x);
    // more dims than one launch takes: peel the outermost one that has extent
    size_t k0 = 0;
    while (shape[k0] == 1) ++k0;
    for (size_t i = 0; i < shape[k0]; ++i) {
        const ptrdiff_t k = (ptrdiff_t)i;
        int rc = step_any<T>(ctx, flags, state + k * ss[k0], ss + k0 + 1, g + k * sg[k0], sg + k0 + 1, x + k * sx[k0], sx + k0 + 1,
                             rank - k0 - 1, shape + k0 + 1);
        if (rc) return rc;
    }
    return RTB_OK;
}

}  // namespace
}  // namespace rtb

using namespace rtb;

static inline Ctx *C(rtb_ctx *c) { return reinterpret_cast<Ctx *>(c); }

static size_t count_of(size_t rank, const size_t *shape) {
    size_t n = 1;
    for (size_t k = 0; k < rank; ++k) n *= shape[k];
    return n;
}

RTB_API int rtb_gated_scan(rtb_ctx *c, int dtype, int flags, const void *gate, const ptrdiff_t *stride_g, size_t off_g, const void *x,
                           const ptrdiff_t *stride_x, size_t off_x, const void *h0, void *h, size_t rank, const size_t *shape, size_t axis) {
    int rc = check_scan(c, dtype, flags, rank, shape, axis);
    if (rc) return rc;
    const size_t total = count_of(rank, shape);
    if (total == 0) return RTB_OK;
    if (!gate || !x || !h || !stride_g || !stride_x) return fail(RTB_ERR_INVALID, "null argument");
    Ctx *ctx = C(c);
    if ((rc = use_device(ctx))) return rc;
    ScanCall call{};
    call.gate = View{gate, stride_g, off_g};
    call.b = View{x, stride_x, off_x};
    call.h0 = h0, call.out = h;
    return dtype == RTB_F32 ? run_scan<float>(c, ctx, dtype, flags, call, rank, shape, axis, total)
                            : run_scan<double>(c, ctx, dtype, flags, call, rank, shape, axis, total);
}

RTB_API int rtb_gated_scan_backward(rtb_ctx *c, int dtype, int flags, const void *up, const ptrdiff_t *stride_u, size_t off_u,
                                    const void *gate, const ptrdiff_t *stride_g, size_t off_g, const void *x, const ptrdiff_t *stride_x,
                                    size_t off_x, const void *h, const int8_t *codes, const void *mags, const void *h0, void *d_x,
                                    void *d_gate, void *d_h0, size_t rank, const size_t *shape, size_t axis) {
    int rc = check_scan(c, dtype, flags, rank, shape, axis);
    if (rc) return rc;
    const size_t total = count_of(rank, shape), es = dtype_size(dtype);
    Ctx *ctx = C(c);
    if (!stride_g) return fail(RTB_ERR_INVALID, "null argument");
    bool shared = false;   // the gate is broadcast along some dim: its gradient is summed over it
    size_t gate_n = 1;
    for (size_t k = 0; k < rank; ++k) {
        if (stride_g[k] == 0 && shape[k] != 1) shared = true;
        else gate_n *= shape[k];
    }
    if (total == 0) {
        // no step and no upstream: what is left of the gradients is zero
        if ((rc = use_device(ctx))) return rc;
        size_t lanes = 1;
        for (size_t k = 0; k < rank; ++k)
            if (k != axis) lanes *= shape[k];
        if (d_h0 && lanes) RTB_CUDA(cudaMemsetAsync(d_h0, 0, lanes * es, ctx->stream));
        if (d_gate && gate_n) RTB_CUDA(cudaMemsetAsync(d_gate, 0, gate_n * es, ctx->stream));
        return RTB_OK;
    }
    if (!up || !gate || !stride_u) return fail(RTB_ERR_INVALID, "null argument");
    if (d_gate && !h && (!codes || !mags)) return fail(RTB_ERR_INVALID, "the gate's gradient needs the states or their checkpoint");
    if (h && codes) return fail(RTB_ERR_INVALID, "states and a checkpoint of them at once");
    if (d_gate && (flags & RTB_SCAN_COUPLED) && (!x || !stride_x)) return fail(RTB_ERR_INVALID, "the coupled gate's gradient needs x");
    if (!d_x && !d_gate && !d_h0) return RTB_OK;
    if ((rc = use_device(ctx))) return rc;
    ScanCall call{};
    call.back = true;
    call.gate = View{gate, stride_g, off_g};
    call.b = View{up, stride_u, off_u};
    call.x = View{x, stride_x, off_x};
    call.h0 = h0, call.h = h, call.codes = codes, call.mags = mags;
    call.out = d_x, call.dg = d_gate, call.dh0 = d_h0;
    Temp full(c);
    if (shared && d_gate) {
        if ((rc = rtb_alloc(c, total * es, &full.p))) return rc;
        call.dg = full.p;
    }
    rc = dtype == RTB_F32 ? run_scan<float>(c, ctx, dtype, flags, call, rank, shape, axis, total)
                          : run_scan<double>(c, ctx, dtype, flags, call, rank, shape, axis, total);
    if (rc || !full.p) return rc;
    std::vector<size_t> out_shape(rank);
    return rtb_reduce_to_shape(c, dtype, full.p, rank, shape, stride_g, d_gate, out_shape.data());
}

RTB_API int rtb_gated_step(rtb_ctx *c, int dtype, int flags, void *state, const ptrdiff_t *stride_s, size_t off_s, const void *gate,
                           const ptrdiff_t *stride_g, size_t off_g, const void *x, const ptrdiff_t *stride_x, size_t off_x, size_t rank,
                           const size_t *shape) {
    if (!c) return fail(RTB_ERR_INVALID, "null ctx");
    if (dtype != RTB_F32 && dtype != RTB_F64) return fail(RTB_ERR_DTYPE, "the gated step is defined for f32 and f64 only");
    if (flags & ~RTB_SCAN_COUPLED) return fail(RTB_ERR_INVALID, "unknown step flags %d", flags);
    if (rank > RTB_MAX_RANK) return fail(RTB_ERR_DIM, "rank %zu exceeds %d", rank, RTB_MAX_RANK);
    if (rank && (!shape || !stride_s || !stride_g || !stride_x)) return fail(RTB_ERR_INVALID, "null shape or strides");
    if (count_of(rank, shape) == 0) return RTB_OK;
    if (!state || !gate || !x) return fail(RTB_ERR_INVALID, "null argument");
    for (size_t k = 0; k < rank; ++k)
        if (stride_s[k] == 0 && shape[k] != 1) return fail(RTB_ERR_SHAPE, "the state's dim %zu is broadcast: it cannot be written", k);
    Ctx *ctx = C(c);
    if (int rc = use_device(ctx)) return rc;
    if (dtype == RTB_F32)
        return step_any<float>(ctx, flags, (float *)state + off_s, stride_s, (const float *)gate + off_g, stride_g, (const float *)x + off_x,
                               stride_x, rank, shape);
    return step_any<double>(ctx, flags, (double *)state + off_s, stride_s, (const double *)gate + off_g, stride_g, (const double *)x + off_x,
                            stride_x, rank, shape);
}
