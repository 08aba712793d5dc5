// policy_ops.hip - the C-ABI host side of include/lobpolicy.h and the kernels (gfx950) but for those over segments (policy_scan.hip).
#include "policy_common.h"

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <type_traits>

namespace lobpolicy {

thread_local char g_error[256] = "";

int fail(int code, const char* format, ...) {
    va_list args;
    va_start(args, format);
    vsnprintf(g_error, sizeof g_error, format, args);
    va_end(args);
    return code;
}

template <class T>
int scan_typed(const Walks& w, bool swapped, hipStream_t stream) {
    const int da = w.walk[0].da;
    if (da <= 32) return scan_rows<T, 32>(w, swapped, stream);
    if (da <= 64) return scan_rows<T, 64>(w, swapped, stream);
    return scan_rows<T, 128>(w, swapped, stream);
}

// Few environments and heads, many steps: the steps are split into parts.  A first walk finds what each part adds to the state, join_parts
// turns that into the state in front of each part, a second walk starts from it.  That reads k and v twice, so it pays where the chip is
// otherwise far from full, and then only until it is full: as many parts as fit, not one more (100 units of 128 to 128 in 5 parts 239 us, in 6, of which
// the last 88 workgroups run by themselves, 299).  Whole : split, us in a graph, forwards and with the gradients:
//     32 to 32, bf16:   4096 steps, 32 units 233 : 30, 256 units 236 : 119, 384 units 267 : 227 and 597 : 621;  512 steps, 192 units 35 : 28 and 76 : 63
//     64 to 64, bf16:   4096 steps, 75 units 275 : 82 and 553 : 238, 192 units 278 : 177 and 649 : 529, 220 units 279 : 215 and 653 : 592;  1024 steps, 192 units 77 : 59 and
//                       181 : 170, 220 units 78 : 67 and 185 : 190;  640 steps, 150 units 51 : 41 and 110 : 108, 190 units 51 : 46 and 121 : 129;  512 steps, 128 units 42 : 34 and 90 : 85,
//                       150 units 41 : 37 and 91 : 98
//     64 to 64, f32:    4096 steps, 192 units 388 : 350 and 1153 : 1028, 220 units 397 : 405 and 1166 : 1179;  512 steps, 128 units 56 : 48 and 138 : 130, 150 units 56 : 57 and 138 : 155
//     107 to 53, bf16:  768 steps, 150 units 91 : 71 and 206 : 196, 190 units 93 : 93 and 233 : 248;  640 steps, 128 units 78 : 60 and 174 : 162, 150 units 79 : 71 and 175 : 192
//     128 to 128, bf16: 4096 steps, 75 units 476 : 192 and 946 : 577, 150 units 486 : 347 and 1102 : 1069, 192 units 493 : 460 and 1497 : 1386;  1024 steps, 128 units 121 : 98 and
//                       280 : 302, 150 units 122 : 119 and 286 : 369;  768 steps, 104 units 93 : 74 and 215 : 220, 128 units 94 : 81 and 218 : 253;  512 steps, 75 units 64 : 56 and 134 : 147,
//                       100 units 65 : 60 and 153 : 173
//     128 to 128, f32:  4096 steps, 150 units 972 : 803 and 2558 : 2666, 192 units 984 : 1140 and 3457 : 3485;  768 steps, 128 units 176 : 150 and 484 : 462, 150 units 181 : 187 and 493 : 565
// 512 : 1024 workgroups in all, the latter where they are small: 4096 steps, 128 units of 64 to 64 (bf16) 139 : 124 and 380 : 368, 256 units of 32 to 32 200 : 120, 128 units of
// 128 to 128 292 : 310 and 837 : 915.  Below 512 steps the two further launches take what the parts save (256 steps of 64 to 64, 32 units: 22.2 : 23.0; 512 steps: 39.0 : 25.3).
struct Parts {
    int64_t steps;
    int count;
    Parts(const lobpolicy_attention* a) {
        const int widest = a->dk > a->dv ? a->dk : a->dv, narrowest = a->dk > a->dv ? a->dv : a->dk;
        const int64_t units = a->envs * a->heads, wanted = widest <= 64 ? 1024 : 512;
        int64_t most = 384;  // units
        if (narrowest > 64)
            most = a->steps < 1344 ? 48 + a->steps / 12 : 160;
        else if (widest > 32)
            most = (widest <= 64 ? 208 : 160) * (a->steps < 768 ? a->steps : 768) / 768;
        int64_t n = a->steps < 512 || units >= most ? 1 : wanted / units;
        n = n < ceil_div(a->steps, 128) ? n : ceil_div(a->steps, 128);
        steps = ceil_div(ceil_div(a->steps, n), 64) * 64;
        count = (int)ceil_div(a->steps, steps);
    }
    int64_t matrices(const lobpolicy_attention* a) const { return a->envs * a->heads * count; }
    int64_t bytes(const lobpolicy_attention* a) const { return count == 1 ? 0 : matrices(a) * (a->dk * a->dv + 1) * (int64_t)sizeof(float); }
};

// grid (elements / 256, units): `states` [unit][part] from what each part adds to what is in front of it; the state behind the last to state_out.
// Each element is a chain of its own over the parts, bound by the latency of its loads: 10 us for 8 units of 64 x 64 in 94 parts (30 us with each part's
// load behind the one before), 19 us for 128 units of 128 x 128 in 4 (67 MB there and back).
__global__ __launch_bounds__(256) void join_parts(Scan s, float* states, const float* __restrict__ carries) {
    const int64_t unit = blockIdx.y, matrix = (int64_t)s.da * s.dc, e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (e >= matrix) return;
    const int64_t row = e / s.dc, col = e % s.dc;
    float state = s.state_in ? s.state_in[unit * matrix + row * s.in_row + col * s.in_col] : 0.f;
    const float* carry = carries + unit * s.parts;
    // buffer instructions: what lies behind the last part reads as 0 and is not written, without a branch that would wait for the loads in flight.
    // AT_ONCE parts at a time, the next ones on their way before these are stored (a wait for a load waits for the stores in front of it too)
    constexpr int AT_ONCE = 8;
    const __amdgpu_buffer_rsrc_t buffer = __builtin_amdgcn_make_buffer_rsrc(states + unit * s.parts * matrix, 0, (int)(s.parts * matrix * 4), 0x27000);
    const int at = (int)e * 4, step = (int)matrix * 4;
    float added[AT_ONCE], next[AT_ONCE];
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) next[k] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(buffer, at + k * step, 0, 0));
    for (int first = 0; first < s.parts; first += AT_ONCE) {
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            added[k] = next[k];
            next[k] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(buffer, at + (first + AT_ONCE + k) * step, 0, 0));
        }
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            const int part = first + k;
            const float c = part < s.parts ? carry[part] : 1.f;
            __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, state), buffer, at + part * step, 0, 0);
            state = (c < 0.f ? 0.f : state * c) + added[k];
        }
    }
    if (s.state_out) {
        const int64_t n = unit / s.heads;
        if (s.reverse && length_of(s, n) > 0) state = s.reset && s.reset[n * s.reset_sn] ? 0.f : state * expf(s.log_decay[unit % s.heads]);
        s.state_out[unit * matrix + row * s.out_row + col * s.out_col] = state;
    }
}

int walk(const lobpolicy_attention* a, const Walks& w, bool swapped, hipStream_t stream) {
    return a->dtype == LOBPOLICY_BF16 ? scan_typed<bf16>(w, swapped, stream) : scan_typed<float>(w, swapped, stream);
}

// the states in front of each part of a walk with da = dk and dc = dv, to the workspace; s.state_out
int part_states(const lobpolicy_attention* a, const Scan& s, hipStream_t stream) {
    const Parts parts(a);
    float* states = (float*)a->workspace;
    float* carries = states + parts.matrices(a) * a->dk * a->dv;
    Walks first = {{s}, 1};
    Scan& w = first.walk[0];
    w.a = w.b, w.out = {};
    w.state_in = nullptr, w.state_out = states, w.carry_out = carries;
    if (int e = walk(a, first, false, stream)) return e;
    join_parts<<<dim3((unsigned)ceil_div((int64_t)s.da * s.dc, 256), (unsigned)(a->envs * a->heads)), 256, 0, stream>>>(s, states, carries);
    return launched();
}

int check_workspace(const lobpolicy_attention* a) {
    const int64_t need = Parts(a).bytes(a);
    REQUIRE(need == 0 || (a->workspace && aligned(a->workspace, 16) && a->workspace_bytes >= need), "the workspace has %lld bytes, %lld are needed", (long long)a->workspace_bytes, (long long)need);
    return LOBPOLICY_OK;
}

int check_attention(const lobpolicy_attention* a) {
    REQUIRE(a, "no description");
    REQUIRE(a->dtype == LOBPOLICY_F32 || a->dtype == LOBPOLICY_BF16, "dtype %d", a->dtype);
    REQUIRE(a->heads >= 1 && a->heads <= 65536, "heads = %d", a->heads);
    REQUIRE(a->dk >= 1 && a->dk <= LOBPOLICY_MAX_HEAD && a->dv >= 1 && a->dv <= LOBPOLICY_MAX_HEAD, "dk = %d, dv = %d: 1 to %d", a->dk, a->dv, LOBPOLICY_MAX_HEAD);
    REQUIRE(a->steps >= 1 && a->envs >= 1, "steps and envs are 1 or more");
    REQUIRE(a->steps < (1ll << 31), "steps: at most 2^31 - 1");
    REQUIRE(a->envs <= (1ll << 22) / a->heads, "envs x heads: at most 2^22");
    REQUIRE(a->log_decay, "no log_decay");
    return LOBPOLICY_OK;
}

Rows rows_of(const lobpolicy_operand& o) { return {o.data, o.stride_t, o.stride_n, o.stride_h}; }

Scan scan_of(const lobpolicy_attention* a) {
    Scan s = {};
    s.log_decay = a->log_decay;
    s.reset = a->reset;
    s.reset_st = a->reset_stride_t;
    s.reset_sn = a->reset_stride_n;
    s.lengths = a->lengths;
    s.steps = a->steps;
    s.envs = a->envs;
    s.heads = a->heads;
    s.in_scale = s.out_scale = 1.f;
    const Parts parts(a);
    s.parts = parts.count, s.part_steps = parts.steps;
    return s;
}

// ---------------------------------------------------------------------------------------------------------------------------
// decay attention, one token of every environment
//
// Reads and writes the state once: 8 dk dv bytes per environment and head, next to which the operands are nothing.  One workgroup per
// environment and head; a thread holds VW neighbouring columns of every RG-th row, so that a wave moves whole rows.  Bound by memory: 4096
// environments of 8 heads of 64 x 64 take 189 us (1.09 GB, 5.8 TB/s), 64 of 4 take 4.3 us, a launch's time.  The sum over the rows is in 32 bits, in
// a fixed order: a group's rows, then the groups.

struct Step {
    const void *q, *k, *v;
    void* out;
    int64_t q_sn, q_sh, k_sn, k_sh, v_sn, v_sh, out_sn, out_sh;
    const float* log_decay;
    const uint8_t *reset, *skip;
    int64_t reset_sn;
    float* state;
    int heads, dk, dv;
    float scale;
};

// Rows of whole packs of 4 from a multiple of 16 bytes on, or elements: 61 x 59 of 4096 environments and 4 heads takes 75 us (6.3 TB/s) an element at a
// time, 93 us in packs that begin anywhere.  A thread loads AT_ONCE rows before it stores one: a load behind a store waits for it, as far as the
// compiler knows (100 x 101: 282 us, a row at a time 346).
template <class T, int VW, int LPR, int THREADS>
__global__ __launch_bounds__(THREADS) void step_kernel(Step s) {
    constexpr int RG = THREADS / LPR, AT_ONCE = VW == 1 ? 8 : 4;
    __shared__ float part[RG][LPR * VW];
    const int64_t unit = blockIdx.x, n = unit / s.heads;
    const int h = (int)(unit % s.heads), col = (threadIdx.x % LPR) * VW, group = threadIdx.x / LPR;
    const bool mine = col < s.dv;
    T* out = (T*)s.out + n * s.out_sn + h * s.out_sh;
    if (s.skip && s.skip[n]) {
        if (mine && group == 0)
            for (int i = 0; i < VW; ++i) out[col + i] = (T)0.f;
        return;
    }
    const T* q = (const T*)s.q + n * s.q_sn + h * s.q_sh;
    const T* k = (const T*)s.k + n * s.k_sn + h * s.k_sh;
    const T* v = (const T*)s.v + n * s.v_sn + h * s.v_sh;
    typedef Pack<float, VW> P;
    float* state = s.state + unit * s.dk * s.dv + col;
    const bool fresh = s.reset && s.reset[n * s.reset_sn];
    const float decay = expf(s.log_decay[h]);
    float value[VW], sum[VW];
#pragma unroll
    for (int i = 0; i < VW; ++i) value[i] = mine ? (float)v[col + i] : 0.f, sum[i] = 0.f;
    if (mine)
        for (int first = group; first < s.dk; first += AT_ONCE * RG) {  // (rows behind the last are loaded as the last, and not used)
            P x[AT_ONCE];
            float key[AT_ONCE], query[AT_ONCE];
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                const int row = min(first + u * RG, s.dk - 1);
                key[u] = (float)k[row], query[u] = (float)q[row];
                if (fresh)
                    x[u] = P{};
                else
                    x[u] = *reinterpret_cast<const P*>(state + row * s.dv);
            }
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                const int row = first + u * RG;
                if (row >= s.dk) break;
#pragma unroll
                for (int i = 0; i < VW; ++i) {
                    x[u].v[i] = x[u].v[i] * decay + key[u] * value[i];
                    sum[i] += query[u] * x[u].v[i];
                }
                *reinterpret_cast<P*>(state + row * s.dv) = x[u];
            }
        }
#pragma unroll
    for (int i = 0; i < VW; ++i) part[group][(threadIdx.x % LPR) * VW + i] = sum[i];
    __syncthreads();
    for (int c = threadIdx.x; c < s.dv; c += THREADS) {
        float total = 0.f;
        for (int g = 0; g < RG; ++g) total += part[g][c];
        out[c] = (T)(total * s.scale);
    }
}

// elements of a state that one wave works on, rather than four: 16384 states of 16 x 16 10.9 and 21.7 us, 32 x 32 23 and 32, 48 x 48 48 both, 64 x 64 87 and 83
constexpr int STEP_SMALL = 1024;

template <class T, int VW, int LPR>
int step_launch(const Step& s, int64_t units, hipStream_t stream) {
    if (s.dk * s.dv <= STEP_SMALL)
        step_kernel<T, VW, LPR, 64><<<dim3((unsigned)units), 64, 0, stream>>>(s);
    else
        step_kernel<T, VW, LPR, 256><<<dim3((unsigned)units), 256, 0, stream>>>(s);
    return launched();
}

template <class T>
int step_typed(const Step& s, int64_t units, hipStream_t stream) {
    if (s.dv % 4 == 0 && aligned(s.state, 16)) {
        if (s.dv <= 32) return step_launch<T, 4, 8>(s, units, stream);
        if (s.dv <= 64) return step_launch<T, 4, 16>(s, units, stream);
        return step_launch<T, 4, 32>(s, units, stream);
    }
    if (s.dv <= 8) return step_launch<T, 1, 8>(s, units, stream);
    if (s.dv <= 32) return step_launch<T, 1, 32>(s, units, stream);
    if (s.dv <= 64) return step_launch<T, 1, 64>(s, units, stream);
    step_kernel<T, 1, 128, 256><<<dim3((unsigned)units), 256, 0, stream>>>(s);
    return launched();
}

// ---------------------------------------------------------------------------------------------------------------------------
// the block's end
//
// Bound by memory: every operand is read once and every result written once.  A row lives in the registers of one wave (width up to 1024)
// or of one workgroup, VW neighbouring elements per thread and step, E elements per thread in all; the sums are 32-bit.  65536 rows of 1024 (bf16):
// 155 us forwards (671 MB, 4.3 TB/s; 64 M elements), 219 us backwards (1.07 GB, 4.9 TB/s), 7 us the weights' gradients; 64 rows of 256: 4 us.

struct Block {
    const void *x, *block, *gate, *grad_y, *grad_z;
    int64_t x_sr, block_sr, gate_sr, grad_y_sr, grad_z_sr;
    const float *post, *res, *pre;
    void *y, *z, *grad_x, *grad_block, *grad_gate;
    float* partial;  // [2][gridDim.x][width]
    int* parts;      // host: gridDim.x of the launch
    int64_t rows;
    int width;
    float eps;
};

template <int TPR>
__device__ __forceinline__ void row_sums(float* v, int count, float* shared) {
    for (int i = 0; i < count; ++i) v[i] = wave_sum(v[i]);
    if (TPR > 64) {
        __syncthreads();
        if (threadIdx.x % 64 == 0)
            for (int i = 0; i < count; ++i) shared[(threadIdx.x / 64) * 2 + i] = v[i];
        __syncthreads();
        for (int i = 0; i < count; ++i) {
            v[i] = 0.f;
#pragma unroll
            for (int k = 0; k < TPR / 64; ++k) v[i] += shared[2 * k + i];
        }
    }
}

// A row's elements of one thread.  RAG: rows begin anywhere and are no whole number of packs; the last pack is loaded as the row's last VW elements and
// shifted, without a branch (which would wait for what is on its way).  Where the row has no element, 0.
template <class T, int VW, bool RAG>
__device__ __forceinline__ Pack<T, VW> load_some(const T* row, int width, int col) {
    if constexpr (RAG) {
        const int from = col < width - VW ? col : width - VW;
        return shifted(load_anywhere<T, VW>(row + from), col - from);
    } else {
        Pack<T, VW> x;
        if (col < width)
            x = *reinterpret_cast<const Pack<T, VW>*>(row + col);
        else
#pragma unroll
            for (int i = 0; i < VW; ++i) x.v[i] = (T)0.f;
        return x;
    }
}

template <class T, int VW, int E, int TPR, bool RAG>
__device__ __forceinline__ void load_row(const T* row, int width, int lane, float* out) {
#pragma unroll
    for (int s = 0; s < E / VW; ++s) {
        Pack<T, VW> x;
        if (row)
            x = load_some<T, VW, RAG>(row, width, (s * TPR + lane) * VW);
        else
#pragma unroll
            for (int i = 0; i < VW; ++i) x.v[i] = (T)0.f;
#pragma unroll
        for (int i = 0; i < VW; ++i) out[s * VW + i] = (float)x.v[i];
    }
}

template <class T, int VW, int E, int TPR, bool RAG>
__device__ __forceinline__ void store_row(T* row, int width, int lane, const float* in) {
#pragma unroll
    for (int s = 0; s < E / VW; ++s) {
        const int col = (s * TPR + lane) * VW;
        Pack<T, VW> x;
#pragma unroll
        for (int i = 0; i < VW; ++i) x.v[i] = (T)in[s * VW + i];
        if constexpr (RAG) {
            if (col + VW <= width)
                store_anywhere(row + col, x);
            else
#pragma unroll
                for (int i = 0; i < VW; ++i)
                    if (col + i < width) row[col + i] = x.v[i];
        } else if (col < width)
            *reinterpret_cast<Pack<T, VW>*>(row + col) = x;
    }
}

// one instruction each for 2^x and 1 / x, both within a step of their type: off by about (1 + |u|) 2^-23 of its value
__device__ __forceinline__ float sigmoid(float u) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * u)); }

// A gate for the backward pass: the smaller of sigmoid(u) and sigmoid(-u), which holds the digits of both and of their product however far open or shut the
// gate is, in one register (65536 rows of 1024, bf16: 219 us; 281 us with sigmoid(-u) worked out from the logits at the end, which keeps those in registers).
struct Gate {
    float side;  // below 0 (or -0): sigmoid(-u), negated; else sigmoid(u)
    __device__ __forceinline__ Gate() {}
    __device__ __forceinline__ explicit Gate(float u) {
        const float e = __builtin_amdgcn_exp2f(-1.44269504f * __builtin_fabsf(u));
        side = __builtin_copysignf(e * __builtin_amdgcn_rcpf(1.f + e), -u);
    }
    __device__ __forceinline__ float open() const { return __builtin_bit_cast(int32_t, side) < 0 ? 1.f + side : side; }
    __device__ __forceinline__ float slope() const { return fmaf(-side, side, __builtin_fabsf(side)); }
    static __device__ __forceinline__ Gate none() {
        Gate g;
        g.side = -0.f;
        return g;
    }
};

// A row as it lies in memory, in registers; numbers are converted where they are used, so that the next row fits beside this one
template <class T, int VW, int E, int TPR, bool RAG>
struct RawRow {
    Pack<T, VW> x[E / VW];
    __device__ __forceinline__ void load(const T* row, int width, int lane) {
#pragma unroll
        for (int s = 0; s < E / VW; ++s) {
            if (row)
                x[s] = load_some<T, VW, RAG>(row, width, (s * TPR + lane) * VW);
            else
#pragma unroll
                for (int i = 0; i < VW; ++i) x[s].v[i] = (T)0.f;
        }
    }
    __device__ __forceinline__ float operator[](int i) const { return (float)x[i / VW].v[i % VW]; }
    __device__ __forceinline__ void again() {  // (the compiler is to convert once more, rather than keep the numbers converted)
        if constexpr (sizeof(T) == 2 && VW % 2 == 0)
#pragma unroll
            for (int s = 0; s < E / VW; ++s) {
                typedef uint32_t words __attribute__((ext_vector_type(VW / 2)));
                words w = __builtin_bit_cast(words, x[s]);
                asm volatile("" : "+v"(w));
                x[s] = __builtin_bit_cast(Pack<T, VW>, w);
            }
    }
};

template <class X, class B, int VW, int E, int TPR, bool RAG>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void block_forward_kernel(Block p) {
    __shared__ float shared[TPR > 64 ? TPR / 32 : 1];
    constexpr int RPB = TPR > 256 ? 1 : 256 / TPR;
    const int lane = threadIdx.x % TPR;
    const float share = 1.f / p.width;
    for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR; row < p.rows; row += (int64_t)gridDim.x * RPB) {
        float x[E], b[E], g[E], w[E];
        load_row<X, VW, E, TPR, RAG>((const X*)p.x + row * p.x_sr, p.width, lane, x);
        load_row<B, VW, E, TPR, RAG>((const B*)p.block + row * p.block_sr, p.width, lane, b);
        load_row<B, VW, E, TPR, RAG>(p.gate ? (const B*)p.gate + row * p.gate_sr : nullptr, p.width, lane, g);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) sum += b[i] * b[i];
        row_sums<TPR>(&sum, 1, shared);
        const float rb = 1.f / sqrtf(sum * share + p.eps);
#pragma unroll
        for (int i = 0; i < E; ++i) b[i] *= rb * (p.gate ? sigmoid(g[i]) : 1.f);
        load_row<float, VW, E, TPR, RAG>(p.post, p.width, lane, w);
        load_row<float, VW, E, TPR, RAG>(p.res, p.width, lane, g);
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            x[i] += g[i] * (w[i] * b[i]);
            sum += x[i] * x[i];
        }
        store_row<X, VW, E, TPR, RAG>((X*)p.y + row * p.width, p.width, lane, x);
        row_sums<TPR>(&sum, 1, shared);
        const float ry = 1.f / sqrtf(sum * share + p.eps);
        load_row<float, VW, E, TPR, RAG>(p.pre, p.width, lane, w);
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = x[i] * ry * w[i];
        store_row<B, VW, E, TPR, RAG>((B*)p.z + row * p.width, p.width, lane, x);
    }
}

// With bn = b / rms(b), yn = y / rms(y), sg = sigmoid(gate), f = the gradient of y, what came through z with it:
//     f   = dy + (dz pre - yn mean(dz pre yn)) / rms(y)
//     dx  = f;   dgate = f res bn post sg (1 - sg);   db = (e - bn mean(e bn)) / rms(b),  e = f res sg post
//     dpre = sum dz yn;   m = sum f sg bn:  dpost = res m,  dres = post m
// y is worked out again from x, b and the gate, which costs no memory.  A workgroup keeps its share of the two column sums in registers
// over all its rows and writes it once; column_sums adds the workgroups' shares in their order.  The next row is on its way while one is computed,
// kept as it lies in memory (two rows of 32-bit numbers would not fit beside the sums).
template <class X, class B, int VW, int E, int TPR, bool RAG>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void block_backward_kernel(Block p) {
    constexpr int RPB = TPR > 256 ? 1 : 256 / TPR;
    __shared__ float shared[TPR > 64 ? TPR / 32 : 1];
    __shared__ float fold[TPR == 64 ? 4 * 64 * E : 1];
    const int lane = threadIdx.x % TPR;
    const float share = 1.f / p.width;
    float sum_m[E], sum_p[E];
#pragma unroll
    for (int i = 0; i < E; ++i) sum_m[i] = sum_p[i] = 0.f;
    struct Rows5 {
        RawRow<X, VW, E, TPR, RAG> x, dy;
        RawRow<B, VW, E, TPR, RAG> b, g, dz;
    } now, next;
    auto load = [&](Rows5& r, int64_t row) {
        r.x.load((const X*)p.x + row * p.x_sr, p.width, lane);
        r.b.load((const B*)p.block + row * p.block_sr, p.width, lane);
        r.g.load(p.gate ? (const B*)p.gate + row * p.gate_sr : nullptr, p.width, lane);
        r.dy.load(p.grad_y ? (const X*)p.grad_y + row * p.grad_y_sr : nullptr, p.width, lane);
        r.dz.load(p.grad_z ? (const B*)p.grad_z + row * p.grad_z_sr : nullptr, p.width, lane);
    };
    const int64_t first = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR, step = (int64_t)gridDim.x * RPB;
    if (first < p.rows) load(next, first);
    for (int64_t row = first; row < p.rows; row += step) {
        now = next;
        if (row + step < p.rows) load(next, row + step);
        float sums[2] = {0.f, 0.f}, y[E], w[E], r[E];
        Gate gate[E];
#pragma unroll
        for (int i = 0; i < E; ++i) sums[0] += now.b[i] * now.b[i];
        row_sums<TPR>(sums, 1, shared);
        const float rb = 1.f / sqrtf(sums[0] * share + p.eps);
        now.b.again();
        load_row<float, VW, E, TPR, RAG>(p.post, p.width, lane, w);
        load_row<float, VW, E, TPR, RAG>(p.res, p.width, lane, r);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            gate[i] = p.gate ? Gate(now.g[i]) : Gate::none();
            w[i] *= r[i];
            y[i] = now.x[i] + w[i] * (gate[i].open() * (now.b[i] * rb));
        }
        load_row<float, VW, E, TPR, RAG>(p.pre, p.width, lane, r);
        sums[0] = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            sums[0] += y[i] * y[i];
            sums[1] += y[i] * (now.dz[i] * r[i]);
        }
        row_sums<TPR>(sums, 2, shared);
        const float ry = 1.f / sqrtf(sums[0] * share + p.eps), mean = sums[1] * ry * share;
        now.b.again(), now.dz.again();
        sums[0] = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) {  // y becomes f, r the gradient of the gate, w is times the gate from here on
            const float yn = y[i] * ry, bn = now.b[i] * rb;
            sum_p[i] += now.dz[i] * yn;
            y[i] = now.dy[i] + ry * (now.dz[i] * r[i] - yn * mean);
            const float sg = gate[i].open(), t = y[i] * bn;
            sum_m[i] += t * sg;
            r[i] = t * w[i] * gate[i].slope();
            w[i] *= sg;
            sums[0] += t * w[i];
        }
        store_row<X, VW, E, TPR, RAG>((X*)p.grad_x + row * p.width, p.width, lane, y);
        if (p.gate) store_row<B, VW, E, TPR, RAG>((B*)p.grad_gate + row * p.width, p.width, lane, r);
        row_sums<TPR>(sums, 1, shared);
        const float back = sums[0] * share;
        now.b.again();
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float bn = now.b[i] * rb;
            y[i] = rb * (y[i] * w[i] - bn * back);
        }
        store_row<B, VW, E, TPR, RAG>((B*)p.grad_block + row * p.width, p.width, lane, y);
    }
    float* to = p.partial + (int64_t)blockIdx.x * p.width;
    const int64_t second = (int64_t)gridDim.x * p.width;
    if (TPR > 64) {
        store_row<float, VW, E, TPR, RAG>(to, p.width, lane, sum_m);
        store_row<float, VW, E, TPR, RAG>(to + second, p.width, lane, sum_p);
    } else {
        const int wave = threadIdx.x / 64;
        for (int which = 0; which < 2; ++which) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < E; ++i) fold[(wave * E + i) * 64 + lane] = which ? sum_p[i] : sum_m[i];
            __syncthreads();
            for (int e = threadIdx.x; e < E * 64; e += 256) {
                const int i = e / 64, col = ((i / VW) * 64 + e % 64) * VW + i % VW;
                if (col < p.width) to[which * second + col] = fold[e] + fold[E * 64 + e] + fold[2 * E * 64 + e] + fold[3 * E * 64 + e];
            }
        }
    }
}

// grid (columns / 32, 2): 32 columns, 32 threads to each; blockIdx.y 0: post and res, 1: pre
__global__ __launch_bounds__(1024) void column_sums(const float* partial, int parts, int width, const float* post, const float* res, float* grad_post, float* grad_res, float* grad_pre) {
    __shared__ float fold[32][33];
    const int c = threadIdx.x % 32, r = threadIdx.x / 32, col = blockIdx.x * 32 + c;
    const float* from = partial + (int64_t)blockIdx.y * parts * width;
    float sum = 0.f;
    if (col < width)
        for (int i = r; i < parts; i += 32) sum += from[(int64_t)i * width + col];
    fold[r][c] = sum;
    __syncthreads();
    if (r == 0 && col < width) {
        sum = 0.f;
        for (int i = 0; i < 32; ++i) sum += fold[i][c];
        if (blockIdx.y)
            grad_pre[col] = sum;
        else {
            grad_post[col] = res[col] * sum;
            grad_res[col] = post[col] * sum;
        }
    }
}

constexpr int64_t BLOCK_PARTS = 512;

// Workgroups of the backward pass.  A wave or a workgroup takes a row at a time, so at most 4 rows are in a workgroup at once, and one where the row needs more
// than a wave: which kernel that is depends on the operands' alignment too, so the workspace is for the larger number.
// 512 rows of 750 (bf16), whose 256 threads hold one row: 512 workgroups 8.3 + 6.9 us for their sums, 128 workgroups 16.3 + 3.8 us; 1000 rows 12.2 + 6.6, 17.6 + 4.1.
int64_t backward_parts(int64_t rows, int64_t at_once) {
    const int64_t groups = ceil_div(rows, at_once);
    return groups < BLOCK_PARTS ? groups : BLOCK_PARTS;
}
int64_t most_parts(const lobpolicy_block* b) { return backward_parts(b->rows, b->width <= 512 ? 4 : 1); }

template <class X, class B, int VW, int E, int TPR, bool RAG, bool BACKWARD>
int block_launch(const Block& p, hipStream_t stream) {
    constexpr int threads = TPR > 256 ? TPR : 256;
    if constexpr (BACKWARD) {
        *p.parts = (int)backward_parts(p.rows, threads / TPR);
        block_backward_kernel<X, B, VW, E, TPR, RAG><<<dim3((unsigned)*p.parts), threads, 0, stream>>>(p);
    } else {
        const int64_t groups = ceil_div(p.rows, threads / TPR);
        block_forward_kernel<X, B, VW, E, TPR, RAG><<<dim3((unsigned)(groups < (1 << 20) ? groups : (1 << 20))), threads, 0, stream>>>(p);
    }
    return launched();
}

// A row to a wave as long as its registers hold it, then to as many threads as it needs: idle threads cost as much as busy ones.  64 M elements (bf16), us in a
// graph, forwards and with the gradients: 1024 wide a wave to a row 151 and 365, 256 threads to a row 208 and 639 (sums through LDS, every column sum in four
// times the threads); 4096 wide 512 threads 158 and 415, without them (1024 forwards, half of which are idle, 512 of 16 elements backwards) 295 and 605; 8192 wide,
// forwards 1024 threads 190 (512: 230), with the gradients, which take 512, 436 (1024, whose 128 registers do not hold a row and the next: 640 - 230 + 190 = 600).
template <class X, class B, int VW, bool RAG, bool BACKWARD>
int block_long(const Block& p, hipStream_t stream) {  // more than 512
    if constexpr (RAG) {  // (the shifted packs of 16 elements to a lane are more than the registers hold)
        if (p.width <= 1024) return block_launch<X, B, VW, 4, 256, RAG, BACKWARD>(p, stream);
    } else if (p.width <= 1024)
        return block_launch<X, B, VW, 16, 64, RAG, BACKWARD>(p, stream);
    if (p.width <= 2048) return block_launch<X, B, VW, 8, 256, RAG, BACKWARD>(p, stream);
    if (p.width <= 4096) return block_launch<X, B, VW, 8, 512, RAG, BACKWARD>(p, stream);
    if constexpr (!RAG && BACKWARD && VW > 1)
        return block_launch<X, B, VW, 16, 512, RAG, BACKWARD>(p, stream);
    else
        return block_launch<X, B, VW, 8, 1024, RAG, BACKWARD>(p, stream);
}

template <class X, class B, int VW, bool BACKWARD>
int block_short(const Block& p, hipStream_t stream) {  // up to 512
    if constexpr (VW < 8)
        if (p.width <= 256) return block_launch<X, B, VW, 4, 64, false, BACKWARD>(p, stream);
    return block_launch<X, B, VW, 8, 64, false, BACKWARD>(p, stream);
}

template <class X, class B, bool BACKWARD>
int block_typed(const Block& p, hipStream_t stream) {
    auto fits = [&](int w) {
        const int64_t xs = w * sizeof(X) < 16 ? w * sizeof(X) : 16, bs = w * sizeof(B) < 16 ? w * sizeof(B) : 16, fs = w * 4 < 16 ? w * 4 : 16;
        bool ok = p.width % w == 0 && p.x_sr % w == 0 && p.block_sr % w == 0 && p.gate_sr % w == 0 && p.grad_y_sr % w == 0 && p.grad_z_sr % w == 0;
        ok = ok && aligned(p.x, xs) && aligned(p.y, xs) && aligned(p.grad_y, xs) && aligned(p.grad_x, xs);
        ok = ok && aligned(p.block, bs) && aligned(p.gate, bs) && aligned(p.z, bs) && aligned(p.grad_z, bs) && aligned(p.grad_block, bs) && aligned(p.grad_gate, bs);
        return ok && aligned(p.post, fs) && aligned(p.res, fs) && aligned(p.pre, fs) && aligned(p.partial, fs);
    };
    // packs of 8 where a wave is full of them, else of 4; 1024 wide, 65536 rows, forwards and with the gradients, of 8 : of 4: 151 : 165 and 365 : 977 us (bf16), 191 : 194
    // and 474 : 937 (x f32), 254 : 238 and 664 : 645 (f32 only, where both are two loads, and of 4 are 2 to 5 % faster up to 2048 wide, 3 to 20 % slower beyond).  Rows of
    // no whole packs an element at a time up to 512 wide (65536 rows of 330: 62 + 177 us of kernels, in packs that begin anywhere 67 + 205; f32 46 + 212 and 81 + 273), and
    // long ones of f32 (8192 rows of 4001: 145 and 398 us, in packs 186 and 586), but long ones of 16-bit numbers in packs (118 and 436, an element at a time 409 and 608).
    const bool pack8 = p.width > 256 && fits(8), pack4 = fits(4);
    if (p.width <= 512) {
        if (pack8) return block_short<X, B, 8, BACKWARD>(p, stream);
        return pack4 ? block_short<X, B, 4, BACKWARD>(p, stream) : block_short<X, B, 1, BACKWARD>(p, stream);
    }
    if (pack8) return block_long<X, B, 8, false, BACKWARD>(p, stream);
    if (pack4) return block_long<X, B, 4, false, BACKWARD>(p, stream);
    if constexpr (sizeof(X) == 4 && sizeof(B) == 4)
        return block_long<X, B, 1, false, BACKWARD>(p, stream);
    else
        return block_long<X, B, 4, true, BACKWARD>(p, stream);
}

template <bool BACKWARD>
int block_any(const lobpolicy_block* b, const Block& p, void* stream) {
    hipStream_t s = (hipStream_t)stream;
    if (b->stream_dtype == LOBPOLICY_F32)
        return b->dtype == LOBPOLICY_F32 ? block_typed<float, float, BACKWARD>(p, s) : block_typed<float, bf16, BACKWARD>(p, s);
    return b->dtype == LOBPOLICY_F32 ? block_typed<bf16, float, BACKWARD>(p, s) : block_typed<bf16, bf16, BACKWARD>(p, s);
}

int check_block(const lobpolicy_block* b) {
    REQUIRE(b, "no description");
    for (int d : {b->stream_dtype, b->dtype}) REQUIRE(d == LOBPOLICY_F32 || d == LOBPOLICY_BF16, "dtype %d", d);
    REQUIRE(b->rows >= 1 && b->rows <= (1ll << 40), "rows = %lld: 1 to 2^40", (long long)b->rows);
    REQUIRE(b->width >= 1 && b->width <= LOBPOLICY_MAX_WIDTH, "width = %lld: 1 to %d", (long long)b->width, LOBPOLICY_MAX_WIDTH);
    REQUIRE(b->x && b->block && b->post && b->res && b->pre, "an operand is missing");
    return LOBPOLICY_OK;
}

Block block_of(const lobpolicy_block* b) {
    Block p = {};
    p.x = b->x, p.block = b->block, p.gate = b->gate;
    p.x_sr = b->x_stride, p.block_sr = b->block_stride, p.gate_sr = b->gate ? b->gate_stride : 0;
    p.post = b->post, p.res = b->res, p.pre = b->pre;
    p.rows = b->rows, p.width = (int)b->width, p.eps = b->eps;
    return p;
}

// ---------------------------------------------------------------------------------------------------------------------------
// the global norm, and clipping
//
// Two passes, each bound by memory (150 M values of both types, 457 MB: 100 us for the first, 4.6 TB/s, and 140 us for the second, 6.5 TB/s of reads
// and writes, of which the caches hold some): the squares are summed in 64 bits (which neither overflows nor loses what many small gradients add), one
// number per workgroup, in a fixed order; the second pass begins by adding those numbers up, in every workgroup alike, and scales.
// The tensors' table travels as a kernel argument: nothing is copied to the device, and a captured graph holds it.

constexpr int CLIP_TENSORS = 128;        // per launch: 3 KB of arguments
constexpr int64_t CLIP_CHUNK = 8192;     // elements
constexpr int64_t CLIP_FEW = 16;         // chunks of one launch
constexpr int64_t CLIP_PARTS = 2048;     // workgroups per launch, at most

struct ClipTable {
    void* data[CLIP_TENSORS];
    int64_t count[CLIP_TENSORS];
    uint32_t first[CLIP_TENSORS + 1];  // chunk at which each begins
    uint8_t dtype[CLIP_TENSORS];
    int n;
};

__device__ __forceinline__ int find_tensor(const ClipTable& t, uint32_t chunk) {
    int lo = 0, hi = t.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (t.first[mid] <= chunk)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

template <bool MAX>
__device__ __forceinline__ double join(double a, double b) {
    if (!MAX) return a + b;
    return a != a || a > b ? a : b;  // (not a number stays: b is taken where a > b is false, and b != b where a is one)
}

template <bool MAX>
__device__ __forceinline__ double joined(double x, double* shared) {  // over the workgroup, in a fixed order
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) x = join<MAX>(x, __shfl_xor(x, d));
    __syncthreads();
    if (threadIdx.x % 64 == 0) shared[threadIdx.x / 64] = x;
    __syncthreads();
    return join<MAX>(join<MAX>(shared[0], shared[1]), join<MAX>(shared[2], shared[3]));
}

// f(pointer to W elements, W) over the chunk's elements: single ones up to the first 16-byte boundary of the tensor and behind the last
template <class T, class One, class Many>
__device__ __forceinline__ void over_chunk(T* data, int64_t count, uint32_t chunk, One one, Many many) {
    constexpr int W = 16 / sizeof(T);
    const int thread = threadIdx.x % 256;
    int64_t head = (16 - (int64_t)((uintptr_t)data % 16)) % 16 / (int64_t)sizeof(T);
    head = head < count ? head : count;
    const int64_t begin = head + (int64_t)chunk * CLIP_CHUNK;
    int64_t end = begin + CLIP_CHUNK;
    end = end < count ? end : count;
    if (chunk == 0 && thread < head) one(data + thread);
    const int64_t whole = begin + (end - begin) / W * W;
    if (whole - begin == CLIP_CHUNK) {  // all loads of a whole chunk at once
#pragma unroll
        for (int k = 0; k < CLIP_CHUNK / (256 * W); ++k) many(data + begin + thread * W + k * 256 * W);
    } else {
#pragma unroll 4
        for (int64_t i = begin + thread * W; i < whole; i += 256 * W) many(data + i);
    }
    if (whole + thread < end) one(data + whole + thread);
}

template <bool MAX>
__global__ __launch_bounds__(256) void norm_kernel(ClipTable t, double* partial) {
    __shared__ double shared[4];
    double sum = 0.0;
    auto take = [&](float x) { sum = MAX ? join<true>(sum, (double)fabsf(x)) : fma((double)x, (double)x, sum); };
    for (uint32_t chunk = blockIdx.x; chunk < t.first[t.n]; chunk += gridDim.x) {
        const int i = find_tensor(t, chunk);
        auto go = [&](auto* data) {
            using T = std::remove_pointer_t<decltype(data)>;
            over_chunk(data, t.count[i], chunk - t.first[i], [&](T* p) { take((float)*p); },
                       [&](T* p) {
                           float x[16 / sizeof(T)];
                           load_pack<T, 16 / sizeof(T)>(p, x);
#pragma unroll
                           for (int e = 0; e < 16 / (int)sizeof(T); ++e) take(x[e]);
                       });
        };
        if (t.dtype[i] == LOBPOLICY_BF16)
            go((bf16*)t.data[i]);
        else
            go((float*)t.data[i]);
    }
    sum = joined<MAX>(sum, shared);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

template <bool MAX>
__global__ __launch_bounds__(256) void clip_kernel(ClipTable t, const double* partial, int parts, double max_norm, float* norm_out) {
    __shared__ double shared[4];
    double sum = 0.0;
    for (int i = threadIdx.x; i < parts; i += 256) sum = join<MAX>(sum, partial[i]);
    sum = joined<MAX>(sum, shared);
    const double norm = MAX ? sum : sqrt(sum);
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    const double ratio = max_norm / (norm + 1e-6);
    const float by = ratio > 1.0 ? 1.f : (float)ratio;  // (not a number stays one)
    if (by == 1.f) return;  // times one: the elements stay as they are
    // backwards: what the first pass read last is what the caches still hold
    for (uint32_t back = blockIdx.x; back < t.first[t.n]; back += gridDim.x) {
        const uint32_t chunk = t.first[t.n] - 1 - back;
        const int i = find_tensor(t, chunk);
        auto go = [&](auto* data) {
            using T = std::remove_pointer_t<decltype(data)>;
            over_chunk(data, t.count[i], chunk - t.first[i], [&](T* p) { *p = (T)((float)*p * by); },
                       [&](T* p) {
                           float x[16 / sizeof(T)];
                           load_pack<T, 16 / sizeof(T)>(p, x);
#pragma unroll
                           for (int e = 0; e < 16 / (int)sizeof(T); ++e) x[e] *= by;
                           store_pack<T, 16 / sizeof(T)>(p, x);
                       });
        };
        if (t.dtype[i] == LOBPOLICY_BF16)
            go((bf16*)t.data[i]);
        else
            go((float*)t.data[i]);
    }
}

// Few values: one workgroup does both passes in one launch, each quarter of it a chunk at a time.  What that saves is the second launch, which a program pays for that
// calls it as it goes along; in a captured graph, where launches are cheap, the kernel alone counts, which from 8 chunks on is slower than the two.  One
// launch : two, us a call, eager and in a graph: 1000 values 12.9 : 15.3 and 3.0 : 4.1; 65 536 11.2 : 14.2 and 4.9 : 5.0; six tensors of 69 636 in 13 chunks
// 16.6 : 19.7 and 6.3 : 5.1; 131 072 11.4 : 14.1 and 7.0 : 5.0.  The rule is for the eager call, and by the sizes alone, so that both give the same bits.
template <bool MAX>
__global__ __launch_bounds__(1024) void clip_few_kernel(ClipTable t, double max_norm, float* norm_out) {
    __shared__ double shared[16];
    double sum = 0.0;
    auto take = [&](float x) { sum = MAX ? join<true>(sum, (double)fabsf(x)) : fma((double)x, (double)x, sum); };
    // a quarter of the workgroup to a chunk, as over_chunk has it
    const uint32_t quarter = __builtin_amdgcn_readfirstlane(threadIdx.x / 256);
    for (uint32_t chunk = quarter; chunk < t.first[t.n]; chunk += 4) {
        const int i = find_tensor(t, chunk);
        auto go = [&](auto* data) {
            using T = std::remove_pointer_t<decltype(data)>;
            over_chunk(data, t.count[i], chunk - t.first[i], [&](T* p) { take((float)*p); },
                       [&](T* p) {
                           float x[16 / sizeof(T)];
                           load_pack<T, 16 / sizeof(T)>(p, x);
#pragma unroll
                           for (int e = 0; e < 16 / (int)sizeof(T); ++e) take(x[e]);
                       });
        };
        if (t.dtype[i] == LOBPOLICY_BF16)
            go((bf16*)t.data[i]);
        else
            go((float*)t.data[i]);
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) sum = join<MAX>(sum, __shfl_xor(sum, d));
    if (threadIdx.x % 64 == 0) shared[threadIdx.x / 64] = sum;
    __syncthreads();
    sum = shared[0];
#pragma unroll
    for (int k = 1; k < 16; ++k) sum = join<MAX>(sum, shared[k]);
    const double norm = MAX ? sum : sqrt(sum);
    if (threadIdx.x == 0) *norm_out = (float)norm;
    const double ratio = max_norm / (norm + 1e-6);
    const float by = ratio > 1.0 ? 1.f : (float)ratio;
    if (by == 1.f) return;
    for (uint32_t chunk = quarter; chunk < t.first[t.n]; chunk += 4) {
        const int i = find_tensor(t, chunk);
        auto go = [&](auto* data) {
            using T = std::remove_pointer_t<decltype(data)>;
            over_chunk(data, t.count[i], chunk - t.first[i], [&](T* p) { *p = (T)((float)*p * by); },
                       [&](T* p) {
                           float x[16 / sizeof(T)];
                           load_pack<T, 16 / sizeof(T)>(p, x);
#pragma unroll
                           for (int e = 0; e < 16 / (int)sizeof(T); ++e) x[e] *= by;
                           store_pack<T, 16 / sizeof(T)>(p, x);
                       });
        };
        if (t.dtype[i] == LOBPOLICY_BF16)
            go((bf16*)t.data[i]);
        else
            go((float*)t.data[i]);
    }
}

__global__ void zero_norm(float* norm) { *norm = 0.f; }

struct ClipPlan {  // the next up to CLIP_TENSORS tensors that are not empty, from index i on
    ClipTable table;
    int64_t next;
    int64_t parts;
};

ClipPlan clip_plan(void* const* tensors, const int64_t* counts, const int32_t* dtypes, int64_t n, int64_t i) {
    ClipPlan p;
    p.table.n = 0;
    uint64_t chunks = 0;
    for (; i < n && p.table.n < CLIP_TENSORS; ++i) {
        if (counts[i] == 0) continue;
        // (by the count alone: the elements in front of the first 16-byte boundary can only make it fewer chunks, and an empty chunk does nothing)
        const uint64_t more = (uint64_t)ceil_div(counts[i], CLIP_CHUNK);
        if (chunks + more > 0x7fffffffull && p.table.n) break;
        const int k = p.table.n++;
        p.table.data[k] = tensors ? tensors[i] : nullptr;
        p.table.count[k] = counts[i];
        p.table.dtype[k] = (uint8_t)dtypes[i];
        p.table.first[k] = (uint32_t)chunks;
        chunks += more;
        p.table.first[k + 1] = (uint32_t)chunks;
    }
    p.next = i;
    p.parts = (int64_t)(chunks < (uint64_t)CLIP_PARTS ? chunks : (uint64_t)CLIP_PARTS);
    return p;
}

int check_clip(const int64_t* counts, const int32_t* dtypes, int64_t n) {
    REQUIRE(n >= 0 && n <= 1000000, "n = %lld tensors", (long long)n);
    REQUIRE(n == 0 || (counts && dtypes), "no counts or dtypes");
    for (int64_t i = 0; i < n; ++i) {
        REQUIRE(counts[i] >= 0 && counts[i] <= (1ll << 43), "tensor %lld has %lld elements", (long long)i, (long long)counts[i]);
        REQUIRE(dtypes[i] == LOBPOLICY_F32 || dtypes[i] == LOBPOLICY_BF16, "tensor %lld: dtype %d", (long long)i, dtypes[i]);
    }
    return LOBPOLICY_OK;
}

int64_t clip_parts(const int64_t* counts, const int32_t* dtypes, int64_t n) {
    int64_t parts = 0;
    for (int64_t i = 0; i < n;) {
        const ClipPlan p = clip_plan(nullptr, counts, dtypes, n, i);
        parts += p.parts;
        i = p.next;
    }
    return parts;
}

}  // namespace lobpolicy

using namespace lobpolicy;

// ---------------------------------------------------------------------------------------------------------------------------
// the C-ABI

extern "C" {

int lobpolicy_abi_version(void) { return LOBPOLICY_ABI_VERSION; }
const char* lobpolicy_last_error(void) { return g_error; }

int64_t lobpolicy_attention_workspace(const lobpolicy_attention* a) {
    if (int e = check_attention(a)) return e;
    return Parts(a).bytes(a);
}

int lobpolicy_attention_forward(const lobpolicy_attention* a, void* stream) {
    if (int e = check_attention(a)) return e;
    REQUIRE(a->q.data && a->k.data && a->v.data && a->out.data, "an operand is missing");
    if (int e = check_workspace(a)) return e;
    Scan s = scan_of(a);
    s.a = rows_of(a->q), s.b = rows_of(a->k), s.c = rows_of(a->v), s.out = rows_of(a->out);
    s.da = a->dk, s.dc = a->dv;
    s.out_scale = a->scale;
    s.state_in = a->state_in, s.state_out = a->state_out;
    s.in_row = s.out_row = a->dv, s.in_col = s.out_col = 1;
    if (s.parts > 1) {
        if (int e = part_states(a, s, (hipStream_t)stream)) return e;
        s.state_in = (const float*)a->workspace, s.state_out = nullptr;
    }
    return walk(a, Walks{{s}, 1}, false, (hipStream_t)stream);
}

int lobpolicy_attention_backward(const lobpolicy_attention* a, void* stream) {
    if (int e = check_attention(a)) return e;
    REQUIRE(a->q.data && a->k.data && a->v.data && a->out.data, "an operand is missing");
    REQUIRE(a->grad_q.data && a->grad_k.data && a->grad_v.data, "a gradient is missing");
    if (int e = check_workspace(a)) return e;
    const Rows q = rows_of(a->q), k = rows_of(a->k), v = rows_of(a->v), d = rows_of(a->out);
    // backwards, the state's gradient: for dv, and transposed for dk; forwards, the state, transposed: for dq
    Scan s = scan_of(a);
    s.a = k, s.b = q, s.c = d, s.out = rows_of(a->grad_v);
    s.da = a->dk, s.dc = a->dv, s.in_row = s.out_row = a->dv, s.in_col = s.out_col = 1;
    s.reverse = true, s.in_scale = a->scale;
    s.state_in = a->grad_state_out, s.state_out = a->grad_state_in;
    const float* states = a->state_in;
    if (s.parts > 1) {
        REQUIRE(a->forward_workspace && aligned(a->forward_workspace, 16), "no forward_workspace");
        if (int e = part_states(a, s, (hipStream_t)stream)) return e;
        s.state_in = (const float*)a->workspace, s.state_out = nullptr;
        states = (const float*)a->forward_workspace;
    }
    Walks w = {{s, s, s}, 3};
    for (int i = 1; i < 3; ++i) w.walk[i].da = a->dv, w.walk[i].dc = a->dk, w.walk[i].in_row = 1, w.walk[i].in_col = a->dv, w.walk[i].state_out = nullptr;
    w.walk[1].a = v, w.walk[1].b = d, w.walk[1].c = q, w.walk[1].out = rows_of(a->grad_k);
    w.walk[2].a = d, w.walk[2].b = v, w.walk[2].c = k, w.walk[2].out = rows_of(a->grad_q);
    w.walk[2].reverse = false, w.walk[2].in_scale = 1.f, w.walk[2].out_scale = a->scale, w.walk[2].state_in = states;
    return walk(a, w, true, (hipStream_t)stream);
}

int lobpolicy_attention_step(const lobpolicy_attention* a, void* stream) {
    if (int e = check_attention(a)) return e;
    REQUIRE(a->steps == 1, "a step takes one token of every environment: steps = %lld", (long long)a->steps);
    REQUIRE(a->q.data && a->k.data && a->v.data && a->out.data && a->state_out, "an operand is missing");
    Step s = {};
    s.q = a->q.data, s.k = a->k.data, s.v = a->v.data, s.out = a->out.data;
    s.q_sn = a->q.stride_n, s.q_sh = a->q.stride_h, s.k_sn = a->k.stride_n, s.k_sh = a->k.stride_h;
    s.v_sn = a->v.stride_n, s.v_sh = a->v.stride_h, s.out_sn = a->out.stride_n, s.out_sh = a->out.stride_h;
    s.log_decay = a->log_decay, s.reset = a->reset, s.reset_sn = a->reset_stride_n, s.skip = a->skip;
    s.state = a->state_out, s.heads = a->heads, s.dk = a->dk, s.dv = a->dv, s.scale = a->scale;
    const int64_t units = a->envs * a->heads;
    return a->dtype == LOBPOLICY_BF16 ? step_typed<bf16>(s, units, (hipStream_t)stream) : step_typed<float>(s, units, (hipStream_t)stream);
}

int64_t lobpolicy_block_workspace(const lobpolicy_block* b) {
    if (int e = check_block(b)) return e;
    return 2 * most_parts(b) * b->width * (int64_t)sizeof(float);
}

int lobpolicy_block_forward(const lobpolicy_block* b, void* stream) {
    if (int e = check_block(b)) return e;
    REQUIRE(b->y && b->z, "a result is missing");
    Block p = block_of(b);
    p.y = b->y, p.z = b->z;
    return block_any<false>(b, p, stream);
}

int lobpolicy_block_backward(const lobpolicy_block* b, void* stream) {
    if (int e = check_block(b)) return e;
    REQUIRE(b->grad_x && b->grad_block && (b->grad_gate || !b->gate) && b->grad_post && b->grad_res && b->grad_pre, "a gradient is missing");
    REQUIRE(b->workspace && b->workspace_bytes >= lobpolicy_block_workspace(b), "the workspace has %lld bytes", (long long)b->workspace_bytes);
    Block p = block_of(b);
    p.grad_y = b->grad_y, p.grad_z = b->grad_z, p.grad_y_sr = b->grad_y ? b->grad_y_stride : 0, p.grad_z_sr = b->grad_z ? b->grad_z_stride : 0;
    p.grad_x = b->grad_x, p.grad_block = b->grad_block, p.grad_gate = b->grad_gate;
    p.partial = (float*)b->workspace;
    int parts = 0;
    p.parts = &parts;
    if (int e = block_any<true>(b, p, stream)) return e;
    column_sums<<<dim3((unsigned)ceil_div(b->width, 32), 2), 1024, 0, (hipStream_t)stream>>>(p.partial, parts, p.width, b->post, b->res, b->grad_post, b->grad_res, b->grad_pre);
    return launched();
}

int64_t lobpolicy_clip_workspace(const int64_t* counts, const int32_t* dtypes, int64_t n) {
    if (int e = check_clip(counts, dtypes, n)) return e;
    return clip_parts(counts, dtypes, n) * (int64_t)sizeof(double);
}

int lobpolicy_clip(void* const* tensors, const int64_t* counts, const int32_t* dtypes, int64_t n, int32_t kind, double max_norm, float* norm, void* workspace,
                   int64_t workspace_bytes, void* stream) {
    if (int e = check_clip(counts, dtypes, n)) return e;
    REQUIRE(kind == 0 || kind == 2, "kind = %d: 0 (largest) or 2 (squares)", kind);
    REQUIRE(max_norm >= 0.0, "max_norm = %g", max_norm);
    REQUIRE(norm && (n == 0 || tensors), "an operand is missing");
    for (int64_t i = 0; i < n; ++i)
        REQUIRE(counts[i] == 0 || (tensors[i] && aligned(tensors[i], dtypes[i] == LOBPOLICY_BF16 ? 2 : 4)), "tensor %lld: no data, or not aligned to its type", (long long)i);
    hipStream_t s = (hipStream_t)stream;
    const int64_t parts = clip_parts(counts, dtypes, n);
    if (parts == 0) {
        zero_norm<<<1, 1, 0, s>>>(norm);
        return launched();
    }
    REQUIRE(parts <= 0x7fffffff && workspace && aligned(workspace, 8) && workspace_bytes >= parts * (int64_t)sizeof(double), "the workspace has %lld bytes", (long long)workspace_bytes);
    const ClipPlan all = clip_plan(tensors, counts, dtypes, n, 0);
    if (all.next == n && parts <= CLIP_FEW) {
        if (kind == 0)
            clip_few_kernel<true><<<1, 1024, 0, s>>>(all.table, max_norm, norm);
        else
            clip_few_kernel<false><<<1, 1024, 0, s>>>(all.table, max_norm, norm);
        return launched();
    }
    double* partial = (double*)workspace;
    int64_t at = 0;
    for (int64_t i = 0; i < n;) {
        const ClipPlan p = clip_plan(tensors, counts, dtypes, n, i);
        if (p.parts) {
            if (kind == 0)
                norm_kernel<true><<<dim3((unsigned)p.parts), 256, 0, s>>>(p.table, partial + at);
            else
                norm_kernel<false><<<dim3((unsigned)p.parts), 256, 0, s>>>(p.table, partial + at);
            if (int e = launched()) return e;
        }
        at += p.parts;
        i = p.next;
    }
    float* first = norm;  // the first launch writes it
    for (int64_t i = 0; i < n;) {
        const ClipPlan p = clip_plan(tensors, counts, dtypes, n, i);
        if (p.parts) {
            if (kind == 0)
                clip_kernel<true><<<dim3((unsigned)p.parts), 256, 0, s>>>(p.table, partial, (int)parts, max_norm, first);
            else
                clip_kernel<false><<<dim3((unsigned)p.parts), 256, 0, s>>>(p.table, partial, (int)parts, max_norm, first);
            if (int e = launched()) return e;
            first = nullptr;
        }
        i = p.next;
    }
    return LOBPOLICY_OK;
}

}  // extern "C"
