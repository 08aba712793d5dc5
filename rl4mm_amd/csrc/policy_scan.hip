// policy_scan.hip - decay attention over segments: the kernels of one type and one width of a state's rows, chosen by -DLOBPOLICY_TYPE and
// -DLOBPOLICY_ROWS (the library holds the six of float and __bf16 with 32, 64 and 128).
#include "policy_common.h"

namespace lobpolicy {

// ---- chunks of tokens on the matrix units ------------------------------------------------------------------------------------
//
// CH tokens at a time, with the state S at their beginning (p: place in the chunk, e^g = l):
//     out_i = out_scale ( l^(i+1) a_i S + sum_{j <= i} l^(i-j) in_scale (a_i . b_j) c_j ),    S <- l^CH S + sum_j l^(CH-1-j) in_scale b_j c_j^T
// where a reset between j and i takes the term away.  Four products of tiles, on 16x16 matrix instructions; one workgroup walks the
// chunks of one environment and head (or of a part of its steps), its waves share the state by columns:
//   - scores, transposed (rows j, columns i), weighted and put to LDS as T, each tile by one wave
//   - out, transposed (rows c, columns i), each wave its own columns of the state: S as it lies in the accumulators is the left operand
//     of a_i S (an accumulator holds rows 4 (lane / 16) .. + 3 of column lane % 16, which read the other way round is the operand's
//     layout), so the state never leaves the registers
//   - the state's update
// The tiles a, b, c lie in LDS as they lie in memory; what needs them by columns reads them transposed (bf16: the transposing LDS load,
// f32: single words).  Rows are padded by 16 bytes, which spreads 16 rows over all banks.  The next chunk's tiles are on their way from
// memory while one is computed.
//
// Exponents are never negative (all products are of j <= i), so no decay overflows.  What is masked is selected away, not multiplied by
// 0; a chunk that holds an infinity or a NaN anywhere is computed token by token instead, from the same LDS tiles, because a matrix
// product would spread it to tokens that do not see it.
//
// bf16: what multiplies a bf16 operand is split, so that a result is rounded once, as it is stored: scores and the state's copy that multiplies a into two
// bf16 (the number, and what its rounding leaves: off by 2^-16 of a term), the weighted c of the state's update, which adds up over all steps, into
// three (24 bits).  The second halves cost (kernels): 4500 steps, 128 units of 128 to 128, forwards 176 -> 199 us, the three walks of the backward pass 494 -> 561 us,
// four fifths of it the state's; 128 steps, 2048 units of 64 to 64, forwards, 47 us in chunks of 64 without them, 46 us in chunks of 32 with them.
//
// Few chunks are bound by what a chunk's products wait for in turn, many by the issue of instructions: at 128 to 128 (bf16, 4500 steps, 128 units, forwards and the
// three walks) the matrix units work 21 %, the vector units 38 %, LDS 24 % of the time, at 1.5 waves to a SIMD; at 64 to 64 (bf16, 128 steps, 2048 units) 11, 53 and
// 27 %.  Forwards, kernels, us:
//     128 steps, 2048 units of 64 to 64, bf16      46    4.4 TB/s of operands, results and states
//     20 steps, 16384 units of 32 to 32, f32       91    3.3 TB/s
//     18000 steps, 8 units of 64 to 64, f32        81    22 the parts' states, 10 joined, 49 the outputs
//     4500 steps, 128 units of 128 to 128, bf16   297    79, 19, 199
// The token by token recurrence took 350 us of the first (the state's row in registers, a read and a write of LDS to each token) and 37 700 of the third.

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// a lane's place in a 16 x 16 tile.  `fresh` makes it a value that the compiler knows nothing of: what is worked out from it inside the walk
// (addresses, comparisons) is then worked out where it is used, and not kept in registers from chunk to chunk
struct Lane {
    int l, g;
    __device__ __forceinline__ void fresh() { asm volatile("" : "+v"(l), "+v"(g)); }
};

// Two numbers rounded to bf16, and what that leaves of them
__device__ __forceinline__ bf16x2 rounded(float& x, float& y) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const bf16x2 two = __builtin_convertvector((f32x2{x, y}), bf16x2);
    const uint32_t both = __builtin_bit_cast(uint32_t, two);
    x -= __builtin_bit_cast(float, both << 16);
    y -= __builtin_bit_cast(float, both & 0xffff0000u);
    return two;
}

template <class T>
struct Tile;

template <>
struct Tile<float> {  // a fragment: 16 of the summed index, places 4 (lane / 16) + r in its word r
    typedef f32x4 Frag;
    static constexpr int K = 16, PAD = 4;
    static __device__ __forceinline__ f32x4 product(Frag a, Frag b, f32x4 c) {
#pragma unroll
        for (int r = 0; r < 4; ++r) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], b[r], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ Frag rows(Lane at, const float* tile, int stride, int row, int k) {  // tile[row + lane % 16][k ..]
        return *reinterpret_cast<const f32x4*>(tile + (row + at.l) * stride + k + 4 * at.g);
    }
    static __device__ __forceinline__ Frag rows_as_state(Lane at, const float* tile, int stride, int row, int k) { return rows(at, tile, stride, row, k); }
    static __device__ __forceinline__ Frag columns(Lane at, const float* tile, int stride, int k, int column) {  // tile[k ..][column + lane % 16]
        Frag f;
#pragma unroll
        for (int r = 0; r < 4; ++r) f[r] = tile[(k + 4 * at.g + r) * stride + column + at.l];
        return f;
    }
    static __device__ __forceinline__ int place(Lane at, int e) { return 4 * at.g + e; }  // of a fragment's element e in `columns`
    static constexpr int HALVES = 1;  // fragments that hold 32-bit numbers where they multiply operands of T
    static __device__ __forceinline__ void of_state(const f32x4* s, Frag* f) { f[0] = s[0]; }
    static constexpr int SPLITS = 1;
    // c's columns times w, as SPLITS fragments whose sum is the product
    static __device__ __forceinline__ void weighted(Frag c, const float* w, Frag* f) {
#pragma unroll
        for (int r = 0; r < 4; ++r) f[0][r] = c[r] * w[r];
    }
};

template <>
struct Tile<bf16> {  // a fragment: 32 of the summed index, places 8 (lane / 16) + e
    typedef bf16x8 Frag;
    static constexpr int K = 32, PAD = 8;
    static __device__ __forceinline__ f32x4 product(Frag a, Frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ Frag rows(Lane at, const bf16* tile, int stride, int row, int k) {
        return *reinterpret_cast<const bf16x8*>(tile + (row + at.l) * stride + k + 8 * at.g);
    }
    // the order in which two accumulators one above the other hold the summed index: 4 (lane / 16) + r, then 16 more
    static __device__ __forceinline__ Frag rows_as_state(Lane at, const bf16* tile, int stride, int row, int k) {
        const bf16x4 lo = *reinterpret_cast<const bf16x4*>(tile + (row + at.l) * stride + k + 4 * at.g), hi = *reinterpret_cast<const bf16x4*>(tile + (row + at.l) * stride + k + 16 + 4 * at.g);
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    // 16 lanes that address 4 rows of 16 elements, 4 elements each, get a column each
    static __device__ __forceinline__ Frag columns(Lane at, const bf16* tile, int stride, int k, int column) {
        typedef __attribute__((address_space(3))) s16x4 lds;
        const bf16* from = tile + (k + 8 * at.g + at.l / 4) * stride + column + at.l % 4 * 4;
        const bf16x4 lo = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds*)(from)));
        const bf16x4 hi = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds*)(from + 4 * stride)));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    static __device__ __forceinline__ int place(Lane at, int e) { return 8 * at.g + e; }
    static constexpr int HALVES = 2;  // a number and what its rounding leaves, rounded: 17 bits
    static __device__ __forceinline__ void of_state(const f32x4* s, Frag* f) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            float x = s[e / 4][e % 4], y = s[e / 4][e % 4 + 1];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const bf16x2 two = rounded(x, y);
                f[half][e] = two[0], f[half][e + 1] = two[1];
            }
        }
    }
    static constexpr int SPLITS = 3;
    static __device__ __forceinline__ void weighted(Frag c, const float* w, Frag* f) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            uint32_t x = __builtin_bit_cast(uint32_t, (float)c[e] * w[e]), y = __builtin_bit_cast(uint32_t, (float)c[e + 1] * w[e + 1]);
#pragma unroll
            for (int i = 0; i < 3; ++i) {  // the upper 8 bits of what is left, exactly (cut off, not rounded), two at a time
                const uint32_t both = __builtin_amdgcn_perm(y, x, 0x07060302);
                const bf16x2 two = __builtin_bit_cast(bf16x2, both);
                f[i][e] = two[0], f[i][e + 1] = two[1];
                x = __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, x) - __builtin_bit_cast(float, x & 0xffff0000u));
                y = __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, y) - __builtin_bit_cast(float, y & 0xffff0000u));
            }
        }
    }
};

template <class T, int CH, int DA, int DC>
struct Shape {
    // tiles of 16 of the state's columns to a wave: each operand that waves share is read from LDS once for both (4096 steps, 128 units of 128 to 128,
    // bf16: 295 us, with the gradients 850; one tile to a wave 328 and 1060; at 64 columns two tiles leave two waves to a workgroup)
    static constexpr int COLS = DC == 128 ? 2 : 1;
    static constexpr int WAVES = DC / 16 / COLS, THREADS = 64 * WAVES;
    static constexpr int PAD = Tile<T>::PAD, SA = DA + PAD, SC = DC + PAD, SP = CH + PAD;
};

// A tile's share of a thread, on its way: CH places in the order of the walk, 16 bytes at a time.  `at` is the thread's first row in the chunk to be
// loaded next, `step` the bytes from place to place (negative where the walk goes backwards).  Rows behind the last place are loaded from the
// chunk's first row instead and become 0 when they are stored: a branch around a load would make the next wait one for every load.
// MODE 2: the rows begin at multiples of 16 bytes and are whole packs.  1: they begin anywhere and are one pack long or longer, and the last pack is
// loaded as the row's last elements and shifted when it is stored.  0: anything, an element at a time.
template <class T, int CH, int D, int THREADS, int MODE>
struct Moving {
    static constexpr int VW = 16 / (int)sizeof(T), ROW = D / VW, ROWS = THREADS / ROW, N = CH > ROWS ? CH / ROWS : 1;
    static_assert(THREADS % ROW == 0 && (CH % ROWS == 0 || ROWS % CH == 0), "");
    static __device__ __forceinline__ int first_row() { return threadIdx.x / ROW; }
    static __device__ __forceinline__ int column() { return threadIdx.x % ROW * VW; }
    static __device__ __forceinline__ bool takes_part() { return ROWS <= CH || first_row() < CH; }
    Pack<T, VW> x[N];
    const char *origin, *at;  // the chunk's first row, and the thread's
    int64_t step;
    int width;

    __device__ __forceinline__ int start() const {  // the column that is loaded for column()
        if (MODE == 1) return column() < width - VW ? column() : width - VW;
        return column() < width ? column() : 0;
    }
    __device__ __forceinline__ void begin(const void* base, int64_t st, int64_t first_token, bool reverse, int elements) {
        step = (reverse ? -st : st) * (int64_t)sizeof(T);
        width = elements;
        origin = (const char*)base + first_token * st * (int64_t)sizeof(T);
        at = origin + first_row() * step + start() * (int)sizeof(T);
    }
    __device__ __forceinline__ void load(int places) {  // and on to the next chunk
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const T* from = reinterpret_cast<const T*>(first_row() + n * ROWS < places ? at + n * ROWS * step : origin);
            if (MODE == 2)
                x[n] = *reinterpret_cast<const Pack<T, VW>*>(from);
            else if (MODE == 1)
                x[n] = load_anywhere<T, VW>(from);
            else {
#pragma unroll
                for (int e = 0; e < VW; ++e) x[n].v[e] = column() + e < width ? from[e] : (T)0.f;
            }
        }
        origin += CH * step;
        at += CH * step;
    }
    __device__ __forceinline__ void store(T* tile, int stride, int places) {
        if (places < CH || width < D) {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                if (MODE == 1) x[n] = shifted(x[n], column() - start());
                if (first_row() + n * ROWS >= places || column() >= width) x[n] = __builtin_bit_cast(Pack<T, VW>, make_uint4(0, 0, 0, 0));
            }
        }
        if (!takes_part()) return;
#pragma unroll
        for (int n = 0; n < N; ++n) *reinterpret_cast<Pack<T, VW>*>(tile + (first_row() + n * ROWS) * stride + column()) = x[n];
    }
};

// 4 columns from j on of an output's row
template <class T, int MODE>
__device__ __forceinline__ void store_columns(T* to, int j, int width, f32x4 x) {
    Pack<T, 4> y;
#pragma unroll
    for (int r = 0; r < 4; ++r) y.v[r] = (T)x[r];
    if (MODE == 2) {
        if (j < width) *reinterpret_cast<Pack<T, 4>*>(to + j) = y;
    } else if (MODE == 1 && j + 4 <= width)
        store_anywhere(to + j, y);
    else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (j + r < width) to[j + r] = y.v[r];
    }
}

// A column of a state's matrix, by buffer instructions: a load from behind the buffer's end gives 0, a store there does nothing
struct Column {
    __amdgpu_buffer_rsrc_t buffer;
    int at, row, rows;  // bytes
    __device__ __forceinline__ Column(const float* base, const Scan& s, int64_t row_stride, int64_t col_stride, int column)
        : buffer(__builtin_amdgcn_make_buffer_rsrc((void*)base, 0, s.da * s.dc * 4, 0x27000)), at(column < s.dc ? column * (int)col_stride * 4 : 0x40000000), row((int)row_stride * 4), rows(s.da) {}
    __device__ __forceinline__ int offset(int i) const {
        const int inside = at + i * row;
        return i < rows ? inside : 0x40000000;
    }
    __device__ __forceinline__ float load(int i) const { return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(buffer, offset(i), 0, 0)); }
    __device__ __forceinline__ void store(int i, float x) const { __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, x), buffer, offset(i), 0, 0); }
};

// 4 neighbouring scores to LDS: to each half, `apart` elements from one to the next; their sum are the scores
template <class T>
__device__ __forceinline__ void put_scores(T* to, int apart, f32x4 x) {
#pragma unroll
    for (int half = 0; half < Tile<T>::HALVES; ++half) {
        Pack<T, 4> p;
        if constexpr (Tile<T>::HALVES == 2) {
#pragma unroll
            for (int r = 0; r < 4; r += 2) {
                float a = x[r], b = x[r + 1];
                const bf16x2 two = rounded(a, b);
                p.v[r] = two[0], p.v[r + 1] = two[1];
                x[r] = a, x[r + 1] = b;
            }
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) p.v[r] = (T)x[r];
        }
        *reinterpret_cast<Pack<T, 4>*>(to + half * apart) = p;
    }
}

// What a workgroup keeps in LDS
template <class T, int CH, int DA, int DC, bool OUT>
struct Room {
    typedef Shape<T, CH, DA, DC> S;
    alignas(16) T a[OUT ? CH * S::SA : 8];
    alignas(16) T b[CH * S::SA];
    alignas(16) T c[CH * S::SC];
    alignas(16) T p[OUT ? Tile<T>::HALVES * CH * S::SP : 8];
    alignas(16) float leave[CH];              // l^(CH - 1 - j) in_scale
    float power[CH + 1], enter[CH + 1];       // l^k, and times out_scale
    uint32_t spoiled[2];
};

// One part of one walk.  OUT: its outputs; without it the state behind the part alone, from a state of 0 in front of it
template <class T, int CH, int DA, int DC, bool OUT, int MODE>
__device__ __forceinline__ void walk_part(const Scan& s, int64_t unit, int64_t part, Room<T, CH, DA, DC, OUT>& room) {
    typedef Shape<T, CH, DA, DC> S;
    typedef Tile<T> M;
    typedef typename M::Frag Frag;
    // whether the next chunk is on its way while one is computed: not where the registers end (128 to 128, the case above: ahead 300 and 878 us)
    constexpr bool AHEAD = !OUT || DA + DC < 256;
    constexpr int KA = DA / M::K, KC = CH / M::K, DT = DA / 16, PER = M::K / 16, HALVES = M::HALVES, APART = CH * S::SP;
    T *const tile_a = room.a, *const tile_b = room.b, *const tile_c = room.c, *const tile_p = room.p;
    float *const power = room.power, *const enter = room.enter, *const leave = room.leave;
    uint32_t* const spoiled = room.spoiled;
    const bool reverse = s.reverse;
    const int64_t n = (uint32_t)unit / (uint32_t)s.heads;
    const int h = (int)((uint32_t)unit % (uint32_t)s.heads);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, column = wave * S::COLS * 16;
    Lane at = {lane % 16, lane / 16};

    const int64_t length = __builtin_amdgcn_readfirstlane((int)length_of(s, n)), begin = part * s.part_steps;
    const int64_t end = begin + s.part_steps < length ? begin + s.part_steps : length;
    const int64_t first_token = reverse ? length - 1 - begin : begin;
    T* out = OUT ? (T*)s.out.data + n * s.out.sn + h * s.out.sh : nullptr;
    // (without resets some byte that is there is loaded, and not used: no branch around the load)
    const uint8_t* reset = s.reset ? s.reset + n * s.reset_sn : (const uint8_t*)s.log_decay;
    const int64_t reset_st = s.reset ? s.reset_st : 0;
    // of the chunk from place `first` on: whether nothing in front of place first + lane reaches it, loaded ahead and looked at later
    auto has_flag = [&](int64_t first) { return s.reset && lane < CH && first + lane < end && (!reverse || first + lane > 0); };
    auto load_flag = [&](int64_t first) -> uint32_t { return reset[(has_flag(first) ? (reverse ? length - (first + lane) : first + lane) : 0) * reset_st]; };

    const float log_decay = s.log_decay[h];
    Moving<T, CH, DA, S::THREADS, MODE> move_a, move_b;
    Moving<T, CH, DC, S::THREADS, MODE> move_c;
    uint32_t flag = 0;
    if (OUT) move_a.begin((const T*)s.a.data + n * s.a.sn + h * s.a.sh, s.a.st, first_token, reverse, s.da);
    move_b.begin((const T*)s.b.data + n * s.b.sn + h * s.b.sh, s.b.st, first_token, reverse, s.da);
    move_c.begin((const T*)s.c.data + n * s.c.sn + h * s.c.sh, s.c.st, first_token, reverse, s.dc);
    auto load = [&](int64_t first) {
        const int places = end - first < CH ? (int)(end - first) : CH;
        if (OUT) move_a.load(places);
        move_b.load(places);
        move_c.load(places);
        flag = load_flag(first);
    };
    if (AHEAD && begin < end) load(begin);

    const int64_t matrix = (int64_t)s.da * s.dc, which = s.parts == 1 ? unit : unit * s.parts + part;
    f32x4 state[S::COLS][DT];  // rows 16 t + 4 g + r, column `column` + 16 ct + l
#pragma unroll
    for (int ct = 0; ct < S::COLS; ++ct) {
#pragma unroll
        for (int t = 0; t < DT; ++t) state[ct][t] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (s.state_in) {
            const Column from(s.state_in + which * matrix, s, s.in_row, s.in_col, column + 16 * ct + at.l);
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) state[ct][t][r] = from.load(16 * t + 4 * at.g + r);
        }
    }

    auto decay_of = [&](int k) { return k == 0 ? 1.f : expf(log_decay * (float)k); };  // (k = 0: not 0 * infinity)
    for (int k = threadIdx.x; k <= CH; k += S::THREADS) {
        const float x = decay_of(k);
        power[k] = x;
        enter[k] = x * s.out_scale;
        if (k < CH) leave[CH - 1 - k] = x * s.in_scale;
    }
    if (threadIdx.x < 2) spoiled[threadIdx.x] = 0;
    // (the state has arrived before the walk begins: inside, a wait for it would be one for the loads ahead too)
#pragma unroll
    for (int ct = 0; ct < S::COLS; ++ct)
#pragma unroll
        for (int t = 0; t < DT; ++t) asm volatile("" : "+v"(state[ct][t]));

    __syncthreads();
    float w_diagonal[4], w_below[4];  // of a score tile on the diagonal, and of the one below it
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int gap = at.l - 4 * at.g - r;
        w_diagonal[r] = gap >= 0 ? enter[gap >= 0 ? gap : 0] * s.in_scale : 0.f;
        w_below[r] = enter[16 + gap] * s.in_scale;
    }

    int parity = 0;
    uint64_t any_cut = 0;
    for (int64_t first = begin; first < end; first += CH, parity ^= 1) {
        at.fresh();
        const int places = end - first < CH ? (int)(end - first) : CH;
        if (!AHEAD) load(first);
        if (OUT) move_a.store(tile_a, S::SA, places);
        move_b.store(tile_b, S::SA, places);
        move_c.store(tile_c, S::SC, places);
        const uint64_t cuts = __ballot(has_flag(first) && flag != 0);
        any_cut |= cuts;
        __syncthreads();
        if (AHEAD && first + CH < end) load(first + CH);
        const int enters = reverse && first == 0 ? 0 : 1;  // decays between what comes into the chunk and its first place
        const int tiles = (places + 15) / 16;
        Frag values[S::COLS][KC];  // c, by columns
#pragma unroll
        for (int ct = 0; ct < S::COLS; ++ct)
#pragma unroll
            for (int kk = 0; kk < KC; ++kk) values[ct][kk] = M::columns(at, tile_c, S::SC, kk * M::K, column + 16 * ct);
        if (OUT) {
            float spoils = 0.f;  // becomes NaN with the first number that is none, or infinite
            // scores: tile k = (it, jt), jt <= it, holds rows j = 16 jt + .., columns i = 16 it + ..; two at once, whose latencies overlap
            const int count = tiles * (tiles + 1) / 2;
            for (int k0 = wave; k0 < count; k0 += 2 * S::WAVES) {
                int it[2], jt[2];
                f32x4 x[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int k = k0 + u * S::WAVES < count ? k0 + u * S::WAVES : k0;
                    it[u] = k >= 6 ? 3 : k >= 3 ? 2 : k >= 1 ? 1 : 0, jt[u] = k - it[u] * (it[u] + 1) / 2;
                }
#pragma unroll
                for (int kk = 0; kk < KA; ++kk)
#pragma unroll
                    for (int u = 0; u < 2; ++u)
                        x[u] = M::product(M::rows(at, tile_b, S::SA, 16 * jt[u], kk * M::K), M::rows(at, tile_a, S::SA, 16 * it[u], kk * M::K), x[u]);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int i = 16 * it[u] + at.l;
                    const bool diagonal = it[u] == jt[u];
                    const float far = it[u] - jt[u] > 1 ? power[16 * (it[u] - jt[u] - 1)] : 1.f;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        x[u][r] *= diagonal ? w_diagonal[r] : w_below[r] * far;
                        spoils = fmaf(x[u][r], 0.f, spoils);  // (the tiles on the diagonal see every row of a and b; weighted, as halves of an infinity are none)
                    }
                    if (cuts) {
                        const uint64_t before = cuts & (~0ull >> (63 - i));
                        const int from = before ? 63 - __builtin_clzll(before) : 0;  // the first place that i sees
#pragma unroll
                        for (int r = 0; r < 4; ++r) x[u][r] = 16 * jt[u] + 4 * at.g + r >= from ? x[u][r] : 0.f;
                    }
                    T* to = tile_p + i * S::SP + 16 * jt[u] + 4 * at.g;
                    put_scores(to, APART, x[u]);
                    // the tile above the diagonal that shares a fragment with it
                    if (PER == 2 && diagonal && it[u] % 2 == 0) put_scores(to + 16, APART, f32x4{0.f, 0.f, 0.f, 0.f});
                }
            }
            if (spoils != 0.f) spoiled[parity] = 1;
            __syncthreads();
        }
        bool by_token = OUT && __builtin_amdgcn_readfirstlane(spoiled[parity]) != 0;
        if (OUT && threadIdx.x == 0) spoiled[parity ^ 1] = 0;
        auto token = [&](int p) { return (reverse ? length - 1 - (first + p) : first + p) * s.out.st; };

        if (OUT && !by_token) {
            Frag left[S::COLS][KA][HALVES];
#pragma unroll
            for (int ct = 0; ct < S::COLS; ++ct)
#pragma unroll
                for (int kk = 0; kk < KA; ++kk) M::of_state(&state[ct][kk * PER], left[ct][kk]);
            T* to = out + token(at.l);
            const int64_t on = (reverse ? -16 : 16) * s.out.st;
            float spoils = 0.f;
#pragma unroll 1
            for (int pair = 0; pair < tiles; pair += 2) {  // two tiles at once; a second one behind the last is computed, and dropped
                at.fresh();
                f32x4 x[2][S::COLS];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int ct = 0; ct < S::COLS; ++ct) x[u][ct] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kk = 0; kk < KA; ++kk)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const Frag right = M::rows_as_state(at, tile_a, S::SA, 16 * (pair + u), kk * M::K);
#pragma unroll
                        for (int ct = 0; ct < S::COLS; ++ct)
#pragma unroll
                            for (int half = 0; half < HALVES; ++half) x[u][ct] = M::product(left[ct][kk][half], right, x[u][ct]);
                    }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int i = 16 * (pair + u) + at.l;
                    const float w = enter[i + enters];
#pragma unroll
                    for (int ct = 0; ct < S::COLS; ++ct) x[u][ct] *= w;
                    if (cuts) {
                        const bool sees = (cuts & (~0ull >> (63 - i))) == 0;
#pragma unroll
                        for (int ct = 0; ct < S::COLS; ++ct)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                spoils = fmaf(x[u][ct][r], 0.f, spoils);  // (the last tile need not see the state)
                                x[u][ct][r] = sees ? x[u][ct][r] : 0.f;
                            }
                    }
                }
#pragma unroll
                for (int kk = 0; kk < KC; ++kk)
#pragma unroll
                    for (int u = 0; u < 2; ++u)
                        if (kk * PER <= pair + (PER == 2 ? 0 : u)) {
#pragma unroll
                            for (int half = 0; half < HALVES; ++half) {
                                const Frag right = M::rows(at, tile_p + half * APART, S::SP, 16 * (pair + u), kk * M::K);
#pragma unroll
                                for (int ct = 0; ct < S::COLS; ++ct) x[u][ct] = M::product(values[ct][kk], right, x[u][ct]);
                            }
                        }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    if (pair + u == tiles - 1) {
#pragma unroll
                        for (int ct = 0; ct < S::COLS; ++ct)
#pragma unroll
                            for (int r = 0; r < 4; ++r) spoils = fmaf(x[u][ct][r], 0.f, spoils);
                    }
                    if (16 * (pair + u) + at.l < places) {
#pragma unroll
                        for (int ct = 0; ct < S::COLS; ++ct) store_columns<T, MODE>(to, column + 16 * ct + 4 * at.g, s.dc, x[u][ct]);
                    }
                    to += on;
                }
            }
            // the last tile's products see every c: one that is not finite in this wave's columns (or the state) shows in them, and the wave, whose
            // columns are its own, begins again token by token
            by_token = __ballot(spoils != 0.f) != 0;
        }
        if (by_token) {
#pragma unroll 1
            for (int p = 0; p < places; ++p) {
                const bool cut = cuts >> p & 1;
                const float carry = power[p == 0 ? enters : 1];
                at.fresh();
#pragma unroll
                for (int ct = 0; ct < S::COLS; ++ct) {
                    const int j = column + 16 * ct + at.l;
                    const float value = (float)tile_c[p * S::SC + j] * s.in_scale;
                    float sum = 0.f;
#pragma unroll
                    for (int t = 0; t < DT; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int i = 16 * t + 4 * at.g + r;
                            const float x = (cut ? 0.f : state[ct][t][r] * carry) + (float)tile_b[p * S::SA + i] * value;
                            state[ct][t][r] = i < s.da ? x : 0.f;
                            sum += i < s.da ? (float)tile_a[p * S::SA + i] * x : 0.f;
                        }
                    sum += __shfl_xor(sum, 16);
                    sum += __shfl_xor(sum, 32);
                    if (at.g == 0 && j < s.dc) out[token(p) + j] = (T)(sum * s.out_scale);
                }
            }
        } else {
            // the state: what comes in decays by the whole chunk, place j by what lies behind it
            const int last_cut = cuts ? 63 - __builtin_clzll(cuts) : 0;
            const float whole = power[places - 1 + enters];
            if (cuts) {
#pragma unroll
                for (int ct = 0; ct < S::COLS; ++ct)
#pragma unroll
                    for (int t = 0; t < DT; ++t) state[ct][t] = f32x4{0.f, 0.f, 0.f, 0.f};
            } else {
#pragma unroll
                for (int ct = 0; ct < S::COLS; ++ct)
#pragma unroll
                    for (int t = 0; t < DT; ++t) state[ct][t] *= whole;
            }
            float w[KC][M::K / 4];
            if (places == CH && !cuts) {
#pragma unroll
                for (int kk = 0; kk < KC; ++kk) load_pack<float, M::K / 4>(leave + kk * M::K + M::place(at, 0), w[kk]);
            } else {
#pragma unroll
                for (int kk = 0; kk < KC; ++kk)
#pragma unroll
                    for (int e = 0; e < M::K / 4; ++e) {
                        const int j = kk * M::K + M::place(at, e);
                        w[kk][e] = j >= last_cut && j < places ? power[places - 1 - j] * s.in_scale : 0.f;
                    }
            }
#pragma unroll
            for (int kk = 0; kk < KC; ++kk) {
                Frag right[S::COLS][M::SPLITS];
#pragma unroll
                for (int ct = 0; ct < S::COLS; ++ct) M::weighted(values[ct][kk], w[kk], right[ct]);
#pragma unroll
                for (int t = 0; t < DT; ++t) {
                    const Frag left = M::columns(at, tile_b, S::SA, kk * M::K, 16 * t);
#pragma unroll
                    for (int ct = 0; ct < S::COLS; ++ct)
#pragma unroll
                        for (int i = 0; i < M::SPLITS; ++i) state[ct][t] = M::product(left, right[ct][i], state[ct][t]);
                }
            }
        }
        __syncthreads();
    }
    if (!OUT) {
        // What is not finite has stayed in the state, or was cut off.  Whether it is infinite or no number at all is told by a walk of the wave's columns token
        // by token: parts of an infinity, an infinity times decays whose product is 0 in 32 bits, and an infinity times the 0 of a cut are no numbers above
        float spoils = 0.f;
#pragma unroll
        for (int ct = 0; ct < S::COLS; ++ct)
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) spoils = fmaf(state[ct][t][r], 0.f, spoils);
        if (__ballot(spoils != 0.f)) {
            const T *rows_b = (const T*)s.b.data + n * s.b.sn + h * s.b.sh, *rows_c = (const T*)s.c.data + n * s.c.sn + h * s.c.sh;
#pragma unroll
            for (int ct = 0; ct < S::COLS; ++ct)
#pragma unroll
                for (int t = 0; t < DT; ++t) state[ct][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
            for (int64_t place = begin; place < end; ++place) {
                const int64_t token = reverse ? length - 1 - place : place;
                const bool cut = s.reset && (!reverse || place > 0) && reset[(reverse ? length - place : place) * reset_st];
                at.fresh();
#pragma unroll
                for (int ct = 0; ct < S::COLS; ++ct) {
                    const int j = column + 16 * ct + at.l;
                    const float value = j < s.dc ? (float)rows_c[token * s.c.st + j] * s.in_scale : 0.f;
#pragma unroll
                    for (int t = 0; t < DT; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int i = 16 * t + 4 * at.g + r;
                            if (i < s.da) state[ct][t][r] = (cut ? 0.f : state[ct][t][r] * power[1]) + (float)rows_b[token * s.b.st + i] * value;
                        }
                }
            }
        }
    }

    if (OUT && part == s.parts - 1 && length < s.steps)  // rows behind the last token
        for (int64_t t = length + threadIdx.x / 32; t < s.steps; t += S::THREADS / 32)
            for (int j = threadIdx.x % 32; j < s.dc; j += 32) out[t * s.out.st + j] = (T)0.f;
    if (!OUT && threadIdx.x == 0) {
        // the least number above 0 for a product of decays that is 0 in 32 bits: an infinite state stays infinite, and of a finite one less than 5e-7 is left
        const float carry = decay_of(begin < end ? (int)(end - begin) - (reverse && begin == 0 ? 1 : 0) : 0);
        s.carry_out[which] = any_cut ? -1.f : carry == 0.f && power[1] != 0.f ? 0x1p-149f : carry;
    }
    if (s.state_out) {
        const bool leaves = reverse && s.parts == 1 && length > 0, cut = leaves && s.reset && reset[0];
        const float carry = leaves ? power[1] : 1.f;
#pragma unroll
        for (int ct = 0; ct < S::COLS; ++ct) {
            const Column to(s.state_out + which * matrix, s, s.out_row, s.out_col, column + 16 * ct + at.l);
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) to.store(16 * t + 4 * at.g + r, cut ? 0.f : state[ct][t][r] * carry);
        }
    }
}

// ---- short segments: all three gradients at once -----------------------------------------------------------------------------
//
// Where the steps are one chunk of 32, a workgroup reads q, k, v and do once and writes dq, dk, dv and the gradient of the initial state: with
// A = l^(i-j) scale (q_i . k_j) and Z = l^(i-j) scale (do_i . v_j), lower triangles without what a reset cuts, S0 the initial state, R the gradient
// of the final one,
//     dq_i = sum_j Z_ij k_j + scale l^(i+1) S0 do_i          dk_j = sum_i Z_ij q_i + l^(L-1-j) R v_j
//     dv_j = sum_i A_ij do_i + l^(L-1-j) R^T k_j             dS0 = l^L R + scale sum_i l^(i+1) q_i do_i^T
// Both score matrices lie in LDS by rows i: dq reads them by rows, dk and dv by columns.  Each wave has 16 columns of every result.  Three walks
// read 9 operands instead of 4 and make 3 score matrices instead of 2: 20 steps x 16384 units, with the forward pass, take
// 314 us that way and 257 us this (32 to 32, f32: 27 KB of LDS, 2 waves to a SIMD), 195 and 169 us (32 to 32, bf16), 584 and 490 us (64 to 64, bf16).
// A chunk with an infinity or a NaN is left to the walks.

template <class T, int DK, int DV>
struct OnceRoom {
    static constexpr int CH = 32;
    static constexpr int SK = DK + Tile<T>::PAD, SV = DV + Tile<T>::PAD, SP = CH + Tile<T>::PAD, APART = CH * SP;
    alignas(16) T q[CH * SK], k[CH * SK], v[CH * SV], d[CH * SV], a[Tile<T>::HALVES * APART], z[Tile<T>::HALVES * APART];
    float power[CH + 1];
    uint32_t spoiled;
};

// E floats as fragments of T, whose sum they are; what is not finite is the first one's alone
template <class T, int E>
__device__ __forceinline__ void in_halves(const float* x, typename Tile<T>::Frag* f) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
        f[0][e] = (T)x[e];
        if constexpr (Tile<T>::HALVES == 2) f[1][e] = (T)(__builtin_isfinite((float)f[0][e]) ? x[e] - (float)f[0][e] : 0.f);
    }
}

// Fragments of a matrix of floats in memory, [rows][columns] without gaps (NULL: zeros), the summed index in the order of Tile::rows
template <class T, bool VEC, int K>
__device__ __forceinline__ void matrix_rows(typename Tile<T>::Frag* f, __amdgpu_buffer_rsrc_t buffer, Lane at, int rows, int columns, int row, int k) {
    constexpr int E = K / 4;
    float x[E];
    const int i = row + at.l, j = k + E * at.g;
    if constexpr (VEC) {
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
            const u32x4 y = __builtin_amdgcn_raw_buffer_load_b128(buffer, i < rows ? (j + e < columns ? (i * columns + j + e) * 4 : 0x40000000) : 0x40000000, 0, 0);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const uint32_t word = y[u];
                x[e + u] = __builtin_bit_cast(float, word);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
            x[e] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(buffer, i < rows ? (j + e < columns ? (i * columns + j + e) * 4 : 0x40000000) : 0x40000000, 0, 0));
    }
    in_halves<T, E>(x, f);
}
template <class T, int K>
__device__ __forceinline__ void matrix_columns(typename Tile<T>::Frag* f, __amdgpu_buffer_rsrc_t buffer, Lane at, int rows, int columns, int k, int column) {
    constexpr int E = K / 4;
    float x[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int i = k + E * at.g + e, j = column + at.l;
        x[e] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(buffer, i < rows ? (j < columns ? (i * columns + j) * 4 : 0x40000000) : 0x40000000, 0, 0));
    }
    in_halves<T, E>(x, f);
}

// A kernel's first argument, read from memory from here on: what only a later part of the kernel needs is not kept in registers up to there
template <class A>
__device__ __forceinline__ const A& argument_again() {
    auto from = (const __attribute__((address_space(4))) A*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(from));
    return *(const A*)from;
}

template <class T, int DK, int DV, int MODE>
__global__ __launch_bounds__((DK > DV ? DK : DV) * 4) void gradients_once(Walks w) {
    typedef Tile<T> M;
    typedef typename M::Frag Frag;
    typedef OnceRoom<T, DK, DV> R;
    constexpr int CH = R::CH;
    constexpr int WAVES = (DK > DV ? DK : DV) / 16, THREADS = 64 * WAVES, PER = M::K / 16, KC = CH / M::K, KK = DK / M::K, KV = DV / M::K, HALVES = M::HALVES;
    static_assert((Shape<T, CH, DK, DV>::THREADS > Shape<T, CH, DV, DK>::THREADS ? Shape<T, CH, DK, DV>::THREADS : Shape<T, CH, DV, DK>::THREADS) == THREADS, "");
    union Shared {
        R once;
        Room<T, CH, DK, DV, true> one;
        Room<T, CH, DV, DK, true> other;
    };
    __shared__ __align__(16) char room[sizeof(Shared)];
    Shared& shared = *reinterpret_cast<Shared*>(room);
    R& s = shared.once;

    const Scan &of_v = w.walk[0], &of_k = w.walk[1], &of_q = w.walk[2];
    const uint32_t each = gridDim.x / 8, more = gridDim.x % 8, die = blockIdx.x % 8, unit = die * each + (die < more ? die : more) + blockIdx.x / 8;
    const int64_t n = unit / (uint32_t)of_v.heads;
    const int h = (int)(unit % (uint32_t)of_v.heads), dk = of_v.da, dv = of_v.dc;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, column = 16 * wave;
    Lane at = {lane % 16, lane / 16};
    const int length = __builtin_amdgcn_readfirstlane((int)length_of(of_v, n)), tiles = ((length + 15) / 16 + PER - 1) / PER * PER;
    const float scale = of_v.in_scale, log_decay = of_v.log_decay[h];

    Moving<T, CH, DK, THREADS, MODE> move_q, move_k;
    Moving<T, CH, DV, THREADS, MODE> move_v, move_d;
    move_q.begin((const T*)of_v.b.data + n * of_v.b.sn + h * of_v.b.sh, of_v.b.st, 0, false, dk);
    move_k.begin((const T*)of_v.a.data + n * of_v.a.sn + h * of_v.a.sh, of_v.a.st, 0, false, dk);
    move_v.begin((const T*)of_k.a.data + n * of_k.a.sn + h * of_k.a.sh, of_k.a.st, 0, false, dv);
    move_d.begin((const T*)of_v.c.data + n * of_v.c.sn + h * of_v.c.sh, of_v.c.st, 0, false, dv);
    move_q.load(length), move_k.load(length), move_v.load(length), move_d.load(length);
    const bool flagged = of_v.reset && lane < length && of_v.reset[n * of_v.reset_sn + (lane < length ? lane : 0) * of_v.reset_st];

    // the two states, as the results need them
    const int bytes = dk * dv * 4;
    const bool with_s0 = of_q.state_in, with_r = of_v.state_in;
    const __amdgpu_buffer_rsrc_t s0 = __builtin_amdgcn_make_buffer_rsrc((void*)(of_q.state_in + (int64_t)unit * dk * dv), 0, with_s0 ? bytes : 0, 0x27000);
    const __amdgpu_buffer_rsrc_t rr = __builtin_amdgcn_make_buffer_rsrc((void*)(of_v.state_in + (int64_t)unit * dk * dv), 0, with_r ? bytes : 0, 0x27000);
    Frag s0_rows[KV][HALVES], r_rows[KV][HALVES], r_columns[KK][HALVES];
#pragma unroll
    for (int kk = 0; kk < KV; ++kk) {
        matrix_rows<T, MODE == 2, M::K>(s0_rows[kk], s0, at, dk, dv, column, kk * M::K);
        matrix_rows<T, MODE == 2, M::K>(r_rows[kk], rr, at, dk, dv, column, kk * M::K);
    }
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) matrix_columns<T, M::K>(r_columns[kk], rr, at, dk, dv, kk * M::K, column);

    for (int k = threadIdx.x; k <= CH; k += THREADS) s.power[k] = k == 0 ? 1.f : expf(log_decay * (float)k);
    if (threadIdx.x == 0) s.spoiled = 0;
    move_q.store(s.q, R::SK, length), move_k.store(s.k, R::SK, length), move_v.store(s.v, R::SV, length), move_d.store(s.d, R::SV, length);
    const uint64_t cuts = __ballot(flagged);
    __syncthreads();
    float w_diagonal[4], w_below[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int gap = at.l - 4 * at.g - r;
        w_diagonal[r] = gap >= 0 ? s.power[gap >= 0 ? gap : 0] * scale : 0.f;
        w_below[r] = s.power[16 + gap] * scale;
    }
    float spoils = 0.f;  // becomes NaN with the first number that is none, or infinite
    const int count = tiles * (tiles + 1) / 2;
    for (int k0 = wave; k0 < count; k0 += WAVES) {
        const int it = k0 >= 1 ? 1 : 0, jt = k0 == 2 ? 1 : 0, i = 16 * it + at.l;
        f32x4 x[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) x[0] = M::product(M::rows(at, s.k, R::SK, 16 * jt, kk * M::K), M::rows(at, s.q, R::SK, 16 * it, kk * M::K), x[0]);
#pragma unroll
        for (int kk = 0; kk < KV; ++kk) x[1] = M::product(M::rows(at, s.v, R::SV, 16 * jt, kk * M::K), M::rows(at, s.d, R::SV, 16 * it, kk * M::K), x[1]);
        const uint64_t before = cuts & (~0ull >> (63 - i));
        const int from = before ? 63 - __builtin_clzll(before) : 0;  // the first place that i sees
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            T* to = (u ? s.z : s.a) + i * R::SP + 16 * jt + 4 * at.g;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float y = x[u][r] * (it == jt ? w_diagonal[r] : w_below[r]);
                spoils = fmaf(y, 0.f, spoils);
                x[u][r] = 16 * jt + 4 * at.g + r >= from ? y : 0.f;
            }
            put_scores(to, R::APART, x[u]);
            // the tile above the diagonal that shares a fragment with it
            if (PER == 2 && it == jt && it % 2 == 0) put_scores(to + 16, R::APART, f32x4{0.f, 0.f, 0.f, 0.f});
        }
    }
    if (spoils != 0.f) s.spoiled = 1;
    __syncthreads();
    const bool by_walks = __builtin_amdgcn_readfirstlane(s.spoiled) != 0;
    if (by_walks) {  // (the walk with fewer waves last: the others have ended by then)
        const Scan &of_v = argument_again<Walks>().walk[0], &of_k = argument_again<Walks>().walk[1], &of_q = argument_again<Walks>().walk[2];
        __syncthreads();
        constexpr int first = Shape<T, CH, DK, DV>::THREADS, others = Shape<T, CH, DV, DK>::THREADS;
        if (first >= others) {
            walk_part<T, CH, DK, DV, true, MODE>(of_v, unit, 0, shared.one);
            __syncthreads();
            if (threadIdx.x >= others) return;
        }
        walk_part<T, CH, DV, DK, true, MODE>(of_k, unit, 0, shared.other);
        __syncthreads();
        walk_part<T, CH, DV, DK, true, MODE>(of_q, unit, 0, shared.other);
        if (first < others) {
            __syncthreads();
            if (threadIdx.x >= first) return;
            walk_part<T, CH, DK, DV, true, MODE>(of_v, unit, 0, shared.one);
        }
        return;
    }

    const int last_cut = cuts ? 63 - __builtin_clzll(cuts) : 0;
    // what the state's gradient behind the last token is worth at token j
    auto tail = [&](int j, f32x4 x) {
        const float by = s.power[j < length ? length - 1 - j : 0];
        const bool seen = j >= last_cut;
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = seen ? x[r] * by : 0.f;
        return x;
    };
    if (column < DK) {
        const Scan &of_k = argument_again<Walks>().walk[1], &of_q = argument_again<Walks>().walk[2];
        T* to_q = (T*)of_q.out.data + n * of_q.out.sn + h * of_q.out.sh;
        T* to_k = (T*)of_k.out.data + n * of_k.out.sn + h * of_k.out.sh;
        Frag keys[KC], queries[KC];
#pragma unroll
        for (int kk = 0; kk < KC; ++kk) keys[kk] = M::columns(at, s.k, R::SK, kk * M::K, column), queries[kk] = M::columns(at, s.q, R::SK, kk * M::K, column);
#pragma unroll 1
        for (int it = 0; it < tiles; ++it) {
            at.fresh();
            const int i = 16 * it + at.l;
            f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kk = 0; kk < KV; ++kk) {
                const Frag gradients = M::rows(at, s.d, R::SV, 16 * it, kk * M::K), values = M::rows(at, s.v, R::SV, 16 * it, kk * M::K);
#pragma unroll
                for (int half = 0; half < HALVES; ++half) {
                    x = M::product(s0_rows[kk][half], gradients, x);
                    y = M::product(r_rows[kk][half], values, y);
                }
            }
            const float by = s.power[i + 1] * scale;
            const bool sees = (cuts & (~0ull >> (63 - i))) == 0;
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = sees ? x[r] * by : 0.f;
            y = tail(i, y);
#pragma unroll
            for (int kk = 0; kk < KC; ++kk) {
#pragma unroll
                for (int half = 0; half < HALVES; ++half) {
                    if (kk * PER <= it) x = M::product(keys[kk], M::rows(at, s.z + half * R::APART, R::SP, 16 * it, kk * M::K), x);
                    if (kk * PER + PER > it && kk * PER < tiles) y = M::product(queries[kk], M::columns(at, s.z + half * R::APART, R::SP, kk * M::K, 16 * it), y);
                }
            }
            if (i < length) {
                store_columns<T, MODE>(to_q + i * of_q.out.st, column + 4 * at.g, dk, x);
                store_columns<T, MODE>(to_k + i * of_k.out.st, column + 4 * at.g, dk, y);
            }
        }
        for (int64_t t = length + lane / 16; t < of_q.steps; t += 4)
            if (column + at.l < dk) to_q[t * of_q.out.st + column + at.l] = to_k[t * of_k.out.st + column + at.l] = (T)0.f;
    }
    if (column < DV) {
        const Scan& of_v = argument_again<Walks>().walk[0];
        T* to = (T*)of_v.out.data + n * of_v.out.sn + h * of_v.out.sh;
        Frag values[KC];
#pragma unroll
        for (int kk = 0; kk < KC; ++kk) values[kk] = M::columns(at, s.d, R::SV, kk * M::K, column);
#pragma unroll 1
        for (int jt = 0; jt < tiles; ++jt) {
            at.fresh();
            const int j = 16 * jt + at.l;
            f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                const Frag keys = M::rows(at, s.k, R::SK, 16 * jt, kk * M::K);
#pragma unroll
                for (int half = 0; half < HALVES; ++half) x = M::product(r_columns[kk][half], keys, x);
            }
            x = tail(j, x);
#pragma unroll
            for (int kk = 0; kk < KC; ++kk)
                if (kk * PER + PER > jt && kk * PER < tiles) {
#pragma unroll
                    for (int half = 0; half < HALVES; ++half) x = M::product(values[kk], M::columns(at, s.a + half * R::APART, R::SP, kk * M::K, 16 * jt), x);
                }
            if (j < length) store_columns<T, MODE>(to + j * of_v.out.st, column + 4 * at.g, dv, x);
        }
        for (int64_t t = length + lane / 16; t < of_v.steps; t += 4)
            if (column + at.l < dv) to[t * of_v.out.st + column + at.l] = (T)0.f;
        if (of_v.state_out) {
            const int first_cut = cuts ? __builtin_ctzll(cuts) : 64;
            const Column to_state(of_v.state_out + (int64_t)unit * dk * dv, of_v, dv, 1, column + at.l);
            const Column from(of_v.state_in + (int64_t)unit * dk * dv, of_v, dv, 1, column + at.l);
            const float whole = s.power[length];
            Frag right[KC][M::SPLITS];
#pragma unroll
            for (int kk = 0; kk < KC; ++kk) {
                float by[M::K / 4];
#pragma unroll
                for (int e = 0; e < M::K / 4; ++e) {
                    const int i = kk * M::K + M::place(at, e);
                    by[e] = i < first_cut && i < length ? s.power[i + 1] * scale : 0.f;
                }
                M::weighted(values[kk], by, right[kk]);
            }
#pragma unroll 1
            for (int t = 0; t < DK / 16; ++t) {
                f32x4 x = {0.f, 0.f, 0.f, 0.f};
                if (with_r && !cuts) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) x[r] = from.load(16 * t + 4 * at.g + r) * whole;
                }
#pragma unroll
                for (int kk = 0; kk < KC; ++kk) {
                    const Frag left = M::columns(at, s.q, R::SK, kk * M::K, 16 * t);
#pragma unroll
                    for (int i = 0; i < M::SPLITS; ++i) x = M::product(left, right[kk][i], x);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) to_state.store(16 * t + 4 * at.g + r, x[r]);
            }
        }
    }
}

// BOTH: the second and third walk have da and dc the other way round
template <class T, int CH, int DA, int DC, bool BOTH>
constexpr int SCAN_THREADS = BOTH && Shape<T, CH, DC, DA>::THREADS > Shape<T, CH, DA, DC>::THREADS ? Shape<T, CH, DC, DA>::THREADS : Shape<T, CH, DA, DC>::THREADS;

template <class T, int CH, int DA, int DC, bool BOTH, bool OUT, int MODE>
__global__ __launch_bounds__((SCAN_THREADS<T, CH, DA, DC, BOTH>), 2) void scan_chunks(Walks w) {
    union Shared {
        Room<T, CH, DA, DC, OUT> one;
        Room<T, CH, BOTH ? DC : DA, BOTH ? DA : DC, OUT> other;
    };
    __shared__ __align__(16) char room[sizeof(Shared)];
    Shared& shared = *reinterpret_cast<Shared*>(room);
    // neighbouring workgroups run on different dies, each with a cache of its own: every die gets a run of neighbouring units, and all walks of a unit
    const uint32_t units = (uint32_t)(w.walk[0].envs * w.walk[0].heads), each = gridDim.x / 8, more = gridDim.x % 8, die = blockIdx.x % 8;
    const uint32_t index = die * each + (die < more ? die : more) + blockIdx.x / 8;
    const uint32_t which = index % (uint32_t)w.count, place = index / (uint32_t)w.count;
    const Scan& s = w.walk[which];
    if (!BOTH || which == 0) {
        if (threadIdx.x < Shape<T, CH, DA, DC>::THREADS) walk_part<T, CH, DA, DC, OUT, MODE>(s, place % units, place / units, shared.one);
    } else if (BOTH) {
        if (threadIdx.x < Shape<T, CH, DC, DA>::THREADS) walk_part<T, CH, BOTH ? DC : DA, BOTH ? DA : DC, OUT, MODE>(s, place % units, place / units, shared.other);
    }
}

// Chunks of 32 tokens, of 64 where both widths of a bf16 state are above 64: scores cost CH instructions' worth a token and take CH * CH of LDS, the state's
// rounding, update and barriers 1 / CH.  32 : 64, us in a graph, forwards or (+) with the gradients:
//     f32    512 steps, 512 units of 64 to 64 94 : 110, +310 : 392, of 32 to 32 +163 : 223
//     bf16   32 to 32: 4096 steps, 512 units +703 : 856, 128 steps, 8192 units +312 : 403;  64 to 64: 128 steps, 2048 units 49 : 55, 4096 steps, 512 units 349 : 343;
//            128 to 32: 1024 steps, 512 units 129 : 129, +404 : 461;  128 to 128: 4500 steps, 128 units +964 : 930, 1024 steps, 512 units +713 : 677
template <class T, int DA, int DC>
constexpr bool LONG_CHUNKS = sizeof(T) == 2 && DA > 64 && DC > 64;

template <class T, int CH, int DA, int DC, bool BOTH, int MODE>
int scan_launch(const Walks& w, hipStream_t stream) {
    const Scan& s = w.walk[0];
    const dim3 grid((unsigned)(s.envs * s.heads * s.parts * w.count));
    constexpr int threads = SCAN_THREADS<T, CH, DA, DC, BOTH>;
    if (s.out.data)
        scan_chunks<T, CH, DA, DC, BOTH, true, MODE><<<grid, threads, 0, stream>>>(w);
    else if constexpr (!BOTH && (CH > 32 || !LONG_CHUNKS<T, DA, DC>))  // (a part's state: there are many steps)
        scan_chunks<T, CH, DA, DC, false, false, MODE><<<grid, threads, 0, stream>>>(w);
    return launched();
}

template <class T, int DK, int DV, int MODE>
int once_launch(const Walks& w, hipStream_t stream) {
    const Scan& s = w.walk[0];
    gradients_once<T, DK, DV, MODE><<<dim3((unsigned)(s.envs * s.heads)), (DK > DV ? DK : DV) * 4, 0, stream>>>(w);
    return launched();
}

template <class T, int CH, int DA, int DC, int MODE>
int scan_mode(const Walks& w, bool swapped, hipStream_t stream) {
    if constexpr (DA <= 64 && DC <= 64)
        if (swapped && w.walk[0].steps <= 32) return once_launch<T, DA, DC, MODE>(w, stream);
    if constexpr (DA != DC)
        if (swapped) return scan_launch<T, CH, DA, DC, true, MODE>(w, stream);
    return scan_launch<T, CH, DA, DC, false, MODE>(w, stream);
}

// Whole packs of 16 bytes where every row begins and ends at one, packs that begin anywhere and shift their last where a row is one or longer (512 steps, 512
// units of 61 to 61, forwards and with the gradients: bf16 62 and 195 us, an element at a time 95 and 332; f32 102 and 340, 124 and 433), else elements
template <class T, int CH, int DA, int DC>
int scan_aligned(const Walks& w, bool swapped, hipStream_t stream) {
    constexpr int W = 16 / sizeof(T);
    bool wide = true, packs = true;
    for (int i = 0; i < w.count; ++i) {
        const Scan& s = w.walk[i];
        packs = packs && s.da >= W && s.dc >= W;
        wide = wide && s.da % W == 0 && s.dc % W == 0 && aligned(s.out.data, 16) && s.out.st % 4 == 0 && s.out.sn % 4 == 0 && s.out.sh % 4 == 0;
        for (const Rows* r : {&s.a, &s.b, &s.c}) wide = wide && aligned(r->data, 16) && r->st % W == 0 && r->sn % W == 0 && r->sh % W == 0;
    }
    if (wide) return scan_mode<T, CH, DA, DC, 2>(w, swapped, stream);
    return packs ? scan_mode<T, CH, DA, DC, 1>(w, swapped, stream) : scan_mode<T, CH, DA, DC, 0>(w, swapped, stream);
}

template <class T, int DA, int DC>
int scan_columns(const Walks& w, bool swapped, hipStream_t stream) {
    if constexpr (LONG_CHUNKS<T, DA, DC>)
        if (w.walk[0].steps > 32) return scan_aligned<T, 64, DA, DC>(w, swapped, stream);
    return scan_aligned<T, 32, DA, DC>(w, swapped, stream);
}

template <class T, int DA>
int scan_rows(const Walks& w, bool swapped, hipStream_t stream) {
    const int dc = w.walk[0].dc;
    if (dc <= 32) return scan_columns<T, DA, 32>(w, swapped, stream);
    if (dc <= 64) return scan_columns<T, DA, 64>(w, swapped, stream);
    return scan_columns<T, DA, 128>(w, swapped, stream);
}

template int scan_rows<LOBPOLICY_TYPE, LOBPOLICY_ROWS>(const Walks&, bool, hipStream_t);

}  // namespace lobpolicy
