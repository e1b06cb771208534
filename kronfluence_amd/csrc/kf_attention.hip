// kf_attention.hip -- attention over whole prompts, forward and backward (see include/kronfluence_hip.h, "Model passes").
//
// Mathematics (per sequence and head; c = scale * log2 e):
//     s_ij = q_i . k_j          p_ij = 2^(c s_ij - L_i)      L_i = log2 sum_j 2^(c s_ij)      o_i = sum_j p_ij v_j
//     D_i = do_i . o_i          ds_ij = p_ij (do_i . v_j - D_i)
//     dq_i = scale sum_j ds_ij k_j     dk_j = scale sum_i ds_ij q_i     dv_j = sum_i p_ij do_i
// j runs over the visible keys of i.  The heads of a group share k and v; their dk, dv are summed in registers (no atomics: the
// result does not depend on the order in which workgroups run).
//
// One pass over the keys with a running maximum and sum: the scores never leave the registers.  Every product is a 32 x 32 matrix
// instruction tile with the LANE as the row that owns softmax statistics:
//     forward, dQ:  S^T = K Q^T  (lane = query, registers = keys)   ->  O^T += V^T P^T,   dQ^T += K^T dS^T
//     dK / dV:      S   = Q K^T  (lane = key,  registers = queries) ->  dV^T += dO^T P,   dK^T += Q^T dS
// The accumulator layout (register r of lane half h holds row 8 (r / 4) + 4 h + r % 4) IS the operand layout of the second product
// once the contraction index is permuted the same way in its other operand, so P and dS go from accumulator to operand by
// conversion alone, with no cross-lane traffic; the other operand is read from LDS column-wise (ds_read_b64_tr_b16).
//
// fp32 runs on the same bf16 instructions: every value is split into three bf16 parts, exactly, and a product is six products of parts
// (struct Split) -- 6/16 of the time of v_mfma_f32_32x32x2_f32 at fp32's accuracy.  Measured against that instruction in the same
// kernels: 64 x 256 x 12 heads x 64, forward 131 to 84 us, backward 470 to 325; 2 x 2048 x 16 x 128 causal, 334 to 223 and 1129 to 817.
// Infinities, and finite values from 3.39e38 on (their first part rounds to infinity), give NaN (inf - inf in the split); parts below 2^-126
// count as 0.
//
// Measured (us; causal but for the first; forward, dq, dk / dv): bf16 256 x <= 128 x 12 heads x 64, padded: 38, all of the backward 83 (latency
// of one-tile sequences); 64 x 512 x 12 x 64: 68, 86, 97 and 16 x 512 x 32/8 x 128: 80, 114, 126 (vector instructions of the
// softmax, few rounds of tiles); 1 x 8192 x 32/8 x 128: 575 (956 TFLOP/s), 757, 1070 + 28; fp32 24 x 29..233 x 12 x 64: 27, 36, 44 (few, uneven
// workgroups).  The low bytes of o cost the forward pass 7 and dq 6 us of the second of these.
//
// Roundings to fewer bits than 32, all with bf16 inputs: P and dS as operands of their second product (half a step, at most 2^-8 of a term
// of a sum whose inputs carry the same rounding), and the outputs once at the end.  Maxima, sums, L, D and all accumulators are fp32.
// Neither rounding may enter D, which a peaked row's gradients are far below (a key that outweighs all others: p -> 1, ds -> 0).  So o is
// divided by the sum of the ROUNDED p, and the forward pass keeps the next eight bits of o (at most 2^-15 of it is left): with e_j the
// relative error of p_j, do_i . o_i is then off by sum_j p_j (e_j - sum_k p_k e_k) do_i . v_j = sum_j e_j ds_j, no more than dS's own rounding.
// Measured against 64 bits, dq as a part of its norm (with the rounded o over the sum of p in brackets): 128 keys, scores with a standard deviation of
// 12, 0.24 % (0.64); one key 10 above 511 others 0.24 % (1.6), 20 above 1.7 % (57; what is left is fp32's); usual scores 0.24 % (0.24).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "../../include/kronfluence_hip.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int THREADS = 256;      // 4 waves
constexpr int ROWS = 128;         // rows (queries; keys in the dK / dV kernel) of a workgroup: 32 per wave
constexpr float SLACK = 8.0f;     // the sum of n terms stays below 2^8 n
constexpr float LOG2E = 1.44269504088896340736f;

struct Tensor {   // [batch][token][head][width], the width contiguous; strides in elements
    const void* p;
    int64_t batch, token, head;
};

struct Args {
    Tensor q, k, v, o, g;          // g: the gradient of o
    Tensor dq, dk, dv;
    Tensor rest;                   // [heads][rows][rest_width(width)]: the low byte of o (see Low); or null
    float* lse;                    // [heads][rows]: L
    float* delta;                  // [heads][rows]: D
    float* partial;                // [parts][dk, dv][kv_heads][rows][width], if the dk / dv kernel's work is split (parts > 1)
    int parts;
    const int32_t* lengths;        // per sequence (padded batch), or null
    const int32_t* offsets;        // [sequences + 1] (packed batch), or null
    const int32_t* order;          // [slots]: the tile slots by falling cost (packed batch), or null
    int64_t rows;                  // token rows in all: batch * length, or the packed total
    int sequences, length;         // length: token rows per sequence (padded batch)
    int heads, group, width, causal;
    int slots;                     // tile slots of all sequences
    int chunk;                     // tile slots that go to one XCD together
    float scale;
};

// ---- element types ---------------------------------------------------------------------------------------------------------
// fp32 whose products are sums of bf16 products: every value is exactly the sum of three bf16 parts (8 + 8 + 8 bits), and of the nine
// products of parts the six greater ones are taken.  Part 1 is at most 2^-8 of the value's power of two and part 2 2^-17, so that the three left
// out come to 2^-24 of the product at most, as one more rounding of it would (below 2^-26 for 97 % of random pairs).
struct Split { float value; };

template <class T>
struct Type;
template <class T> constexpr int PARTS = std::is_same_v<T, Split> ? 3 : 1;    // bf16 images of a tile in LDS

template <>
struct Type<__bf16> {
    typedef __bf16 Memory;
    typedef bf16x8 Frag;                       // 16 bytes: the lane's part of a 16-deep contraction slab
    static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ Frag from_acc(const f32x16& s, int slab) {
        Frag f;
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = static_cast<__bf16>(s[8 * slab + i]);
        return f;
    }
    static __device__ __forceinline__ void store4(void* p, float a, float b, float c, float d) {
        bf16x4 v = {static_cast<__bf16>(a), static_cast<__bf16>(b), static_cast<__bf16>(c), static_cast<__bf16>(d)};
        *reinterpret_cast<bf16x4*>(p) = v;
    }
    static __device__ __forceinline__ float dot(Frag a, Frag b, float acc) {
#pragma unroll
        for (int i = 0; i < 8; ++i) acc = fmaf(static_cast<float>(a[i]), static_cast<float>(b[i]), acc);
        return acc;
    }
    static __device__ __forceinline__ float total(Frag a, float acc) {   // two elements an instruction
        typedef __bf16 Pair __attribute__((ext_vector_type(2)));
        const Pair one = {static_cast<__bf16>(1.0f), static_cast<__bf16>(1.0f)};
#pragma unroll
        for (int i = 0; i < 8; i += 2) acc = __builtin_amdgcn_fdot2_f32_bf16(Pair{a[i], a[i + 1]}, one, acc, false);
        return acc;
    }
};

template <>
struct Type<float> {                           // (the partial sums of the dk / dv kernel)
    static __device__ __forceinline__ void store4(void* p, float a, float b, float c, float d) {
        f32x4 v = {a, b, c, d};
        *reinterpret_cast<f32x4*>(p) = v;
    }
};

// The eight bits of a float below its rounding to bf16, signed: the two together are a float of 16 significant bits.  (Bit patterns of floats
// ascend with their magnitude, so that the difference needs no look at the exponent.)
struct Low {
    int8_t byte;
    // The low halves of two floats as signed numbers are what their roundings leave off, but for the tie 0x8000 that rounds down (to an even
    // high half): one less there, and anywhere the high half is even, is 0x7fff.  Rounded to a byte with saturation, in the byte's place.
    static __device__ __forceinline__ uint32_t two(float x, float y) {
        const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
        const uint32_t low = __builtin_amdgcn_perm(b, a, 0x05040100), even = ~__builtin_amdgcn_perm(b, a, 0x07060302) & 0x00010001;
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_add_sat(__builtin_bit_cast(s16x2, low) - __builtin_bit_cast(s16x2, even), s16x2{0x80, 0x80}));
    }
    static __device__ __forceinline__ float join(__bf16 high, uint32_t low, int byte) {   // byte `byte` of `low`
        return __uint_as_float((static_cast<uint32_t>(__builtin_bit_cast(uint16_t, high)) << 16) + ((static_cast<int32_t>(low << (24 - 8 * byte)) >> 24) << 8));
    }
};
__host__ __device__ constexpr int64_t rest_width(int64_t width) { return (width + 15) / 16 * 16; }   // (stored 16 bytes at a time)

template <>
struct Type<Low> {
    static __device__ __forceinline__ void store4(void* p, float a, float b, float c, float d) {
        *reinterpret_cast<uint32_t*>(p) = __builtin_amdgcn_perm(Low::two(c, d), Low::two(a, b), 0x07050301);
    }
};

template <>
struct Type<Split> {
    typedef float Memory;
    struct Frag { bf16x8 part[3]; };           // a 16-deep slab; the parts from the greatest on
    static __device__ __forceinline__ f32x16 mma(const Frag& a, const Frag& b, f32x16 c) {
        c = Type<__bf16>::mma(a.part[2], b.part[0], c);
        c = Type<__bf16>::mma(a.part[0], b.part[2], c);
        c = Type<__bf16>::mma(a.part[1], b.part[1], c);
        c = Type<__bf16>::mma(a.part[1], b.part[0], c);
        c = Type<__bf16>::mma(a.part[0], b.part[1], c);
        return Type<__bf16>::mma(a.part[0], b.part[0], c);
    }
    // x = part 0 + part 1 + part 2 exactly: each part is the nearest bf16 to what the ones before leave, and the differences are exact
    template <class Values>
    static __device__ __forceinline__ Frag split(const Values& x, int first) {
        Frag f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            f.part[0][i] = static_cast<__bf16>(x[first + i]);
            const float rest = x[first + i] - static_cast<float>(f.part[0][i]);
            f.part[1][i] = static_cast<__bf16>(rest);
            f.part[2][i] = static_cast<__bf16>(rest - static_cast<float>(f.part[1][i]));
        }
        return f;
    }
    static __device__ __forceinline__ Frag from_acc(const f32x16& s, int slab) { return split(s, 8 * slab); }
    static __device__ __forceinline__ Frag from_memory(u32x4 low, u32x4 high) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = __uint_as_float(low[i]);
            x[4 + i] = __uint_as_float(high[i]);
        }
        return split(x, 0);
    }
    static __device__ __forceinline__ void store4(void* p, float a, float b, float c, float d) { Type<float>::store4(p, a, b, c, d); }
    static __device__ __forceinline__ float dot(const Frag& a, const Frag& b, float acc) {
        auto value = [](const Frag& f, int i) {
            return static_cast<float>(f.part[2][i]) + static_cast<float>(f.part[1][i]) + static_cast<float>(f.part[0][i]);   // exact again
        };
#pragma unroll
        for (int i = 0; i < 8; ++i) acc = fmaf(value(a, i), value(b, i), acc);
        return acc;
    }
};

// ---- an operand tile of N rows in LDS: [64-byte column block][row][4 chunks of 16 bytes], the chunk XORed with (row / 4) % 4 -----
// (fp32: one such image per part).  Two kinds of reads meet the same image.  Row fragments: 32 consecutive rows, one chunk each -- any 16 consecutive rows fall into the
// 16 different slots of the 256-byte bank space.  Transposed reads: 4 consecutive rows, 64 bytes each -- 256
// consecutive bytes.  The address of any other slab, block or half differs by a constant of the instruction, but for one bit that
// changes by exclusive or: a lane keeps one register per kind of read.
template <class T, int DP, int N>
struct Image {
    static constexpr int CHUNKS = DP / 8, SLABS = CHUNKS / 2;
    static constexpr int BLOCK = N * 64, PART = CHUNKS / 4 * BLOCK, BYTES = PARTS<T> * PART;
};

template <class T, int DP, int N>
struct Reader {
    typedef Image<T, DP, N> Img;
    typedef __attribute__((address_space(3))) const bf16x8* FragPointer;
    uint32_t row, column;
    __device__ __forceinline__ explicit Reader(int lane) {
        const int r = lane & 31, g = lane >> 4, s = lane & 15;
        row = r * 64 + (((lane >> 5) ^ (r >> 2)) & 3) * 16;
        column = (4 * (g >> 1) + (s >> 2)) * 64 + ((2 * (g & 1) + ((s & 3) >> 1)) ^ (g >> 1)) * 16 + (s & 1) * 8;
    }
    // rows row0 .. row0 + 31 of the tile at LDS address `tile` (row0 a multiple of 32), contraction slab `slab`
    __device__ __forceinline__ bf16x8 rows(uint32_t tile, int row0, int slab) const {
        return *reinterpret_cast<FragPointer>(((tile + row) ^ (slab % 2 * 32)) + slab / 2 * Img::BLOCK + row0 * 64);
    }
    // the TRANSPOSED tile: columns 32 t .. 32 t + 31 as rows, contraction over the tile rows that registers [8 slab, 8 (slab + 1)) of an
    // accumulator over rows row0 .. row0 + 31 stand for
    __device__ __forceinline__ bf16x8 columns(uint32_t tile, int row0, int slab, int t) const {
        union { s16x4 h[2]; bf16x8 v; } u;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            u.h[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<__attribute__((address_space(3))) s16x4*>(
                ((tile + column) ^ (32 * i)) + t * Img::BLOCK + (row0 + 16 * slab + 8 * i) * 64));
        return u.v;
    }
};

template <int DP, int N>
struct Reader<Split, DP, N> : Reader<__bf16, DP, N> {   // one image per part
    typedef Reader<__bf16, DP, N> Base;
    typedef typename Type<Split>::Frag Frag;
    static constexpr int PART = Image<Split, DP, N>::PART;
    using Base::Base;
    __device__ __forceinline__ Frag rows(uint32_t tile, int row0, int slab) const {
        return Frag{{Base::rows(tile, row0, slab), Base::rows(tile + PART, row0, slab), Base::rows(tile + 2 * PART, row0, slab)}};
    }
    __device__ __forceinline__ Frag columns(uint32_t tile, int row0, int slab, int t) const {
        return Frag{{Base::columns(tile, row0, slab, t), Base::columns(tile + PART, row0, slab, t), Base::columns(tile + 2 * PART, row0, slab, t)}};
    }
};

__device__ __forceinline__ uint32_t lds_address(const void* p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const void*)p));
}

// Rows of one head of one sequence as a buffer: a load behind the last row, or of a column behind the head width, returns 0 without
// touching memory -- what stands there may be anything, and its weight is 0.  The descriptor is rebuilt per tile (scalar
// arithmetic), so that the 32-bit offsets span one tile only.
constexpr uint32_t NO_COLUMN = 0x80000000u;         // an offset no descriptor reaches
constexpr int64_t MAX_RECORDS = 0x7fffffff;
struct Rows {
    const char* base;
    int64_t token;     // bytes between rows
    int length, width; // rows; bytes of a row
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t from(int row0) const {
        const int64_t bytes = (length - row0 - 1) * token + width;
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base + row0 * token), 0, row0 < length ? static_cast<int>(min(bytes, MAX_RECORDS)) : 0,
                                                 0x00020000);
    }
};

// N rows of a tile into registers (every thread a few 16-byte chunks: four threads a 64-byte piece of a row), and from there to LDS,
// where the n-th chunk of the workgroup goes to byte 16 n but for the exclusive or.
template <class T, int DP, int N>
struct Stage {
    typedef Image<T, DP, N> Img;
    static constexpr int ALL = Img::BYTES / 16, PER = (ALL + THREADS - 1) / THREADS;
    u32x4 r[PER];
    uint32_t at[PER];   // byte offsets of the thread's chunks inside a tile in memory
    int to;             // byte offset of the first one in LDS; the others follow every 16 THREADS bytes
    __device__ __forceinline__ Stage(int64_t token, int width, int tid) {
        to = (tid * 16) ^ ((tid >> 4 & 3) * 16);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int n = tid + i * THREADS, row = n / 4 % N, chunk = n / 4 / N * 4 + n % 4;
            at[i] = chunk * 16 < width ? static_cast<uint32_t>(row * static_cast<int>(token) + chunk * 16) : NO_COLUMN;
        }
    }
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rows) {
#pragma unroll
        for (int i = 0; i < PER; ++i) r[i] = __builtin_amdgcn_raw_buffer_load_b128(rows, at[i], 0, 0);
    }
    __device__ __forceinline__ void store(char* tile) const {
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (ALL % THREADS == 0 || i + 1 < PER || to + i * 16 * THREADS < Img::BYTES) *reinterpret_cast<u32x4*>(tile + to + i * 16 * THREADS) = r[i];
    }
};

// fp32 rows into the images of their parts: 8 values a chunk.
template <int DP, int N>
struct Stage<Split, DP, N> {
    typedef Image<Split, DP, N> Img;
    static constexpr int ALL = Img::PART / 16, PER = (ALL + THREADS - 1) / THREADS;
    u32x4 r[PER][2];
    uint32_t at[PER][2];
    int to;
    __device__ __forceinline__ Stage(int64_t token, int width, int tid) {
        to = (tid * 16) ^ ((tid >> 4 & 3) * 16);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int n = tid + i * THREADS, row = n / 4 % N, chunk = n / 4 / N * 4 + n % 4;
#pragma unroll
            for (int j = 0; j < 2; ++j)
                at[i][j] = chunk * 32 + j * 16 < width ? static_cast<uint32_t>(row * static_cast<int>(token) + chunk * 32 + j * 16) : NO_COLUMN;
        }
    }
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rows) {
#pragma unroll
        for (int i = 0; i < PER; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) r[i][j] = __builtin_amdgcn_raw_buffer_load_b128(rows, at[i][j], 0, 0);
    }
    __device__ __forceinline__ void store(char* tile) const {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (ALL % THREADS != 0 && i + 1 == PER && to + i * 16 * THREADS >= Img::PART) continue;
            const Type<Split>::Frag f = Type<Split>::from_memory(r[i][0], r[i][1]);
#pragma unroll
            for (int p = 0; p < 3; ++p) *reinterpret_cast<bf16x8*>(tile + p * Img::PART + to + i * 16 * THREADS) = f.part[p];
        }
    }
};

// ---- which rows a workgroup works on --------------------------------------------------------------------------------------
struct Place {
    int64_t sequence, start;   // batch index; first token row (packed)
    int64_t stat;              // row of lse / delta of the sequence's token 0
    int length, written;       // visible tokens; token rows whose outputs this sequence owns (>= length: the rest is set to 0)
    int row0;                  // first row of the workgroup's tile
};

// Tile slots.  Padded batch: ceil(length / ROWS) per sequence.  Packed batch: sequence s takes slots [c_s / ROWS + s,
// c_{s+1} / ROWS + s + 1) with c the offsets -- at least ceil(len / ROWS) of them, found by a binary search without a table or a
// host copy of the offsets; the rows behind the last sequence are one more sequence of no visible tokens.  So are the rows in front of
// the first one: they take the slots below c_0 / ROWS, and their last, partial tile the slot behind all others.  Offsets outside
// [0, rows] are clamped, so that no content of the offsets can send an access out of bounds.
__device__ __forceinline__ bool locate(const Args& a, int slot, bool last_first, Place& w) {
    if (a.offsets == nullptr) {
        const int tiles = (a.length + ROWS - 1) / ROWS, s = slot / tiles, t = slot - s * tiles;
        w.sequence = s; w.start = 0; w.stat = static_cast<int64_t>(s) * a.length;
        w.written = a.length;
        w.length = a.lengths ? min(max(a.lengths[s], 0), a.length) : a.length;
        w.row0 = (last_first ? tiles - 1 - t : t) * ROWS;
        return true;
    }
    const int total = static_cast<int>(a.rows);
    auto offset = [&](int s) { return s > a.sequences ? total : min(max(a.offsets[s], 0), total); };
    auto first_slot = [&](int s) { return offset(s) / ROWS + s; };
    const int front = offset(0);
    if (slot < front / ROWS || slot == total / ROWS + a.sequences + 1) {
        w.sequence = 0; w.start = 0; w.stat = 0;
        w.written = front;
        w.length = 0;
        w.row0 = min(slot, front / ROWS) * ROWS;
        return w.row0 < front;
    }
    int lo = 0, hi = a.sequences;   // first_slot(lo) <= slot; the last such
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first_slot(mid) <= slot) lo = mid; else hi = mid - 1;
    }
    const int begin = offset(lo), rows = max(offset(lo + 1) - begin, 0);
    int t = slot - first_slot(lo);
    const int tiles = (rows + ROWS - 1) / ROWS;
    if (t < 0 || t >= tiles) return false;
    if (last_first) t = tiles - 1 - t;
    w.sequence = 0; w.start = begin; w.stat = begin;
    w.written = rows;
    w.length = lo == a.sequences ? 0 : rows;
    w.row0 = t * ROWS;
    return true;
}

// Workgroup -> (slot, kv_head, member of its group).  Consecutive workgroup ids go to the eight XCDs in turn, and each has an L2 of its
// own: what reads the same k and v should go to one XCD, but no XCD may be left with the longest sequences.  Where (sequence, key /
// value head) pairs of equal size are many, whole pairs are dealt to the XCDs (a.chunk = the tiles of a sequence), the heads of a
// sequence one after the other (24 sequences of 29 to 233 tokens, 12 heads x 64, in fp32 products: 210 us, 264 with the sequences of a
// head one after the other).  An XCD deals its workgroups to its compute units in turn, too, and the tiles of a pair are of very different cost, if
// causal.  So the pairs of an XCD are worked on in blocks of about BLOCK_UNITS, the first (dearest) tiles of all pairs of a block first:
// pair after pair, every unit would get the same tile each time, and the last dear tiles would start last (causal bf16: 64 x 512 x 12
// heads x 64, dk / dv 121 us pair after pair, 98 in blocks; 4 x 2048 x 16 x 64, forward 77 and 53, backward 215 and 158).  In larger
// blocks k and v leave the L2 (the first of these with 32 pairs a block: 102).
// Otherwise single tiles are dealt, the heads of a tile one after the other: with 1, 2, 4 or a multiple of 8 heads an XCD then sees the
// same heads in every tile.  The `members` query heads of a group stay together.  False: nothing left (the grid is rounded up).
constexpr int XCDS = 8, BLOCK_UNITS = 16;
struct Item { int slot, kv_head, member; };
__device__ __forceinline__ bool work_item(const Args& a, int members, Item& w) {
    const int kv_heads = a.heads / a.group, id = static_cast<int>(blockIdx.x), n = id / XCDS;
    const int items = a.chunk * members, units = static_cast<int>(gridDim.x) / (XCDS * items);   // (of an XCD; the grid is a multiple)
    const int blocks = (units + BLOCK_UNITS - 1) / BLOCK_UNITS, most = (units + blocks - 1) / blocks;   // units of a block
    const int block = n / (most * items) * most, here = min(most, units - block), in = n - block * items;
    const int tile = in / (here * members), rest = in % (here * members);
    const int64_t unit = static_cast<int64_t>(block + rest / members) * XCDS + id % XCDS;
    w.member = rest % members;
    w.kv_head = static_cast<int>(unit % kv_heads);
    w.slot = static_cast<int>(unit / kv_heads * a.chunk + tile);
    if (unit * a.chunk + tile >= static_cast<int64_t>(a.slots) * kv_heads) return false;
    if (a.order && w.slot < a.slots - 1) w.slot = a.order[w.slot];   // (the last slot, of the rows in front, is not among those ordered)
    return true;
}

// The slots of a packed batch by falling cost: documents come in any order, and a long one whose tiles start last leaves the card
// waiting for it (24 documents of 12011 tokens, 16/4 heads x 128 bf16: forward 101 us in the
// order they come, 85 in this one; dq 131 and 123, dk / dv 183 and 152).  The cost of a slot is that of its tile in the kernels over
// queries (last tiles first) and in the one over keys (first tiles first) alike: the tiles of its sequence it meets.
// One workgroup: a histogram of costs, places from the highest down; the order inside a cost is of no consequence.
constexpr int COSTS = 2048, MAX_ORDERED = 16384;
__global__ __launch_bounds__(1024) void attention_order_kernel(const Args a, int32_t* order) {
    __shared__ int place[COSTS], sums[1024];
    auto cost_of = [&](int slot) {
        Place w;
        if (!locate(a, slot, false, w) || w.length == 0) return 0;
        const int tiles = (w.length + ROWS - 1) / ROWS;
        return min(a.causal ? tiles - w.row0 / ROWS : tiles, COSTS - 1);
    };
    for (int i = threadIdx.x; i < COSTS; i += 1024) place[i] = 0;
    __syncthreads();
    for (int s = threadIdx.x; s < a.slots; s += 1024) atomicAdd(&place[cost_of(s)], 1);
    __syncthreads();
    // thread t: costs COSTS - 1 - 2 t and the next lower one; sums[t]: the slots of all higher costs
    const int high = COSTS - 1 - 2 * threadIdx.x, n0 = place[high], n1 = place[high - 1];
    sums[threadIdx.x] = n0 + n1;
    __syncthreads();
    for (int step = 1; step < 1024; step *= 2) {
        const int other = threadIdx.x >= step ? sums[threadIdx.x - step] : 0;
        __syncthreads();
        sums[threadIdx.x] += other;
        __syncthreads();
    }
    const int before = sums[threadIdx.x] - n0 - n1;
    place[high] = before;
    place[high - 1] = before + n0;
    __syncthreads();
    for (int s = threadIdx.x; s < a.slots; s += 1024) order[atomicAdd(&place[cost_of(s)], 1)] = s;
}

// Offsets as the kernels above take them: clamped to the rows, and none below one before it.  One workgroup, a running maximum.
__global__ __launch_bounds__(1024) void attention_starts_kernel(int32_t* starts, const void* offsets, bool wide, int64_t count, int64_t rows) {
    __shared__ int top[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int before = 0;   // the maximum of all earlier offsets
    for (int64_t base = 0; base < count; base += 1024) {
        const int64_t i = base + threadIdx.x;
        int x = 0;
        if (i < count) {
            const int64_t given = wide ? reinterpret_cast<const int64_t*>(offsets)[i] : reinterpret_cast<const int32_t*>(offsets)[i];
            x = static_cast<int>(min(max(given, int64_t{0}), rows));
        }
#pragma unroll
        for (int step = 1; step < 64; step *= 2) {
            const int other = __shfl_up(x, step);
            if (lane >= step) x = max(x, other);
        }
        if (lane == 63) top[wave] = x;
        __syncthreads();
        for (int n = 0; n < 16; ++n) {
            if (n == wave) x = max(x, before);
            before = max(before, top[n]);   // (for every wave that of the whole block in the end)
        }
        if (i < count) starts[i] = x;
        __syncthreads();
    }
}

template <class T>
__device__ __forceinline__ const T* rows_of(const Tensor& t, const Place& w, int head) {
    return reinterpret_cast<const T*>(t.p) + w.sequence * t.batch + w.start * t.token + head * t.head;
}
template <class T>
__device__ __forceinline__ Rows input_rows(const Args& a, const Tensor& t, const Place& w, int head) {
    return Rows{reinterpret_cast<const char*>(rows_of<T>(t, w, head)), t.token * static_cast<int64_t>(sizeof(T)), w.length,
                a.width * static_cast<int>(sizeof(T))};
}
template <class T>
__device__ __forceinline__ T* rows_out(const Tensor& t, const Place& w, int head) { return const_cast<T*>(rows_of<T>(t, w, head)); }

// the value of lane ^ 32
__device__ __forceinline__ float other_half(float x) {
    const auto swapped = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(threadIdx.x & 32 ? swapped[0] : swapped[1]);
}

// The fragments of 32 rows straight from memory (lane & 31 = row): the operand a wave keeps for the whole kernel.
template <class T, int DP>
struct Held {
    static constexpr int SLABS = DP * static_cast<int>(sizeof(T)) / 32;
    typename Type<T>::Frag f[SLABS];
    __device__ __forceinline__ void load(const Rows& rows, int row0, int lane) {
        const __amdgpu_buffer_rsrc_t from = rows.from(row0);
#pragma unroll
        for (int s = 0; s < SLABS; ++s) {
            const int c = 2 * s + (lane >> 5);
            union { u32x4 u; typename Type<T>::Frag f; } v;
            v.u = __builtin_amdgcn_raw_buffer_load_b128(
                from, c * 16 < rows.width ? static_cast<uint32_t>((lane & 31) * static_cast<int>(rows.token) + c * 16) : NO_COLUMN, 0, 0);
            f[s] = v.f;
        }
    }
};

template <int DP>
struct Held<Split, DP> {
    static constexpr int SLABS = DP / 16;
    typename Type<Split>::Frag f[SLABS];
    __device__ __forceinline__ void load(const Rows& rows, int row0, int lane) {
        const __amdgpu_buffer_rsrc_t from = rows.from(row0);
        auto piece = [&](int byte) {
            return __builtin_amdgcn_raw_buffer_load_b128(
                from, byte < rows.width ? static_cast<uint32_t>((lane & 31) * static_cast<int>(rows.token) + byte) : NO_COLUMN, 0, 0);
        };
#pragma unroll
        for (int s = 0; s < SLABS; ++s) {
            const int c = (2 * s + (lane >> 5)) * 32;
            f[s] = Type<Split>::from_memory(piece(c), piece(c + 16));
        }
    }
};

// acc^T (lane = row, registers = columns d) times the lane's `factor` -> rows first .. first + 31 of memory, through LDS: a lane holds
// four columns of a row at a time, and stores of 8 bytes per row cost as much as all the rest of a short sequence (256 x 128 x 12 x 64
// bf16 forward: 43 us, 22 without the stores).  Every wave uses its own piece of `scratch`; the workgroup is done with its tiles.
template <class S, int DP>
struct Pass {   // the columns of one pass: up to 256 bytes of a row, rows 16 bytes further apart in LDS
    static constexpr int COLUMNS = std::min(256 / static_cast<int>(sizeof(S)), DP), STRIDE = COLUMNS * static_cast<int>(sizeof(S)) + 16;
    static constexpr int SCRATCH = ROWS * STRIDE;
};
template <class S, int DP>
__device__ __forceinline__ void store_rows(const f32x16 (&acc)[DP / 32], char* scratch, S* base, int64_t token, int first, int written, int width,
                                           float factor, int wave, int lane) {
    constexpr int COLUMNS = Pass<S, DP>::COLUMNS, STRIDE = Pass<S, DP>::STRIDE;
    constexpr int CHUNKS = COLUMNS * static_cast<int>(sizeof(S)) / 16, PER = 16 / static_cast<int>(sizeof(S));
    char* own = scratch + wave * 32 * STRIDE;
    asm volatile("" : "+v"(lane));   // addresses are made here, not kept in registers across the caller's loop
#pragma unroll
    for (int c0 = 0; c0 < DP; c0 += COLUMNS) {
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int t = c0 / 32; t < (c0 + COLUMNS < DP ? c0 + COLUMNS : DP) / 32; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                Type<S>::store4(own + (lane & 31) * STRIDE + (32 * t - c0 + 8 * i + 4 * (lane >> 5)) * static_cast<int>(sizeof(S)),
                                acc[t][4 * i] * factor, acc[t][4 * i + 1] * factor, acc[t][4 * i + 2] * factor, acc[t][4 * i + 3] * factor);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < 32 * CHUNKS / 64; ++i) {
            const int n = lane + 64 * i, row = n / CHUNKS, d = c0 + n % CHUNKS * PER;
            const u32x4 v = *reinterpret_cast<const u32x4*>(own + row * STRIDE + n % CHUNKS * 16);
            if (first + row < written && d < width) *reinterpret_cast<u32x4*>(base + (first + row) * token + d) = v;
        }
    }
}

template <class T, int DP, int N_THREADS = THREADS>
__device__ __forceinline__ void zero_rows(T* base, int64_t token, int row0, int written, int width, int tid) {
    constexpr int PER = 16 / static_cast<int>(sizeof(T));
    const int chunks = width / PER;
    for (int n = tid; n < ROWS * chunks; n += N_THREADS) {
        const int row = row0 + n / chunks;
        if (row < written) *reinterpret_cast<u32x4*>(base + row * token + (n % chunks) * PER) = u32x4{0, 0, 0, 0};
    }
}

// A read of a matrix instruction's result needs wait states that the compiler inserts; where a branch stands between the two it has
// left some out on one of the paths (the first read behind the branch then sees the last row of the tile before it was written).  Put
// between the last matrix instruction and such a branch; tests/test_wait_states_cpu.py follows every path of the built code and says where.
__device__ __forceinline__ void settle() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 11");
    __builtin_amdgcn_sched_barrier(0);
}

// ---- forward ------------------------------------------------------------------------------------------------------------
template <class T, int DP, int BK, int WAVES>
__global__ __launch_bounds__(THREADS, WAVES) void attention_forward_kernel(const Args a) {
    typedef Image<T, DP, BK> Img;
    typedef typename Type<T>::Frag Frag;
    constexpr int TILE = Img::BYTES;
    extern __shared__ __align__(16) char lds[];   // [2][k tile, v tile]

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    Item item;
    Place w;
    if (!work_item(a, a.group, item) || !locate(a, item.slot, a.causal, w)) return;
    const int kv_head = item.kv_head, head = kv_head * a.group + item.member;
    T* o = rows_out<T>(a.o, w, head);
    float* lse = a.lse ? a.lse + head * a.rows + w.stat : nullptr;
    if (w.row0 >= w.length) {
        zero_rows<T, DP>(o, a.o.token, w.row0, w.written, a.width, tid);
        if (lse && tid < ROWS && w.row0 + tid < w.written) lse[w.row0 + tid] = INFINITY;
        return;
    }
    const Rows k = input_rows<T>(a, a.k, w, kv_head), v = input_rows<T>(a, a.v, w, kv_head);
    const int first = w.row0 + 32 * wave, query = first + (lane & 31), half = lane >> 5;

    Held<T, DP> q;
    q.load(input_rows<T>(a, a.q, w, head), first, lane);
    f32x16 acc[DP / 32] = {};
    const float c = a.scale * LOG2E;
    float top = -INFINITY, sum = 0.0f;   // a running reference near the maximum of c s; this half's part of the running sum
    float weight = 0.0f;                 // (bf16: the sum of p as the second product's operand has it)

    const int end = a.causal ? min(w.length, w.row0 + ROWS) : w.length, tiles = (end + BK - 1) / BK;
    Stage<T, DP, BK> sk(k.token, k.width, tid), sv(v.token, v.width, tid);
    const Reader<T, DP, BK> read(lane);
    sk.load(k.from(0));
    sv.load(v.from(0));
    sk.store(lds);
    sv.store(lds + TILE);
    for (int t = 0; t < tiles; ++t) {
        const uint32_t kt = lds_address(lds) + (t & 1) * 2 * TILE, vt = kt + TILE;
        const int k0 = t * BK;
        __syncthreads();   // tile t is written; everybody is done with tile t - 1, whose place t + 1 takes below
        if (t + 1 < tiles) {
            sk.load(k.from(k0 + BK));
            sv.load(v.from(k0 + BK));
        }
        if (first < w.length && !(a.causal && k0 > first + 31)) {   // (wave-uniform)
            f32x16 s[BK / 32];
#pragma unroll
            for (int b = 0; b < BK / 32; ++b) {
                s[b] = f32x16{};
#pragma unroll
                for (int i = 0; i < Img::SLABS; ++i) s[b] = Type<T>::mma(read.rows(kt, 32 * b, i), q.f[i], s[b]);
            }
            settle();
            if (k0 + BK > w.length || (a.causal && k0 + BK - 1 > first)) {
                const int visible = a.causal ? min(w.length, query + 1) : w.length;
#pragma unroll
                for (int b = 0; b < BK / 32; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (k0 + 32 * b + 8 * (r / 4) + 4 * half + r % 4 >= visible) s[b][r] = -INFINITY;
            }
            float m = s[0][0];
#pragma unroll
            for (int b = 0; b < BK / 32; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) m = fmaxf(m, s[b][r]);
            m = fmaxf(m, other_half(m)) * c;
            // any reference does that keeps 2^(c s - top) in range: it moves up only when a row has outgrown it by 2^SLACK
            if (__any(m > top + SLACK)) {
                const float now = fmaxf(top, m), shrink = __builtin_amdgcn_exp2f(top - now);   // (m is finite where it is greater)
                if (m > top + SLACK) {
                    sum *= shrink;
                    weight *= shrink;
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d) acc[d] *= shrink;
                    top = now;
                }
            }
            const float base = top == -INFINITY ? 0.0f : top;   // (a row with no finite score yet)
#pragma unroll
            for (int b = 0; b < BK / 32; ++b) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[b][r] = __builtin_amdgcn_exp2f(fmaf(s[b][r], c, -base));
                    sum += s[b][r];
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const Frag p = Type<T>::from_acc(s[b], i);
                    if constexpr (PARTS<T> == 1) weight = Type<T>::total(p, weight);
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d) acc[d] = Type<T>::mma(read.columns(vt, 32 * b, i, d), p, acc[d]);
                }
            }
        }
        if (t + 1 < tiles) {
            sk.store(lds + ((t + 1) & 1) * 2 * TILE);
            sv.store(lds + ((t + 1) & 1) * 2 * TILE + TILE);
        }
    }
    sum += other_half(sum);
    weight = PARTS<T> == 1 ? weight + other_half(weight) : sum;
    const bool real = query < w.length;
    const float by = 1.0f / weight;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) acc[d] = real ? acc[d] * by : f32x16{};   // (a real token's infinity stays out of the rows of none)
    __syncthreads();
    store_rows<T, DP>(acc, lds, o, a.o.token, first, w.written, a.width, 1.0f, wave, lane);
    if constexpr (PARTS<T> == 1) {
        static_assert(Pass<Low, DP>::STRIDE <= Pass<T, DP>::STRIDE, "in the same piece of the scratch as the wave's rows before");
        if (a.rest.p)
            store_rows<Low, DP>(acc, lds + wave * 32 * (Pass<T, DP>::STRIDE - Pass<Low, DP>::STRIDE), rows_out<Low>(a.rest, w, head), a.rest.token, first,
                                w.length, static_cast<int>(rest_width(a.width)), 1.0f, wave, lane);
    }
    if (lse && half == 0 && query < w.written) lse[query] = real ? top + __builtin_amdgcn_logf(sum) : INFINITY;
}

// ---- backward: dq (and D for the second kernel) ---------------------------------------------------------------------------
template <class T, int DP, int BK, int WAVES>
__global__ __launch_bounds__(THREADS, WAVES) void attention_dq_kernel(const Args a) {
    typedef Image<T, DP, BK> Img;
    typedef typename Type<T>::Frag Frag;
    constexpr int TILE = Img::BYTES;
    extern __shared__ __align__(16) char lds[];   // [2][k tile, v tile]

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    Item item;
    Place w;
    if (!work_item(a, a.group, item) || !locate(a, item.slot, a.causal, w)) return;
    const int kv_head = item.kv_head, head = kv_head * a.group + item.member;
    T* dq = rows_out<T>(a.dq, w, head);
    if (w.row0 >= w.length) {
        zero_rows<T, DP>(dq, a.dq.token, w.row0, w.written, a.width, tid);
        return;   // (D of rows that hold no token is never read)
    }
    const Rows k = input_rows<T>(a, a.k, w, kv_head), v = input_rows<T>(a, a.v, w, kv_head);
    const int first = w.row0 + 32 * wave, query = first + (lane & 31), half = lane >> 5;
    const bool real = query < w.length;

    Held<T, DP> q, g;
    q.load(input_rows<T>(a, a.q, w, head), first, lane);
    g.load(input_rows<T>(a, a.g, w, head), first, lane);
    float delta = 0.0f;
    {
        Held<T, DP> o;
        o.load(input_rows<T>(a, a.o, w, head), first, lane);
        if constexpr (PARTS<T> == 1) {   // (no low bytes: rows of no length, zeros without touching memory)
            const Rows rest{reinterpret_cast<const char*>(rows_of<Low>(a.rest, w, head)), a.rest.token, a.rest.p ? w.length : 0, a.width};
            const __amdgpu_buffer_rsrc_t from = rest.from(first);
            u32x2 low[Img::SLABS];
#pragma unroll
            for (int s = 0; s < Img::SLABS; ++s) {
                const int column = 16 * s + 8 * half;
                low[s] = __builtin_amdgcn_raw_buffer_load_b64(from, column < a.width ? static_cast<uint32_t>((lane & 31) * static_cast<int>(rest.token) + column)
                                                                                     : NO_COLUMN, 0, 0);
            }
#pragma unroll
            for (int s = 0; s < Img::SLABS; ++s)
#pragma unroll
                for (int i = 0; i < 8; ++i) delta = fmaf(Low::join(o.f[s][i], low[s][i / 4], i % 4), static_cast<float>(g.f[s][i]), delta);
        } else {
#pragma unroll
            for (int s = 0; s < Img::SLABS; ++s) delta = Type<T>::dot(o.f[s], g.f[s], delta);
        }
        delta += other_half(delta);
    }
    const int64_t stat = head * a.rows + w.stat;
    const float lse = real ? a.lse[stat + query] : INFINITY;
    const bool alone = first < w.length && (a.causal ? min(w.length, first + 32) : w.length) <= 32;   // (wave-uniform)
    if (half == 0 && real && !alone) a.delta[stat + query] = delta;

    f32x16 acc[DP / 32] = {};
    const float c = a.scale * LOG2E;
    const int end = a.causal ? min(w.length, w.row0 + ROWS) : w.length, tiles = (end + BK - 1) / BK;
    Stage<T, DP, BK> sk(k.token, k.width, tid), sv(v.token, v.width, tid);
    const Reader<T, DP, BK> read(lane);
    sk.load(k.from(0));
    sv.load(v.from(0));
    sk.store(lds);
    sv.store(lds + TILE);
    // Rows whose keys all stand in one block: D as the sum of p dp there, in fp32.  out, which D comes from otherwise, is rounded, and where
    // a row sees few keys its gradients are small beside do . out (two keys, bf16: dq and dk off by 1.4 % of their norm, 0.2 % with it).
    if (w.row0 == 0 && (a.causal || w.length <= 32)) {
        __syncthreads();
        if (alone) {
            const uint32_t kt = lds_address(lds), vt = kt + TILE;
            f32x16 s = {}, dp = {};
#pragma unroll
            for (int i = 0; i < Img::SLABS; ++i) s = Type<T>::mma(read.rows(kt, 0, i), q.f[i], s);
#pragma unroll
            for (int i = 0; i < Img::SLABS; ++i) dp = Type<T>::mma(read.rows(vt, 0, i), g.f[i], dp);
            settle();
            const int visible = a.causal ? min(w.length, query + 1) : w.length;
            delta = 0.0f;
#pragma unroll
            for (int r = 0; r < 16; ++r)
                delta = fmaf(8 * (r / 4) + 4 * half + r % 4 < visible ? __builtin_amdgcn_exp2f(fmaf(s[r], c, -lse)) : 0.0f, dp[r], delta);
            delta += other_half(delta);
            if (half == 0 && real) a.delta[stat + query] = delta;
        }
    }
    for (int t = 0; t < tiles; ++t) {
        const uint32_t kt = lds_address(lds) + (t & 1) * 2 * TILE, vt = kt + TILE;
        const int k0 = t * BK;
        __syncthreads();
        if (t + 1 < tiles) {
            sk.load(k.from(k0 + BK));
            sv.load(v.from(k0 + BK));
        }
        if (first < w.length && !(a.causal && k0 > first + 31)) {
            const bool masked = k0 + BK > w.length || (a.causal && k0 + BK - 1 > first);
            const int visible = a.causal ? min(w.length, query + 1) : w.length;
#pragma unroll
            for (int b = 0; b < BK / 32; ++b) {
                f32x16 s = {}, dp = {};
#pragma unroll
                for (int i = 0; i < Img::SLABS; ++i) s = Type<T>::mma(read.rows(kt, 32 * b, i), q.f[i], s);
#pragma unroll
                for (int i = 0; i < Img::SLABS; ++i) dp = Type<T>::mma(read.rows(vt, 32 * b, i), g.f[i], dp);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, -lse)) * (dp[r] - delta);
                if (masked) {
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (k0 + 32 * b + 8 * (r / 4) + 4 * half + r % 4 >= visible) s[r] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const Frag ds = Type<T>::from_acc(s, i);
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d) acc[d] = Type<T>::mma(read.columns(kt, 32 * b, i, d), ds, acc[d]);
                }
            }
        }
        if (t + 1 < tiles) {
            sk.store(lds + ((t + 1) & 1) * 2 * TILE);
            sv.store(lds + ((t + 1) & 1) * 2 * TILE + TILE);
        }
    }
    // a row that sees one key has p = 1 whatever its score: ds is exactly 0, not the difference of two roundings
    const bool lone = a.causal ? query == 0 : w.length == 1;
    if (!real || lone) {
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) acc[d] = f32x16{};
    }
    __syncthreads();
    store_rows<T, DP>(acc, lds, dq, a.dq.token, first, w.written, a.width, a.scale, wave, lane);
}

// ---- backward: dk and dv --------------------------------------------------------------------------------------------------
// VL: the wave's v fragments are re-read from LDS instead of kept in registers (width 128: two 32 x 128 fp32 accumulators and k alone
// take 160 of the 256 registers a wave has when two share a SIMD).
template <class T, int DP, int BQ, bool VL, int WAVES>
__global__ __launch_bounds__(THREADS, WAVES) void attention_dkv_kernel(const Args a) {
    typedef Image<T, DP, BQ> Img;
    typedef typename Type<T>::Frag Frag;
    constexpr int TILE = Img::BYTES, STAGE = 2 * TILE + 2 * BQ * 4;
    static_assert(STAGE % 64 == 0, "tiles start at multiples of 64 bytes");
    extern __shared__ __align__(16) char lds[];   // [2][q tile, g tile, L of its rows, D of its rows], with VL the workgroup's v rows

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    Item item;
    Place w;
    if (!work_item(a, a.parts, item) || !locate(a, item.slot, false, w)) return;
    const int kv_head = item.kv_head;
    T* dk = rows_out<T>(a.dk, w, kv_head);
    T* dv = rows_out<T>(a.dv, w, kv_head);
    if (w.row0 >= w.length) {
        if (a.parts > 1) return;   // (the joining kernel's)
        zero_rows<T, DP>(dk, a.dk.token, w.row0, w.written, a.width, tid);
        zero_rows<T, DP>(dv, a.dv.token, w.row0, w.written, a.width, tid);
        return;
    }
    const int first = w.row0 + 32 * wave, key = first + (lane & 31), half = lane >> 5;
    const Reader<T, DP, BQ> read(lane);
    const Reader<T, DP, ROWS> read_v(lane);
    const uint32_t own_v = lds_address(lds) + 2 * STAGE + 32 * wave * 64;
    Held<T, DP> k, v;
    k.load(input_rows<T>(a, a.k, w, kv_head), first, lane);
    if constexpr (VL) {
        const Rows rows = input_rows<T>(a, a.v, w, kv_head);
        Stage<T, DP, ROWS> sv(rows.token, rows.width, tid);
        sv.load(rows.from(w.row0));
        sv.store(lds + 2 * STAGE);
    } else {
        v.load(input_rows<T>(a, a.v, w, kv_head), first, lane);
    }
    f32x16 ak[DP / 32] = {}, av[DP / 32] = {};
    const float c = a.scale * LOG2E;

    // The query tiles of the group's heads, one head after the other; the workgroup takes its part of these steps.
    const int begin = a.causal ? w.row0 / BQ : 0, tiles = (w.length + BQ - 1) / BQ - begin;
    const int all = tiles * a.group, from = static_cast<int>(static_cast<int64_t>(all) * item.member / a.parts);
    const int steps = static_cast<int>(static_cast<int64_t>(all) * (item.member + 1) / a.parts) - from;
    int next_head = kv_head * a.group + from / tiles, next_tile = begin + from % tiles;   // the tile to stage next
    Rows q = input_rows<T>(a, a.q, w, next_head), g = input_rows<T>(a, a.g, w, next_head);
    Stage<T, DP, BQ> sq(q.token, q.width, tid), sg(g.token, g.width, tid);
    float stat = 0.0f;   // threads 0 .. BQ-1: L, the next BQ: D, of the staged tile's rows
    auto load = [&] {
        const int q0 = next_tile * BQ;
        sq.load(q.from(q0));
        sg.load(g.from(q0));
        if (tid < 2 * BQ) {
            const int row = q0 + tid % BQ;
            const float* stats = (tid < BQ ? a.lse : a.delta) + next_head * a.rows + w.stat;
            stat = row < w.length ? stats[row] : tid < BQ ? INFINITY : 0.0f;   // L = inf: p = 0 for rows that hold no token
        }
        if (++next_tile == begin + tiles) {
            next_tile = begin;
            if (++next_head < (kv_head + 1) * a.group) {
                q.base += a.q.head * static_cast<int64_t>(sizeof(T));
                g.base += a.g.head * static_cast<int64_t>(sizeof(T));
            }
        }
    };
    auto store = [&](char* at) {
        sq.store(at);
        sg.store(at + TILE);
        if (tid < 2 * BQ) reinterpret_cast<float*>(at + 2 * TILE)[tid] = stat;
    };
    int tile = next_tile;
    if (steps > 0) {
        load();
        store(lds);
    }
    for (int n = 0; n < steps; ++n) {
        const uint32_t qt = lds_address(lds) + (n & 1) * STAGE, gt = qt + TILE;
        const float* lse = reinterpret_cast<const float*>(lds + (n & 1) * STAGE + 2 * TILE);
        const float* delta = lse + BQ;
        const int q0 = tile * BQ;
        if (++tile == begin + tiles) tile = begin;
        __syncthreads();
        if (n + 1 < steps) load();
#pragma unroll
        for (int b = 0; b < BQ / 32; ++b) {
            if (first >= w.length || (a.causal && q0 + 32 * b + 32 <= first)) continue;   // (wave-uniform)
            // s; then dp beside p = 2^(c s - L); then dv beside ds = p (dp - D); then dk
            f32x16 s = {}, dp = {};
#pragma unroll
            for (int i = 0; i < Img::SLABS; ++i) s = Type<T>::mma(read.rows(qt, 32 * b, i), k.f[i], s);
#pragma unroll
            for (int i = 0; i < Img::SLABS; ++i) {
                if constexpr (VL) dp = Type<T>::mma(read.rows(gt, 32 * b, i), read_v.rows(own_v, 0, i), dp);
                else dp = Type<T>::mma(read.rows(gt, 32 * b, i), v.f[i], dp);
            }
            const float* rows_lse = lse + 32 * b + 4 * half;
            const float* rows_delta = delta + 32 * b + 4 * half;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 l4 = *reinterpret_cast<const f32x4*>(rows_lse + 8 * i);
#pragma unroll
                for (int j = 0; j < 4; ++j) s[4 * i + j] = __builtin_amdgcn_exp2f(fmaf(s[4 * i + j], c, -l4[j]));
            }
            // (Split: no branches inside the condition -- the compiler's count of wait states went wrong around one)
            if (PARTS<T> == 3 ? ((a.causal & (q0 + 32 * b < first + 31)) | (w.length == 1)) : ((a.causal && q0 + 32 * b < first + 31) || w.length == 1)) {
                const int hidden = a.causal ? key - q0 - 32 * b - 4 * half : -32;   // rows of the block in front of the key
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (8 * (r / 4) + r % 4 < hidden) s[r] = 0.0f;
                // the first row of a causal sequence, or the only one, sees one key: ds is exactly 0
                if (q0 + 32 * b + 4 * half == 0) dp[0] = rows_delta[0];
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const Frag p = Type<T>::from_acc(s, i);
#pragma unroll
                for (int d = 0; d < DP / 32; ++d) av[d] = Type<T>::mma(read.columns(gt, 32 * b, i, d), p, av[d]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 d4 = *reinterpret_cast<const f32x4*>(rows_delta + 8 * i);
#pragma unroll
                for (int j = 0; j < 4; ++j) dp[4 * i + j] = s[4 * i + j] * (dp[4 * i + j] - d4[j]);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const Frag ds = Type<T>::from_acc(dp, i);
#pragma unroll
                for (int d = 0; d < DP / 32; ++d) ak[d] = Type<T>::mma(read.columns(qt, 32 * b, i, d), ds, ak[d]);
            }
            if constexpr (PARTS<T> == 3 && DP > 64) settle();   // (the accumulators leave their registers where the loop ends)
        }
        if (n + 1 < steps) store(lds + ((n + 1) & 1) * STAGE);
    }
    __syncthreads();
    if (a.parts > 1) {   // (w.stat + key: the token's row among all)
        const int64_t head = a.rows * a.width, kv_heads = a.heads / a.group;
        float* to = a.partial + (static_cast<int64_t>(item.member) * 2 * kv_heads + kv_head) * head + w.stat * a.width;
        store_rows<float, DP>(ak, lds, to, a.width, first, w.length, a.width, a.scale, wave, lane);
        store_rows<float, DP>(av, lds, to + kv_heads * head, a.width, first, w.length, a.width, 1.0f, wave, lane);
        return;
    }
    if (key >= w.length) {
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) { ak[d] = f32x16{}; av[d] = f32x16{}; }
    }
    store_rows<T, DP>(ak, lds, dk, a.dk.token, first, w.written, a.width, a.scale, wave, lane);
    store_rows<T, DP>(av, lds, dv, a.dv.token, first, w.written, a.width, 1.0f, wave, lane);
}

// ---- backward of batches of 33 to ROWS tokens a row: all three gradients at once --------------------------------------------
// One workgroup per (sequence, key / value head).  A wave first owns 32 queries and takes their D from p and dp over all keys; then 32 keys,
// and meets all queries, as in the dk / dv kernel, leaving ds in LDS as [key][query]; then 32 queries again, and dq is the product of two
// transposed reads.  Seven products as in the two kernels, but the inputs are read once and o not at all.  Measured (backward, bf16, causal, 12 heads
// x 64; the two kernels in brackets): 256 x 128 tokens 96 us (132), 512 x 64 112 (140), 1024 x 33 198 (224); 256 x 128 x 12 x 32 58 (93).
// Rows of 32 and fewer (1024 x 32: 193) stay with the two kernels, which need no low bytes there.  Bound by latency: LDS and registers
// leave room for two workgroups, and each is load, products, store one after the other.
template <int DP>
struct Short {
    typedef Image<__bf16, DP, ROWS> Img;       // q, do, k
    typedef Image<__bf16, ROWS, ROWS> Grad;    // ds
    static constexpr int G = Pass<__bf16, DP>::SCRATCH, STATS = Img::BYTES;   // results go out over q and the statistics
    static constexpr int DS = G + Img::BYTES, LDS = DS + Grad::BYTES;   // (k and v pass through the place of ds first)
    static_assert(2 * Img::BYTES <= Grad::BYTES, "k and v fit there");
    static_assert(STATS + 2 * ROWS * 4 <= G && G % 64 == 0, "q and the statistics fit under the results' scratch");
};
template <int DP>
__global__ __launch_bounds__(THREADS, DP <= 32 ? 3 : 2) void attention_short_backward_kernel(const Args a) {
    typedef __bf16 T;
    typedef Short<DP> S;
    typedef typename S::Img Img;
    extern __shared__ __align__(16) char lds[];   // [q, L, D][do, then k][ds]

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
    Item item;
    Place w;
    if (!work_item(a, 1, item) || !locate(a, item.slot, false, w)) return;
    const int kv_head = item.kv_head, first = 32 * wave, own = first + (lane & 31), blocks = (w.length + 31) / 32;
    T* dk = rows_out<T>(a.dk, w, kv_head);
    T* dv = rows_out<T>(a.dv, w, kv_head);
    if (w.length == 0) {
        zero_rows<T, DP>(dk, a.dk.token, 0, w.written, a.width, tid);
        zero_rows<T, DP>(dv, a.dv.token, 0, w.written, a.width, tid);
        for (int n = 0; n < a.group; ++n) zero_rows<T, DP>(rows_out<T>(a.dq, w, kv_head * a.group + n), a.dq.token, 0, w.written, a.width, tid);
        return;
    }
    const Reader<T, DP, ROWS> read(lane);
    const Reader<T, ROWS, ROWS> read_ds(lane);
    const uint32_t qt = lds_address(lds), gt = qt + S::G, dt = qt + S::DS;
    float* stats = reinterpret_cast<float*>(lds + S::STATS);   // [L, D][ROWS]
    Held<T, DP> k, v;
    f32x16 ak[DP / 32] = {}, av[DP / 32] = {};
    const float c = a.scale * LOG2E;
    const Rows k_rows = input_rows<T>(a, a.k, w, kv_head), v_rows = input_rows<T>(a, a.v, w, kv_head);
    Stage<T, DP, ROWS> sk(k_rows.token, k_rows.width, tid);
    sk.load(k_rows.from(0));

    for (int head = kv_head * a.group; head < (kv_head + 1) * a.group; ++head) {
        {
            const Rows q = input_rows<T>(a, a.q, w, head), g = input_rows<T>(a, a.g, w, head);
            Stage<T, DP, ROWS> sq(q.token, q.width, tid), sg(g.token, g.width, tid);
            sq.load(q.from(0));
            sg.load(g.from(0));
            const Rows o = input_rows<T>(a, a.o, w, head);
            Stage<T, DP, ROWS> sv(v_rows.token, v_rows.width, tid);
            sv.load(v_rows.from(0));
            float l = INFINITY;   // (p = 0 for rows that hold no token)
            if (tid < ROWS && tid < w.length) l = a.lse[head * a.rows + w.stat + tid];
            __syncthreads();   // (the head before: its dq is out, its ds read)
            sq.store(lds);
            sg.store(lds + S::G);
            sk.store(lds + S::DS);   // k and v pass through the place of ds
            sv.store(lds + S::DS + Img::BYTES);
            if (tid < ROWS) stats[tid] = l;
        }
        __syncthreads();
        if (head == kv_head * a.group) {
#pragma unroll
            for (int i = 0; i < Img::SLABS; ++i) {
                k.f[i] = read.rows(dt, first, i);
                v.f[i] = read.rows(dt + Img::BYTES, first, i);
            }
        }
        // D of the wave's 32 queries as the sum of p dp over their keys, in fp32: nothing of it is rounded, and o is not read
        if (first < w.length) {
            typename Type<T>::Frag q[Img::SLABS], g[Img::SLABS];
#pragma unroll
            for (int i = 0; i < Img::SLABS; ++i) {
                q[i] = read.rows(qt, first, i);
                g[i] = read.rows(gt, first, i);
            }
            const int visible = a.causal ? min(w.length, own + 1) : w.length, end = a.causal ? wave + 1 : blocks;
            const float l = stats[own];
            float delta = 0.0f;
            for (int b = 0; b < end; ++b) {
                f32x16 s = {}, dp = {};
#pragma unroll
                for (int i = 0; i < Img::SLABS; ++i) s = Type<T>::mma(read.rows(dt, 32 * b, i), q[i], s);
#pragma unroll
                for (int i = 0; i < Img::SLABS; ++i) dp = Type<T>::mma(read.rows(dt + Img::BYTES, 32 * b, i), g[i], dp);
                settle();
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    delta = fmaf(32 * b + 8 * (r / 4) + 4 * half + r % 4 < visible ? __builtin_amdgcn_exp2f(fmaf(s[r], c, -l)) : 0.0f, dp[r], delta);
            }
            delta += other_half(delta);
            if (half == 0) stats[ROWS + own] = own < w.length ? delta : 0.0f;
        }
        __syncthreads();
        if (first < w.length) {
            for (int b = a.causal ? wave : 0; b < blocks; ++b) {
                f32x16 s = {}, dp = {};
#pragma unroll
                for (int i = 0; i < Img::SLABS; ++i) s = Type<T>::mma(read.rows(qt, 32 * b, i), k.f[i], s);
#pragma unroll
                for (int i = 0; i < Img::SLABS; ++i) dp = Type<T>::mma(read.rows(gt, 32 * b, i), v.f[i], dp);
                const float* rows_lse = stats + 32 * b + 4 * half;
                const float* rows_delta = rows_lse + ROWS;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 l4 = *reinterpret_cast<const f32x4*>(rows_lse + 8 * i);
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[4 * i + j] = __builtin_amdgcn_exp2f(fmaf(s[4 * i + j], c, -l4[j]));
                }
                settle();
                if ((a.causal & (b == wave)) | (first + 32 > w.length) | (w.length == 1)) {
                    // rows of the block that do not see the key: those in front of it, or all
                    const int hidden = own >= w.length ? 32 : a.causal ? own - 32 * b - 4 * half : -32;
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (8 * (r / 4) + r % 4 < hidden) s[r] = 0.0f;
                    // the first row of a causal sequence, or the only one, sees one key: ds is exactly 0
                    if (32 * b + 4 * half == 0 && (a.causal || w.length == 1)) dp[0] = rows_delta[0];
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const bf16x8 p = Type<T>::from_acc(s, i);
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d) av[d] = Type<T>::mma(read.columns(gt, 32 * b, i, d), p, av[d]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 d4 = *reinterpret_cast<const f32x4*>(rows_delta + 8 * i);
#pragma unroll
                    for (int j = 0; j < 4; ++j) dp[4 * i + j] = s[4 * i + j] * (dp[4 * i + j] - d4[j]);
                    Type<T>::store4(lds + S::DS + b * S::Grad::BLOCK + own * 64 + ((i ^ (own >> 2)) & 3) * 16 + 8 * half, dp[4 * i], dp[4 * i + 1],
                                    dp[4 * i + 2], dp[4 * i + 3]);
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const bf16x8 ds = Type<T>::from_acc(dp, i);
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d) ak[d] = Type<T>::mma(read.columns(qt, 32 * b, i, d), ds, ak[d]);
                }
            }
        }
        __syncthreads();   // q and do are done with
        sk.store(lds + S::G);
        __syncthreads();
        f32x16 aq[DP / 32] = {};
        if (first < w.length) {
            const int end = a.causal ? wave + 1 : blocks;
            for (int b = 0; b < end; ++b)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const bf16x8 ds = read_ds.columns(dt, 32 * b, i, wave);
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d) aq[d] = Type<T>::mma(read.columns(gt, 32 * b, i, d), ds, aq[d]);
                }
        }
        settle();
        if (own >= w.length) {
#pragma unroll
            for (int d = 0; d < DP / 32; ++d) aq[d] = f32x16{};
        }
        store_rows<T, DP>(aq, lds, rows_out<T>(a.dq, w, head), a.dq.token, first, w.written, a.width, a.scale, wave, lane);
    }
    if (own >= w.length) {
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) { ak[d] = f32x16{}; av[d] = f32x16{}; }
    }
    store_rows<T, DP>(ak, lds, dk, a.dk.token, first, w.written, a.width, a.scale, wave, lane);
    store_rows<T, DP>(av, lds, dv, a.dv.token, first, w.written, a.width, 1.0f, wave, lane);
}

// dk and dv as the sums of the parts in order; zero in rows of no sequence.  One thread per four columns.
template <class T>
__global__ __launch_bounds__(THREADS) void attention_join_kernel(const Args a) {
    const int quads = a.width / 4, kv_heads = a.heads / a.group;
    const int64_t n = static_cast<int64_t>(blockIdx.x) * THREADS + threadIdx.x, all = a.rows * kv_heads;
    const int64_t line = n / quads, row = line / kv_heads;
    if (line >= all) return;
    const int column = static_cast<int>(n % quads) * 4, head = static_cast<int>(line % kv_heads);
    int64_t sequence = 0, token = row;
    bool real;
    if (a.offsets) {
        real = row >= a.offsets[0] && row < a.offsets[a.sequences];
    } else {
        sequence = row / a.length;
        token = row % a.length;
        real = !a.lengths || token < a.lengths[sequence];
    }
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        f32x4 sum = {};
        if (real)
            for (int i = 0; i < a.parts; ++i)
                sum += *reinterpret_cast<const f32x4*>(a.partial + (((static_cast<int64_t>(i) * 2 + which) * kv_heads + head) * a.rows + row) * a.width + column);
        const Tensor& to = which ? a.dv : a.dk;
        Type<T>::store4(const_cast<T*>(reinterpret_cast<const T*>(to.p)) + sequence * to.batch + token * to.token + head * to.head + column, sum[0], sum[1],
                        sum[2], sum[3]);
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------------
// Tile rows and waves per SIMD of each kernel: as many waves as the registers allow (a wave's exponentials run beside another's matrix
// instructions), and the tile height that leaves room for them.  Times in us, the other choice in brackets; A: 64 x 512 x 12 heads x 64,
// B: 16 x 512 x 32/8 heads x 128, C: 64 x 512 x 12 heads x 32, all bf16 causal; D: fp32, 24 sequences of 29 to 233 tokens x 12 heads x 64.
//   forward: 64 keys, four waves: A 62 (32 keys: 64), C 46 (32: 50); above width 64 32 keys, three waves: B 74 (64 keys, two waves: 78)
//   dq: 32 keys, four waves: A 84 (64 keys, two waves: 85); above width 64 64 keys: B 110 (32 keys: 115)
//   dk / dv: 32 queries, three waves: A 102 (64 queries, in registers for one wave: 231); width 32 64 queries: all of the backward C 135 (146)
//   v from LDS (VL): A 102 (v in registers: 120), B 131 (213); width 96 has the registers
//   fp32: three, two and two waves: D 27, 36, 44 (two, one and one: 28.5, 38, 62); above width 64 the parts' registers leave one
// What these choices spill: dk / dv bf16 at width 128 10 vector registers (24 bytes of scratch a lane), fp32 at width 64 5 (24 bytes) and at
// width 128 36 (148 bytes); the one-kernel backward 25 to 28 scalar registers, into vector ones.
template <class T, int DP>
struct Shape {
    static constexpr bool SHORT = PARTS<T> == 1 && DP <= 64;   // wider heads and split values leave the LDS no room for two workgroups
    static constexpr bool SPLIT = PARTS<T> == 3, VL = !SPLIT && (DP == 64 || DP > 96);
    static constexpr int FORWARD_KEYS = !SPLIT && DP <= 64 ? 64 : 32, DQ_KEYS = !SPLIT && DP > 64 ? 64 : 32, QUERIES = !SPLIT && DP <= 32 ? 64 : 32;
    static constexpr int FORWARD_WAVES = SPLIT ? (DP <= 64 ? 3 : 1) : DP <= 64 ? 4 : 3, DQ_WAVES = SPLIT ? (DP <= 64 ? 2 : 1) : DP <= 64 ? 4 : 2;
    static constexpr int DKV_WAVES = SPLIT ? (DP <= 64 ? 2 : 1) : DP <= 64 ? 3 : 2;
    static constexpr int FORWARD_LDS = std::max(4 * Image<T, DP, FORWARD_KEYS>::BYTES, Pass<T, DP>::SCRATCH);
    static constexpr int DQ_LDS = std::max(4 * Image<T, DP, DQ_KEYS>::BYTES, Pass<T, DP>::SCRATCH);
    static constexpr int DKV_LDS =
        std::max(4 * Image<T, DP, QUERIES>::BYTES + 4 * QUERIES * 4 + (VL ? Image<T, DP, ROWS>::BYTES : 0), Pass<float, DP>::SCRATCH);
    static constexpr auto forward = &attention_forward_kernel<T, DP, FORWARD_KEYS, FORWARD_WAVES>;
    static constexpr auto dq = &attention_dq_kernel<T, DP, DQ_KEYS, DQ_WAVES>;
    static constexpr auto dkv = &attention_dkv_kernel<T, DP, QUERIES, VL, DKV_WAVES>;
};

template <class T, int DP>
bool configure() {
    typedef Shape<T, DP> S;
    auto set = [](auto f, int bytes) {
        return hipFuncSetAttribute(reinterpret_cast<const void*>(f), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess;
    };
    if constexpr (S::SHORT)
        if (!set(&attention_short_backward_kernel<DP>, Short<DP>::LDS)) return false;
    return set(S::forward, S::FORWARD_LDS) && set(S::dq, S::DQ_LDS) && set(S::dkv, S::DKV_LDS);
}

// Kernel attribute set-up, once per device, thread-safe.
int configure_kernels() {
    constexpr int DEVICES = 64;
    static std::once_flag flags[DEVICES];
    static int status[DEVICES] = {};
    int device = 0;
    if (hipGetDevice(&device) != hipSuccess || device < 0 || device >= DEVICES) return KF_ERR_LAUNCH_FAILED;
    std::call_once(flags[device], [device] {
        if (!(configure<__bf16, 32>() && configure<__bf16, 64>() && configure<__bf16, 96>() && configure<__bf16, 128>() && configure<Split, 32>() &&
              configure<Split, 64>() && configure<Split, 96>() && configure<Split, 128>()))
            status[device] = KF_ERR_LAUNCH_FAILED;
    });
    return status[device];
}

// The rows that attention_short_backward_kernel takes: it and rows that see 32 keys at most have D from p and dp, and need no remainder.
bool short_rows(int dtype, int64_t length, int64_t width, bool packed) { return dtype == KF_BF16 && !packed && length > 32 && length <= ROWS && width <= 64; }
bool keeps_rest(int dtype, int64_t length, int64_t width, bool packed) {
    return dtype == KF_BF16 && (packed || length > 32) && !short_rows(dtype, length, width, packed);
}

template <class T, int DP>
int launch_width(Args& a, bool backward, hipStream_t stream) {
    typedef Shape<T, DP> S;
    const int64_t round = XCDS * a.chunk, slots = (static_cast<int64_t>(a.slots) * (a.heads / a.group) + round - 1) / round * round;
    const unsigned items = static_cast<unsigned>(slots * a.group);
    if (!backward) {
        S::forward<<<items, THREADS, S::FORWARD_LDS, stream>>>(a);
    } else {
        if constexpr (S::SHORT)
            if (short_rows(KF_BF16, a.length, a.width, a.offsets != nullptr)) {
                attention_short_backward_kernel<DP><<<static_cast<unsigned>(slots), THREADS, Short<DP>::LDS, stream>>>(a);
                return hipGetLastError() == hipSuccess ? KF_OK : KF_ERR_LAUNCH_FAILED;
            }
        S::dq<<<items, THREADS, S::DQ_LDS, stream>>>(a);
        S::dkv<<<static_cast<unsigned>(slots * a.parts), THREADS, S::DKV_LDS, stream>>>(a);
        if (a.parts > 1) {
            const int64_t threads = a.rows * (a.heads / a.group) * (a.width / 4);
            attention_join_kernel<typename Type<T>::Memory><<<static_cast<unsigned>((threads + THREADS - 1) / THREADS), THREADS, 0, stream>>>(a);
        }
    }
    return hipGetLastError() == hipSuccess ? KF_OK : KF_ERR_LAUNCH_FAILED;
}

template <class T>
int launch_type(Args& a, bool backward, hipStream_t stream) {
    if (a.width <= 32) return launch_width<T, 32>(a, backward, stream);
    if (a.width <= 64) return launch_width<T, 64>(a, backward, stream);
    if (a.width <= 96) return launch_width<T, 96>(a, backward, stream);
    return launch_width<T, 128>(a, backward, stream);
}

// (packed: without the last slot, which holds a tile of the rows in front of the first sequence at most)
int64_t tile_slots(int64_t sequences, int64_t length, int64_t rows, bool packed) {
    return packed ? rows / ROWS + sequences + 1 : sequences * ((length + ROWS - 1) / ROWS);
}

constexpr int64_t MAX_PARTS = 4, RESIDENT = 512;   // (two workgroups on each of 256 compute units)

int64_t delta_bytes(int64_t rows, int64_t heads) { return (rows * heads * 4 + 15) / 16 * 16; }

// How many workgroups share the queries of one key tile in the dk / dv kernel.  512 workgroups of it fit the card at a time, and
// the first tile of a causal sequence has twice the mean work: with all of them resident at once the kernel takes as long as its
// largest item.  Measured (bf16, causal, width 128): one document of 8192 tokens, 32/8 heads, 512 items: 1867 us whole, 1138 + 28 us
// (join) in two parts, 1135 + 58 in four; 24 documents of 12011 tokens in all, 16/4 heads, 472 items: 425 us whole, 235 + 21 in two,
// 159 + 36 in four; 16 x 512 tokens, 32/8 heads, 512 items of at most 64 steps: 128 us whole, 108 + 30 in two.
// A part of at least 128 steps (all of the backward, us; at least 64, at least 256): 1 x 2048 x 8/2 x 128 274 (180, 459), 1 x 2048 x 32/4 x 64 175
// (175, 281), 1 x 8192 x 8 x 64 360 (360, 419), 2 x 2048 x 16 x 64 136 (137, 137).  The lengths of packed documents are not known here,
// and their steps are counted as if all rows were one: right for 41 of 100 to 2000 tokens, 16/4 heads x 128 (198 us, whole 461), a loss for short ones
// (64 of 128 tokens, 16/4 x 128: 118 us, whole 81; 96 of 64, 12/4 x 64: 51 and 32).
int64_t dkv_parts(int64_t sequences, int64_t length, int64_t rows, int64_t heads, int64_t kv_heads, bool packed, bool causal) {
    const int64_t items = tile_slots(sequences, length, rows, packed) * kv_heads, steps = ((packed ? rows : length) + 31) / 32 * (heads / kv_heads);
    const int64_t wanted = ((packed ? 2048 : causal ? 1024 : 512) + items - 1) / items;
    return std::max<int64_t>(1, std::min(std::min(wanted, MAX_PARTS), steps / 128));
}

// the statistics that the forward call leaves for the backward one: L, and where it is kept the remainder
void place_stats(Args& a, float* stats, int dtype, bool packed) {
    a.lse = stats;
    if (stats == nullptr || !keeps_rest(dtype, a.length, a.width, packed)) return;
    const int64_t token = rest_width(a.width);
    a.rest = Tensor{reinterpret_cast<const char*>(stats) + delta_bytes(a.rows, a.heads), packed ? 0 : a.length * token, token, a.rows * token};
}

Tensor tensor_of(const kf_heads_view* v) { return Tensor{v->p, v->batch_stride, v->token_stride, v->head_stride}; }

// 16-byte chunks, rows that do not overlap (a load behind the last row must fall behind the buffer's end), and a tile's span below
// 2^30 bytes
bool usable(const kf_heads_view* v, int64_t per, int64_t width) {
    return v != nullptr && v->p != nullptr && reinterpret_cast<uintptr_t>(v->p) % 16 == 0 && v->batch_stride % per == 0 && v->token_stride % per == 0 &&
           v->head_stride % per == 0 && v->token_stride >= width && v->token_stride <= (int64_t{1} << 23) / (16 / per);
}

int fill(Args& a, int dtype, int64_t sequences, int64_t length, int64_t rows, int64_t heads, int64_t kv_heads, int64_t width, const int32_t* lengths,
         const int32_t* offsets, int causal, float scale) {
    if (dtype != KF_BF16 && dtype != KF_F32) return KF_ERR_UNSUPPORTED_DTYPE;
    const int64_t per = dtype == KF_BF16 ? 8 : 4, limit = 0x7fffffff;
    if (sequences <= 0 || rows <= 0 || rows > limit - ROWS || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || width <= 0 || width > 128 ||
        width % per != 0 || !(scale > 0.0f) || !isfinite(scale))
        return KF_ERR_INVALID_ARGUMENT;
    if (offsets ? lengths != nullptr : (length <= 0 || sequences > limit / length || rows != sequences * length)) return KF_ERR_INVALID_ARGUMENT;
    const int64_t slots = tile_slots(sequences, length, rows, offsets != nullptr) + (offsets != nullptr);
    const int64_t tiles = offsets ? 0 : slots / sequences, groups = offsets ? 0 : sequences * kv_heads;
    // Whole pairs from 64 on (all of the backward, us, causal bf16; single tiles in brackets): 8 x 2048 x 8 x 64 158 (211), 16 x 512 x 8 x 64 44
    // (49), 64 x 512 x 2/1 x 64 55 (57); fewer pairs of few tiles are even: 4 x 512 x 8/4 x 128 80 (79), 2 x 2048 x 8 x 64 113 (113), and at
    // 32 pairs of many tiles whole ones would gain: 4 x 2048 x 8 x 64 122 (138).
    const int64_t chunk = groups >= 64 ? tiles : 1;
    if (sequences >= limit || slots > (limit / MAX_PARTS - XCDS * chunk * heads) / heads) return KF_ERR_INVALID_ARGUMENT;
    a.chunk = static_cast<int>(chunk);
    a.lengths = lengths;
    a.offsets = offsets;
    a.rows = rows;
    a.sequences = static_cast<int>(sequences);
    a.length = static_cast<int>(length);
    a.heads = static_cast<int>(heads);
    a.group = static_cast<int>(heads / kv_heads);
    a.width = static_cast<int>(width);
    a.causal = causal != 0;
    a.slots = static_cast<int>(slots);
    a.scale = scale;
    return KF_OK;
}

}  // namespace

extern "C" {

int64_t kf_attention_order_bytes(int64_t sequences, int64_t rows, int64_t heads) {
    if (sequences <= 0 || rows <= 0 || heads <= 0) return 0;
    const int64_t slots = tile_slots(sequences, 0, rows, true);
    return slots <= MAX_ORDERED && slots * heads > RESIDENT ? slots * 4 : 0;
}

int kf_attention_starts(int32_t* starts, const void* offsets, int offsets_dtype, int64_t sequences, int64_t rows, void* stream) {
    if (offsets_dtype != KF_I32 && offsets_dtype != KF_I64) return KF_ERR_UNSUPPORTED_DTYPE;
    if (starts == nullptr || offsets == nullptr || sequences < 0 || rows < 0 || rows > 0x7fffffff) return KF_ERR_INVALID_ARGUMENT;
    attention_starts_kernel<<<1, 1024, 0, reinterpret_cast<hipStream_t>(stream)>>>(starts, offsets, offsets_dtype == KF_I64, sequences + 1, rows);
    return hipGetLastError() == hipSuccess ? KF_OK : KF_ERR_LAUNCH_FAILED;
}

int kf_attention_order(int32_t* order, const int32_t* offsets, int64_t sequences, int64_t rows, int causal, void* stream) {
    if (order == nullptr || offsets == nullptr || sequences <= 0 || rows <= 0 || tile_slots(sequences, 0, rows, true) > MAX_ORDERED)
        return KF_ERR_INVALID_ARGUMENT;
    Args a = {};
    a.offsets = offsets;
    a.rows = rows;
    a.sequences = static_cast<int>(sequences);
    a.causal = causal != 0;
    a.slots = static_cast<int>(tile_slots(sequences, 0, rows, true));
    attention_order_kernel<<<1, 1024, 0, reinterpret_cast<hipStream_t>(stream)>>>(a, order);
    return hipGetLastError() == hipSuccess ? KF_OK : KF_ERR_LAUNCH_FAILED;
}

int64_t kf_attention_stats_bytes(int dtype, int64_t length, int64_t rows, int64_t heads, int64_t width, int packed) {
    if (rows <= 0 || heads <= 0 || width <= 0 || (!packed && length <= 0)) return 0;
    return delta_bytes(rows, heads) + (keeps_rest(dtype, length, width, packed) ? rows * heads * rest_width(width) : 0);
}

int kf_attention_forward(const kf_heads_view* out, float* stats, const kf_heads_view* q, const kf_heads_view* k, const kf_heads_view* v, int dtype,
                         int64_t sequences, int64_t length, int64_t rows, int64_t heads, int64_t kv_heads, int64_t width, const int32_t* lengths,
                         const int32_t* offsets, const int32_t* order, int causal, float scale, void* stream) {
    Args a = {};
    if (int s = fill(a, dtype, sequences, length, rows, heads, kv_heads, width, lengths, offsets, causal, scale)) return s;
    const int64_t per = dtype == KF_BF16 ? 8 : 4;
    if (!usable(out, per, width) || !usable(q, per, width) || !usable(k, per, width) || !usable(v, per, width) ||
        reinterpret_cast<uintptr_t>(stats) % 16 != 0)
        return KF_ERR_INVALID_ARGUMENT;
    if (order != nullptr && offsets == nullptr) return KF_ERR_INVALID_ARGUMENT;
    a.order = order;
    if (int s = configure_kernels()) return s;
    a.q = tensor_of(q); a.k = tensor_of(k); a.v = tensor_of(v); a.o = tensor_of(out);
    place_stats(a, stats, dtype, offsets != nullptr);
    const hipStream_t on = reinterpret_cast<hipStream_t>(stream);
    return dtype == KF_BF16 ? launch_type<__bf16>(a, false, on) : launch_type<Split>(a, false, on);
}

int64_t kf_attention_backward_workspace_bytes(int64_t sequences, int64_t length, int64_t rows, int64_t heads, int64_t kv_heads, int64_t width, int packed,
                                              int causal) {
    if (sequences <= 0 || rows <= 0 || heads <= 0 || kv_heads <= 0 || width <= 0 || (!packed && length <= 0)) return 0;
    const int64_t parts = dkv_parts(sequences, length, rows, heads, kv_heads, packed, causal);
    return delta_bytes(rows, heads) + (parts > 1 ? parts * 2 * kv_heads * rows * width * 4 : 0);
}

int kf_attention_backward(const kf_heads_view* dq, const kf_heads_view* dk, const kf_heads_view* dv, const kf_heads_view* grad, const kf_heads_view* out,
                          const float* stats, const kf_heads_view* q, const kf_heads_view* k, const kf_heads_view* v, int dtype, int64_t sequences,
                          int64_t length, int64_t rows, int64_t heads, int64_t kv_heads, int64_t width, const int32_t* lengths, const int32_t* offsets,
                          const int32_t* order, int causal, float scale, void* workspace, int64_t workspace_bytes, void* stream) {
    Args a = {};
    if (int s = fill(a, dtype, sequences, length, rows, heads, kv_heads, width, lengths, offsets, causal, scale)) return s;
    const int64_t per = dtype == KF_BF16 ? 8 : 4;
    const kf_heads_view* all[] = {dq, dk, dv, grad, out, q, k, v};
    for (const kf_heads_view* t : all)
        if (!usable(t, per, width)) return KF_ERR_INVALID_ARGUMENT;
    if (stats == nullptr || reinterpret_cast<uintptr_t>(stats) % 16 != 0) return KF_ERR_INVALID_ARGUMENT;
    if (workspace == nullptr ||
        workspace_bytes < kf_attention_backward_workspace_bytes(sequences, length, rows, heads, kv_heads, width, offsets != nullptr, causal))
        return KF_ERR_WORKSPACE_TOO_SMALL;
    if (order != nullptr && offsets == nullptr) return KF_ERR_INVALID_ARGUMENT;
    a.order = order;
    if (int s = configure_kernels()) return s;
    a.q = tensor_of(q); a.k = tensor_of(k); a.v = tensor_of(v); a.o = tensor_of(out); a.g = tensor_of(grad);
    a.dq = tensor_of(dq); a.dk = tensor_of(dk); a.dv = tensor_of(dv);
    place_stats(a, const_cast<float*>(stats), dtype, offsets != nullptr);
    a.delta = reinterpret_cast<float*>(workspace);
    a.partial = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + delta_bytes(rows, heads));
    a.parts = static_cast<int>(dkv_parts(sequences, length, rows, heads, kv_heads, offsets != nullptr, causal));
    const hipStream_t on = reinterpret_cast<hipStream_t>(stream);
    return dtype == KF_BF16 ? launch_type<__bf16>(a, true, on) : launch_type<Split>(a, true, on);
}

}  // extern "C"
