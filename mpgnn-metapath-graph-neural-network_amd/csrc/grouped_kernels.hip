// Matrix products grouped by type, relation or expert, over groups of ragged sizes:
//   forward          y[i]  = x[i] @ W[g] + b[g]          for the rows i of group g
//   input gradient   dx[i] = dy[i] @ W[g]^T
//   weight gradient  dW[g] = x_g^T @ dy_g,  db[g] = the column sums of dy_g
// with x [M, K] sorted by group, group g owning rows [ptr[g], ptr[g + 1]), W [G, K, N], and ptr on
// the device: no size is known to the host, so each launch has a workgroup for every tile that
// there could be (rows / tile + groups), and a workgroup finds its tile by a search over ptr.
//
// One kernel computes D[r][n] = sum_c R(r, c) * B(n, c) in tiles on the matrix cores
// (v_mfma_f32_16x16x32, fp32 accumulators) with either operand stored along c or across it:
//   forward          R = x (along c = k)       B = W  (across: n runs fastest)
//   input gradient   R = dy (along c = n)      B = W  (along: c = n runs fastest)
//   weight gradient  R = x (across: c = rows)  B = dy (across)
// An operand stored along c goes to LDS as [index][c] and its fragments are 16-byte reads; one
// stored across goes as [c][index] and its fragments are transposed reads (ds_read_b64_tr_b16: a
// 16-lane group reads 4 c x 16 indices, lane i receives index i). Both layouts place 16-byte
// (32-byte) pieces by an exclusive-or with the row, which keeps each read's lanes on distinct banks.
// B is the first matrix operand, so that a lane ends up with four neighbouring columns of a row.
//
// fp32 operands run on the bf16 matrix cores: an exact split of each value in three bf16 pieces
// and the six products of at least 2^-16 of the full one, which leaves an error of fp32's own
// size at 16/6 of the fp32 matrix rate. (Exact from 2^-110 in magnitude on, 8e-34; smaller values lose what lies below
// the subnormal bf16 numbers, at most 2^-134 each.) An element whose pieces overflow or are not finite gives a
// result that is not finite; such results are computed again from the operands in fp32, so that
// infinities and NaN come out as a sum of products has them.
//
// Bound by the matrix cores where rows are many (32 groups, 32,768 rows, 2048 x 4096 bf16: forward 598, input gradient
// 583, weight gradient 660 us on average, 0.82, 0.85 and 0.75 of a large library product's rate; 8 groups, 32,768 rows,
// 2048 x 2048 fp32: 1369, 1356 and 1383 us, six products at the library's bf16 rate), by splitting and staging the weight
// for every 128 rows where it is small (237 groups, 208k rows, 128 x 128 fp32 77, 75 and 75 + 15 us), by reading the
// weights where rows are few (48 rows, 64 groups, 2048 x 2048 bf16 63 us, the hit weights at 4.8 TB/s), by the loads of
// unaligned rows where widths are odd (20,011 rows, 7 groups, 193 x 301 fp16 20, 22 and 24 + 9 us).
#include <algorithm>

#include "num_types.h"

namespace mpgnn {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

constexpr int kGlThreads = 256;

enum Layout { ALONG, ACROSS };  // c fastest, or the index fastest

struct GroupedArgs {
    const void* r;      // rows operand
    const void* b;      // columns operand
    const void* r_end;  // behind the last element of each
    const void* b_end;
    void* out;
    const void* bias;   // forward: [G][cols] or null
    const void* ptr;    // [G + 1] int32 or int64
    float* slabs;       // weight gradient: [items][K * N (+ N)] partials of groups cut in chunks
    void* dbias;        // weight gradient: [G][cols] or null
    int64_t rows;       // M
    int64_t r_pitch, b_pitch;
    int64_t b_group;    // elements from one group's B to the next (0: B has no groups)
    int32_t groups;
    int32_t ptr64;
    int32_t cc;         // forward, input gradient: length of c
    int32_t out_rows;   // weight gradient: K
    int32_t cols;       // columns of the output
    int32_t col_tiles, row_tiles;
    int32_t chunk;      // weight gradient: rows of a chunk
    int64_t items;      // weight gradient: slabs there are room for
    int32_t run;        // tiles that an XCD takes in a row
};

// 8 values of c of one index from a tile stored across: two transposed reads of 4 c x 16 indices
template <typename V8, typename T>
__device__ __forceinline__ V8 read_across(const T* lo, const T* hi) {
    typedef __attribute__((address_space(3))) i16x4 lds4;
    const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)lo);
    const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)hi);
    return __builtin_bit_cast(V8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

template <typename T>
struct Frag;
template <>
struct Frag<__bf16> {
    typedef bf16x8 type;
    static __device__ __forceinline__ f32x4 mfma(type a, type b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Frag<_Float16> {
    typedef f16x8 type;
    static __device__ __forceinline__ f32x4 mfma(type a, type b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};

// How an element type is staged: 16-bit as itself, fp32 as three bf16 planes.
template <typename T>
struct Stage {
    typedef T elem;
    static constexpr int planes = 1, bk = 64;
};
template <>
struct Stage<float> {
    typedef __bf16 elem;
    static constexpr int planes = 3, bk = 32;
};

// ---------------------------------------------------------------------------------------
// groups and tiles
// ---------------------------------------------------------------------------------------
__device__ __forceinline__ int64_t ptr_at(const GroupedArgs& a, int g) {
    const int64_t v = a.ptr64 ? ((const int64_t*)a.ptr)[g] : (int64_t)((const int32_t*)a.ptr)[g];
    return v < 0 ? 0 : v > a.rows ? a.rows : v;  // no ptr, however wrong, leads outside the tensors
}

__device__ __forceinline__ int64_t scalar(int64_t v) {
    return (int64_t)((uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 |
                     (unsigned)__builtin_amdgcn_readfirstlane((int)v));
}

// The tile of this workgroup. Workgroups go to the eight XCDs in turn, each of which has an L2 of its own: an
// XCD takes `run` tiles in a row, so that tiles which read the same rows read them from memory once.
__device__ __forceinline__ int tile_of(const GroupedArgs& a) {
    const unsigned id = blockIdx.x, run = a.run;
    return (int)(id / (8 * run) * (8 * run) + id % 8 * run + id / 8 % run);
}

struct Item {
    int group;    // -1: none; groups: rows that belong to no group
    int part;     // which tile (chunk) of the group
    int parts;    // of how many
    int64_t lo, hi;
};

// Groups that start at row `lo`, `before` groups before them, have their places in a list of parts of `size` rows from
// lo / size + before on: up to the next group's these are one more than the group's rows' whole parts, hence as many as
// its parts at least, one if it has none, and rows / size + groups in all. No sum of the sizes before is needed.
__device__ __forceinline__ int64_t place_of(int64_t lo, int size, int64_t before) {
    return (int64_t)((unsigned long long)lo / (unsigned)size) + before;
}

// Item `id` of the list of all groups' parts: each group has ceil(rows / size) of them, at least
// `least`. With `rest`, the rows before ptr[0] and from ptr[G] on are two more groups.
//
// Up to kScanned groups, by a sum over their parts, THREADS groups a turn: the items lie without gaps, and the last
// workgroups are the idle ones. (Half of the THREADS groups of a turn at most overlap in a decreasing ptr, each no more
// than a launch has workgroups, 2^32 / THREADS: an unsigned count does not wrap around, no two groups get one item.)
//
// Above that by a search over the places, THREADS ways a turn, between which idle workgroups lie. By the sum alone the
// time grew with the square of the groups: 131,072 groups of a row, 16 x 16 bf16, forward 51.6 ms, 2.3 by the search.
// us by the sum and by the search, forward:
//   bf16 (256 threads)   300 groups, 200k rows, 128 x 128  36.6 / 35.0   2,700, 8,192, 64 x 64  48.5 / 28.6
//   fp32 (512 threads)   520 groups, 200k rows, 128 x 128  64.1 / 70.7   2,700, 300k, 64 x 64   86.1 / 63.0
//   bf16, tiles of 256   32 groups, 32,768 rows, 2048 x 4096, training   1811 / 1844
// A ptr that decreases misleads the search; what it finds is still rows inside the tensors, one item a place.
template <int THREADS>
__device__ __forceinline__ Item find_item(const GroupedArgs& a, int id, int size, int least, bool rest) {
    constexpr int kScanned = THREADS == 512 ? 1024 : THREADS;
    __shared__ unsigned s_count[2][THREADS / 64];
    __shared__ Item s_item;
    const int n = a.groups + (rest ? 2 : 0);
    auto parts_of = [&](int64_t lo, int64_t hi) {
        const unsigned parts = (unsigned)((unsigned long long)(hi - lo + size - 1) / (unsigned)size);
        return parts < (unsigned)least ? (unsigned)least : parts;
    };
    if (threadIdx.x == 0) s_item.group = -1;
    if (n <= kScanned) {
        unsigned base = 0;  // parts before g0
        for (int g0 = 0; g0 < n; g0 += THREADS) {
            const int g = g0 + threadIdx.x;
            int64_t lo = 0, hi = 0;
            if (g < a.groups) {
                lo = ptr_at(a, g);
                hi = ptr_at(a, g + 1);
                hi = hi < lo ? lo : hi;
            } else if (g == a.groups) {
                lo = ptr_at(a, a.groups);
                hi = a.rows;
            } else {
                hi = ptr_at(a, 0);
            }
            const unsigned parts = g < n ? parts_of(lo, hi) : 0;
            unsigned sum = parts;  // inclusive scan over the wave
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const unsigned v = __shfl_up(sum, d, 64);
                if ((int)(threadIdx.x % 64) >= d) sum += v;
            }
            unsigned* s_sum = s_count[g0 / THREADS % 2];
            if (threadIdx.x % 64 == 63) s_sum[threadIdx.x / 64] = sum;
            __syncthreads();  // (of two buffers in turn: one barrier a turn is enough)
            unsigned before = base;
#pragma unroll
            for (int w = 0; w < THREADS / 64; ++w) {
                if (w < (int)(threadIdx.x / 64)) before += s_sum[w];
                base += s_sum[w];
            }
            const unsigned end = before + sum, first = end - parts;
            if ((unsigned)id >= first && (unsigned)id < end)
                s_item = Item{g < a.groups ? g : a.groups, (int)((unsigned)id - first), (int)parts, lo, hi};
            if (base > (unsigned)id) break;
        }
    } else {
        auto start = [&](int h) -> int64_t {  // the first row of entry h, and of the one behind the last
            if (!rest) return ptr_at(a, h);
            return h == 0 ? 0 : h <= a.groups + 1 ? ptr_at(a, h - 1) : a.rows;
        };
        int lo = 0, hi = n;  // the entry is in [lo, hi)
        for (int turn = 0;; turn ^= 1) {
            const int step = (int)(((unsigned)(hi - lo) + THREADS - 1) / THREADS);
            const int h = lo + (int)threadIdx.x * step;  // below 2^24 + 512 * 2^16
            const int64_t row = h < hi ? start(h) : 0;
            const bool begun = h < hi && place_of(row, size, h) <= id;
            const unsigned long long lanes = __ballot(begun);
            if (threadIdx.x % 64 == 0) s_count[turn][threadIdx.x / 64] = __popcll(lanes);
            __syncthreads();  // (of two buffers in turn: one barrier a turn is enough)
            int count = 0;
#pragma unroll
            for (int w = 0; w < THREADS / 64; ++w) count += (int)s_count[turn][w];
            count = __builtin_amdgcn_readfirstlane(count);
            if (count == 0) break;
            lo += (count - 1) * step;
            if (step == 1) {
                if ((int)threadIdx.x == count - 1) {
                    int64_t end = start(h + 1);
                    end = end < row ? row : end;
                    const int64_t part = id - place_of(row, size, h);
                    const unsigned parts = parts_of(row, end);
                    if (part >= 0 && part < parts)
                        s_item = Item{!rest ? h : h == 0 || h > a.groups ? a.groups : h - 1, (int)part, (int)parts, row, end};
                }
                break;
            }
            hi = hi - lo < step ? hi : lo + step;
        }
    }
    __syncthreads();
    Item it = s_item;  // the same in every lane: into scalar registers
    it.group = __builtin_amdgcn_readfirstlane(it.group);
    it.part = __builtin_amdgcn_readfirstlane(it.part);
    it.parts = __builtin_amdgcn_readfirstlane(it.parts);
    it.lo = scalar(it.lo);
    it.hi = scalar(it.hi);
    return it;
}

// ---------------------------------------------------------------------------------------
// staging: 8 elements of an operand, in memory (raw) and in LDS (planes)
// ---------------------------------------------------------------------------------------
template <typename T>
struct Raw {
    u32x4 v[sizeof(T) / 2];
};

// `valid` of 8 elements at p (any alignment of an element: the hardware's loads need no more)
template <typename T>
__device__ __forceinline__ Raw<T> load8(const T* p, int valid) {
    Raw<T> r;
    if (valid >= 8) {
        __builtin_memcpy(&r, p, sizeof(r));
    } else {
        T e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = i < valid ? p[i] : (T)0.0f;
        __builtin_memcpy(&r, e, sizeof(r));
    }
    return r;
}

__device__ __forceinline__ unsigned pack_bf16(float a, float b) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2{a, b}), bf16x2));
}

template <typename T>
__device__ __forceinline__ void store8(typename Stage<T>::elem* dst, int plane_size, const Raw<T>& r) {
    if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<u32x4*>(dst) = r.v[0];
    } else {
        // by pairs: one conversion instruction a piece, and the pieces stay packed
        float f[8];
        __builtin_memcpy(f, &r, sizeof(f));
        u32x4 p0, p1, p2;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned u0 = pack_bf16(f[2 * i], f[2 * i + 1]);
            const float a = f[2 * i] - __uint_as_float(u0 << 16);
            const float b = f[2 * i + 1] - __uint_as_float(u0 & 0xffff0000u);
            const unsigned u1 = pack_bf16(a, b);
            p0[i] = u0;
            p1[i] = u1;
            p2[i] = pack_bf16(a - __uint_as_float(u1 << 16), b - __uint_as_float(u1 & 0xffff0000u));
        }
        *reinterpret_cast<u32x4*>(dst) = p0;
        *reinterpret_cast<u32x4*>(dst + plane_size) = p1;
        *reinterpret_cast<u32x4*>(dst + 2 * plane_size) = p2;
    }
}

// A tile of IDX indices x BK of c, staged by THREADS threads.
template <typename T, Layout L, int IDX, int BK, int THREADS>
struct Tile {
    typedef typename Stage<T>::elem E;
    static constexpr int plane = IDX * BK;                      // elements
    static constexpr int chunks = IDX * BK / 8 / THREADS;       // 8-element pieces per thread
    static_assert(chunks >= 1 && chunks * THREADS * 8 == plane, "the threads' pieces make up the tile");

    // piece n of a thread: (index, c) of its first element
    static __device__ __forceinline__ void place(int tid, int n, int& idx, int& c) {
        const int id = tid + n * THREADS;
        if constexpr (L == ALONG) {
            idx = id / (BK / 8);
            c = id % (BK / 8) * 8;
        } else {
            c = id / (IDX / 8);
            idx = id % (IDX / 8) * 8;
        }
    }
    // ACROSS: how the 32-byte blocks of row c trade places. A transposed read takes rows c to c + 3 (and 4
    // on) for its first 16 lanes and c + 8 to c + 11 for the next: these eight lie in eight places of the
    // 256 bytes that the LDS serves in a cycle.
    static_assert(L == ALONG || IDX % 128 == 0 || IDX == 64, "the blocks of a row are four or eights");
    static __device__ __forceinline__ int trade(int c) {
        return IDX == 64 ? (c >> 1 & 1) | (c >> 2 & 2) : (c & 3) | (c >> 1 & 4);
    }
    static __device__ __forceinline__ int turn(int idx) { return BK == 64 ? idx & 7 : (idx >> 1) & 3; }  // ALONG
    static __device__ __forceinline__ int offset(int idx, int c) {
        if constexpr (L == ALONG) return idx * BK + ((c / 8) ^ turn(idx)) * 8 + c % 8;
        else return c * IDX + ((idx / 16) ^ trade(c)) * 16 + idx % 16;
    }
    // The fragment of indices i0 + i .. + 15 and c .. c + 31, of which a lane has 8 values of c from c + 8 *
    // (lane / 16) on, of index i0 + i + lane % 16: at(i0) is the lane's place for i = c = 0, and i and c,
    // constants in the unrolled loops, change bits of it that it leaves alone (i < 128, and i0 a multiple
    // of a power of two above i; c a multiple of 32).
    static __device__ __forceinline__ unsigned at(int i0) {
        const int lane = threadIdx.x % 64;
        return L == ALONG ? offset(i0 + lane % 16, lane / 16 * 8)
                          : offset(i0, lane / 16 * 8 + (lane % 16) / 4) + lane % 4 * 4;
    }
    static __device__ __forceinline__ typename Frag<E>::type frag(const E* lds, unsigned at, int i, int c) {
        if constexpr (L == ALONG) {
            return *reinterpret_cast<const typename Frag<E>::type*>(lds + (at ^ c) + i * BK);
        } else {
            const E* p = lds + (at ^ i) + c * IDX;
            return read_across<typename Frag<E>::type>(p, p + 4 * IDX);  // c + 4 trades as c does
        }
    }
    // how many of the 8 elements at index i and c = k lie inside i_n and c_n
    static __device__ __forceinline__ int inside(int64_t i, int64_t i_n, int64_t k, int64_t c_n) {
        const int64_t left = L == ALONG ? (i < i_n ? c_n - k : 0) : (k < c_n ? i_n - i : 0);
        return left >= 8 ? 8 : left > 0 ? (int)left : 0;
    }
    // The tile of `p` whose indices start at i0 (of i_n) and whose c at c0 (of c_n); outside: zero. All pieces are
    // asked for before any is looked at: a piece that is cut is read whole and masked, unless that leads past
    // `end`, the end of the tensor.
    static __device__ __forceinline__ void load(Raw<T> (&raw)[chunks], int tid, const T* p, int64_t pitch, int64_t i0,
                                                int64_t i_n, int64_t c0, int64_t c_n, const T* end) {
        const T* at[chunks];
        int valid[chunks];
#pragma unroll
        for (int n = 0; n < chunks; ++n) {
            int idx, c;
            place(tid, n, idx, c);
            valid[n] = inside(i0 + idx, i_n, c0 + c, c_n);
            at[n] = p + (L == ALONG ? (i0 + idx) * pitch + c0 + c : (c0 + c) * pitch + i0 + idx);
            raw[n] = Raw<T>{};
            if (valid[n] && at[n] + 8 <= end) __builtin_memcpy(&raw[n], at[n], sizeof(raw[n]));
        }
#pragma unroll
        for (int n = 0; n < chunks; ++n) {
            if (valid[n] == 8) continue;
            T e[8];
            __builtin_memcpy(e, &raw[n], sizeof(e));
            const bool short_end = valid[n] && at[n] + 8 > end;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (k >= valid[n]) e[k] = (T)0.0f;
                else if (short_end) e[k] = at[n][k];
            }
            __builtin_memcpy(&raw[n], e, sizeof(e));
        }
    }
    static __device__ __forceinline__ void store(E* lds, int tid, const Raw<T> (&raw)[chunks]) {
#pragma unroll
        for (int n = 0; n < chunks; ++n) {
            int idx, c;
            place(tid, n, idx, c);
            store8<T>(lds + offset(idx, c), plane, raw[n]);
        }
    }

    // load() and store() a piece at a time: the few registers of what runs once a tile
    static __device__ __forceinline__ void copy(E* lds, int tid, const T* p, int64_t pitch, int64_t i0, int64_t i_n,
                                                int64_t c0, int64_t c_n) {
#pragma unroll 1
        for (int n = 0; n < chunks; ++n) {
            int idx, c;
            place(tid, n, idx, c);
            const int64_t i = i0 + idx, k = c0 + c;
            const int valid = inside(i, i_n, k, c_n);
            store8<T>(lds + offset(idx, c), plane,
                      load8<T>(valid ? p + (L == ALONG ? i * pitch + k : k * pitch + i) : p, valid));
        }
    }

    // Tiles whose c lie inside are read without a branch from addresses found once: indices past the
    // end read the last ones instead, whose results nobody stores. Not so where such an end cuts a
    // piece (`whole` is false): those tiles go through load().
    static __device__ __forceinline__ bool whole(int64_t i0, int64_t i_n) {
        return L == ALONG || i0 + IDX <= i_n || i_n % 8 == 0;
    }
    struct Walk {
        const T* at[chunks];
        int64_t step;  // elements from one tile to the next

        __device__ __forceinline__ Walk(int tid, const T* p, int64_t pitch, int64_t i0, int64_t i_n, int64_t c0) {
#pragma unroll
            for (int n = 0; n < chunks; ++n) {
                int idx, c;
                place(tid, n, idx, c);
                set(n, p, pitch, i0 + idx, i_n, c0 + c);
            }
            step = L == ALONG ? BK : BK * pitch;
        }
        __device__ __forceinline__ void set(int n, const T* p, int64_t pitch, int64_t i, int64_t i_n, int64_t k) {
            if constexpr (L == ALONG) at[n] = p + (i < i_n ? i : i_n - 1) * pitch + k;
            else at[n] = p + k * pitch + (i < i_n ? i : i_n - 8);
        }
        __device__ __forceinline__ void next(Raw<T> (&raw)[chunks]) {
#pragma unroll
            for (int n = 0; n < chunks; ++n) {
                __builtin_memcpy(&raw[n], at[n], sizeof(raw[n]));
                at[n] += step;
            }
        }
    };

    // The same straight into LDS (16-bit types, 16-byte aligned operands): a wave's instruction fills 1 KB in
    // a row, so the pieces are permuted by the addresses that the lanes read, bytes from a uniform base.
    struct Direct {
        unsigned at[chunks];
        unsigned wave_at;  // the wave's part of an instruction's pieces in LDS, bytes
        const T* base;
        int64_t step;

        int end, pitch_;

        __device__ __forceinline__ Direct(const T* p, int64_t pitch, int64_t i0, int64_t i_n, int64_t c0) {
            wave_at = __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * 1024;
            end = i_n - i0 < IDX ? (int)(i_n - i0) : IDX;  // at least 1; ACROSS: at least 8
            pitch_ = (int)pitch;
#pragma unroll
            for (int n = 0; n < chunks; ++n) at[n] = reach(n, BK);
            base = L == ALONG ? p + i0 * pitch + c0 : p + c0 * pitch + i0;
            step = L == ALONG ? BK : BK * pitch;
        }
        // bytes from the base to piece n of the wave's lanes, with c kept inside the first `left` (ALONG: at
        // least 8 of them)
        __device__ __forceinline__ unsigned reach(int n, int left) const {
            const int slot = n * THREADS + threadIdx.x;  // 16-byte piece of the tile in LDS
            if constexpr (L == ALONG) {
                const int idx = slot / (BK / 8), c = ((slot % (BK / 8)) ^ turn(idx)) * 8;
                return (unsigned)((idx < end ? idx : end - 1) * pitch_ + (c < left ? c : left - 8)) * 2;
            } else {
                const int c = slot / (IDX / 8), s = slot % (IDX / 8);
                const int idx = ((s / 2) ^ trade(c)) * 16 + s % 2 * 8;
                return (unsigned)((c < left ? c : left - 1) * pitch_ + (idx < end ? idx : end - 8)) * 2;
            }
        }
        // (Written out, as the compiler would wait for every load before it reads any stage; m0, which holds the place in
        // LDS, is an operand, so that the compiler knows what is in it. The wait states are the ones that m0 needs before
        // a load to LDS and that a scalar from a vector lane needs before a load.)
        template <typename F>
        __device__ __forceinline__ void send(E* lds, F&& from) const {
            typedef __attribute__((address_space(3))) E* lptr;
            const unsigned to = __builtin_amdgcn_readfirstlane((unsigned)(unsigned long long)(lptr)lds + wave_at);
            const int64_t origin = scalar((int64_t)base);
#pragma unroll
            for (int n = 0; n < chunks; ++n)
                asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1"
                             :
                             : "v"(from(n)), "s"(origin), "{m0}"(to + n * THREADS * 16)
                             : "memory");
        }
        __device__ __forceinline__ void next(E* lds) {
            send(lds, [&](int n) { return at[n]; });
            base += step;
        }
        // the last `left` of c, fewer than BK: what lies past them holds copies until cut() clears it
        __device__ __forceinline__ void last(E* lds, int left) const {
            send(lds, [&](int n) { return reach(n, left); });
        }
        static __device__ __forceinline__ void cut(E* lds, int left) {
#pragma unroll 1
            for (int n = 0; n < chunks; ++n) {
                int idx, c;
                place(threadIdx.x, n, idx, c);
                if (c >= left) *reinterpret_cast<u32x4*>(lds + offset(idx, c)) = u32x4{};
            }
        }
    };
};

// ---------------------------------------------------------------------------------------
// the tile product
// ---------------------------------------------------------------------------------------
// acc += R * B over the BK of c that a stage holds, for the WR x WN part of the tile at (r0, n0)
template <typename T, typename TR, typename TB, int BK, int NR, int NN>
__device__ __forceinline__ void multiply(const typename Stage<T>::elem* lr, const typename Stage<T>::elem* lb, int r0,
                                         int n0, f32x4 (&acc)[NR][NN]) {
    typedef typename Stage<T>::elem E;
    constexpr int P = Stage<T>::planes;
    unsigned at_r = TR::at(r0), at_b = TB::at(n0);
#pragma unroll
    for (int c = 0; c < BK; c += 32) {
        // kept from being found once for every fragment and stage: more registers than there are
        asm volatile("" : "+v"(at_r), "+v"(at_b));
        typename Frag<E>::type fb[P][NN];
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int j = 0; j < NN; ++j) fb[p][j] = TB::frag(lb + p * TB::plane, at_b, j * 16, c);
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            typename Frag<E>::type fr[P];
#pragma unroll
            for (int p = 0; p < P; ++p) fr[p] = TR::frag(lr + p * TR::plane, at_r, i * 16, c);
#pragma unroll
            for (int j = 0; j < NN; ++j) {
                if constexpr (P == 1) {
                    acc[i][j] = Frag<E>::mfma(fb[0][j], fr[0], acc[i][j]);
                } else {  // smallest products first
                    acc[i][j] = Frag<E>::mfma(fb[2][j], fr[0], acc[i][j]);
                    acc[i][j] = Frag<E>::mfma(fb[1][j], fr[1], acc[i][j]);
                    acc[i][j] = Frag<E>::mfma(fb[0][j], fr[2], acc[i][j]);
                    acc[i][j] = Frag<E>::mfma(fb[1][j], fr[0], acc[i][j]);
                    acc[i][j] = Frag<E>::mfma(fb[0][j], fr[1], acc[i][j]);
                    acc[i][j] = Frag<E>::mfma(fb[0][j], fr[0], acc[i][j]);
                }
            }
        }
    }
}

// Every load that a wave has sent to LDS is there, and every wave of the workgroup is here.
__device__ __forceinline__ void arrive() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// A workgroup's BR x BN tile, its waves side by side. DIRECT: the operands go straight to LDS, into
// two stages in turn, of which one is on its way while the other is multiplied. Else through
// registers (any alignment, fp32's split) into one.
template <typename T, Layout LR, Layout LB, int BR, int BN, int THREADS, bool DIRECT>
struct Product {
    typedef typename Stage<T>::elem E;
    static constexpr int BK = Stage<T>::bk, P = Stage<T>::planes;
    typedef Tile<T, LR, BR, BK, THREADS> TR;
    typedef Tile<T, LB, BN, BK, THREADS> TB;
    static constexpr int waves_r = 2, waves_n = THREADS / 64 / waves_r;
    static constexpr int WR = BR / waves_r, WN = BN / waves_n;
    static constexpr int NR = WR / 16, NN = WN / 16;
    static constexpr int stage = P * (TR::plane + TB::plane);   // elements

    static __device__ __forceinline__ void step(const E* lds, f32x4 (&acc)[NR][NN]) {
        const int wave = threadIdx.x / 64;
        multiply<T, TR, TB, BK, NR, NN>(lds, lds + P * TR::plane, wave / waves_n * WR, wave % waves_n * WN, acc);
    }

    // acc += R[r0.., c] * B[n0.., c] over c in [c_lo, c_hi). `seen(stage of B)` is called on each stage. r_end and
    // b_end: the ends of the tensors.
    template <typename F>
    static __device__ __forceinline__ void run(E* s0, E* s1, f32x4 (&acc)[NR][NN], const T* r, int64_t r_pitch,
                                               int64_t r0, int64_t r_n, const T* r_end, const T* b, int64_t b_pitch,
                                               int64_t n0, int64_t b_n, const T* b_end, int64_t c_lo, int64_t c_hi,
                                               F&& seen) {
        const int tid = threadIdx.x;
        if (c_lo >= c_hi) return;
        int64_t c = c_lo;
        const bool whole = TR::whole(r0, r_n) && TB::whole(n0, b_n);
        const int full = __builtin_amdgcn_readfirstlane(whole ? (int)((c_hi - c_lo) / BK) : 0);
        c = c_lo + (int64_t)full * BK;
        if constexpr (DIRECT) {
            // a rest of c that cuts no piece goes the same way as the whole stages
            const int rest = __builtin_amdgcn_readfirstlane(
                whole && ((LR == ACROSS && LB == ACROSS) || (c_hi - c) % 8 == 0) ? (int)(c_hi - c) : 0);
            const int stages = full + (rest > 0);
            if (stages > 0) {
                typename TR::Direct wr(r, r_pitch, r0, r_n, c_lo);
                typename TB::Direct wb(b, b_pitch, n0, b_n, c_lo);
                auto fill = [&](int k, E* s) {
                    if (k < full) {
                        wr.next(s);
                        wb.next(s + TR::plane);
                    } else {
                        wr.last(s, rest);
                        wb.last(s + TR::plane, rest);
                    }
                };
                fill(0, s0);
                auto turn = [&](int k, E* now, E* next) {
                    arrive();  // stage `now` is filled, and nobody reads `next` any more
                    if (k + 1 < stages) fill(k + 1, next);
                    seen(now + TR::plane);
                    step(now, acc);
                };
                int k = 0;
                for (; k + 2 <= full; k += 2) {
                    turn(k, s0, s1);
                    turn(k + 1, s1, s0);
                }
                // (no exit from the middle of the loop: the accumulators would have a copy per exit)
                if (k < full) turn(k, s0, s1);
                if (rest > 0) {
                    E* s = full % 2 ? s1 : s0;
                    arrive();
                    TR::Direct::cut(s, rest);
                    TB::Direct::cut(s + TR::plane, rest);
                    __syncthreads();
                    seen(s + TR::plane);
                    step(s, acc);
                }
                c += rest;
            }
            for (; c < c_hi; c += BK) {  // tiles at an end, or a rest of c, that cuts a piece
                __syncthreads();
                TR::copy(s0, tid, r, r_pitch, r0, r_n, c, c_hi);
                TB::copy(s0 + TR::plane, tid, b, b_pitch, n0, b_n, c, c_hi);
                __syncthreads();
                seen(s0 + TR::plane);
                step(s0, acc);
            }
        } else {
            Raw<T> rr[TR::chunks], rb[TB::chunks];
            auto put = [&] {
                __syncthreads();  // the last step's reads are done
                TR::store(s0, tid, rr);
                TB::store(s0 + P * TR::plane, tid, rb);
                __syncthreads();
            };
            if (full > 0) {
                typename TR::Walk wr(tid, r, r_pitch, r0, r_n, c_lo);
                typename TB::Walk wb(tid, b, b_pitch, n0, b_n, c_lo);
                wr.next(rr);
                wb.next(rb);
                for (int k = 0; k < full; ++k) {
                    put();
                    if (k + 1 < full) {
                        wr.next(rr);
                        wb.next(rb);
                    }
                    seen(s0 + P * TR::plane);
                    step(s0, acc);
                }
            }
            for (; c < c_hi; c += BK) {
                TR::load(rr, tid, r, r_pitch, r0, r_n, c, c_hi, r_end);
                TB::load(rb, tid, b, b_pitch, n0, b_n, c, c_hi, b_end);
                put();
                seen(s0 + P * TR::plane);
                step(s0, acc);
            }
        }
    }

    // this lane's results: four columns from col(j) on of row row(i)
    static __device__ __forceinline__ int row(int i) {
        return threadIdx.x / 64 / waves_n * WR + i * 16 + threadIdx.x % 16;
    }
    static __device__ __forceinline__ int col(int j) {
        return threadIdx.x / 64 % waves_n * WN + j * 16 + threadIdx.x % 64 / 16 * 4;
    }
};

__device__ __forceinline__ bool finite(float v) { return __builtin_fabsf(v) <= 3.402823466e38f; }

template <typename T>
__device__ __forceinline__ void store4(T* p, const f32x4& v, int valid) {
    if (valid >= 4) {
        T e[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) e[k] = (T)v[k];
        __builtin_memcpy(p, e, sizeof(e));
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k < valid) p[k] = (T)v[k];
    }
}

// Is a result of this wave not finite? (0 * v is not a number then.) The split of an fp32 infinity or NaN
// gives none of the results that a sum of products has, nor does one that overflows in its pieces.
template <int NR, int NN>
__device__ __forceinline__ bool any_lost(const f32x4 (&acc)[NR][NN]) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int j = 0; j < NN; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) s = __builtin_fmaf(acc[i][j][k], 0.0f, s);
    return __any(!(s == 0.0f));
}

// One result of the forward or input gradient from the operands.
template <typename T, Layout LB>
__device__ float product_again(const GroupedArgs& a, const T* b, int64_t row, int64_t col) {
    const T* r = (const T*)a.r + row * a.r_pitch;
    float s = 0.0f;
    for (int c = 0; c < a.cc; ++c)
        s = __builtin_fmaf((float)r[c], (float)(LB == ALONG ? b[col * a.b_pitch + c] : b[c * a.b_pitch + col]), s);
    return s;
}

__device__ __forceinline__ int valid4(int64_t col, int64_t cols) {
    return col >= cols ? 0 : cols - col < 4 ? (int)(cols - col) : 4;
}

// the bias of four columns, zeros where there is none
template <typename T>
__device__ __forceinline__ f32x4 bias4(const GroupedArgs& a, const Item& it, int64_t col) {
    f32x4 v = {};
    const int valid = valid4(col, a.cols);
    if (!a.bias || it.group >= a.groups || !valid) return v;
    const T* p = (const T*)a.bias + (int64_t)it.group * a.cols + col;
    if (valid == 4) {
        T e[4];
        __builtin_memcpy(e, p, sizeof(e));
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = (float)e[k];
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k < valid) v[k] = (float)p[k];
    }
    return v;
}

// One tile of the forward (LB = ACROSS) or input gradient (LB = ALONG).
template <typename T, Layout LB, int BR, int BN, int THREADS, bool DIRECT>
__device__ __forceinline__ void rows_tile(const GroupedArgs& a, const Item& it, int64_t r0, int64_t n0,
                                          typename Stage<T>::elem* s0, typename Stage<T>::elem* s1) {
    typedef Product<T, ALONG, LB, BR, BN, THREADS, DIRECT> X;
    f32x4 acc[X::NR][X::NN] = {};
    const T* b = (const T*)a.b + (int64_t)it.group * a.b_group;
    if (it.group < a.groups)
        X::run(s0, s1, acc, (const T*)a.r, a.r_pitch, r0, it.hi, (const T*)a.r_end, b, a.b_pitch, n0, a.cols,
               (const T*)a.b_end, 0, a.cc, [](auto*) {});
    if constexpr (sizeof(T) == 4) {
        if (it.group < a.groups && any_lost(acc)) {
#pragma unroll
            for (int i = 0; i < X::NR; ++i)
#pragma unroll
                for (int j = 0; j < X::NN; ++j)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (r0 + X::row(i) < it.hi && n0 + X::col(j) + k < a.cols && !finite(acc[i][j][k]))
                            acc[i][j][k] = product_again<T, LB>(a, b, r0 + X::row(i), n0 + X::col(j) + k);
        }
    }
    f32x4 add[X::NN];
#pragma unroll
    for (int j = 0; j < X::NN; ++j) add[j] = bias4<T>(a, it, n0 + X::col(j));
#pragma unroll
    for (int i = 0; i < X::NR; ++i) {
        const int64_t row = r0 + X::row(i);
        if (row >= it.hi) continue;
#pragma unroll
        for (int j = 0; j < X::NN; ++j) {
            const int64_t col = n0 + X::col(j);
            const int valid = valid4(col, a.cols);
            if (valid) store4<T>((T*)a.out + row * a.cols + col, acc[i][j] + add[j], valid);
        }
    }
}

// A workgroup per row tile and column tile. At 256 rows a group's last tile of at most 128 rows costs half, at
// 128 columns a last one of at most 64 (36k rows, 6 groups, 602 x 51 fp16 41 us, 33 so).
template <typename T, Layout LB, int BR, int BN, int THREADS, bool DIRECT>
__global__ __launch_bounds__(THREADS, 2) void grouped_rows_kernel(GroupedArgs a) {
    typedef Product<T, ALONG, LB, BR, BN, THREADS, DIRECT> X;
    __shared__ __attribute__((aligned(16))) typename X::E s0[X::stage];
    __shared__ __attribute__((aligned(16))) typename X::E s1[DIRECT ? X::stage : 8];
    const int bid = tile_of(a);
    const Item it = find_item<THREADS>(a, bid / a.col_tiles, BR, 0, true);
    if (it.group < 0) return;
    const int64_t n0 = (int64_t)(bid % a.col_tiles) * BN;
    const int64_t r0 = it.lo + (int64_t)it.part * BR;
    if constexpr (BR == 256) {
        if (it.hi - r0 <= BR / 2) {
            rows_tile<T, LB, BR / 2, BN, THREADS, DIRECT>(a, it, r0, n0, s0, s1);
            return;
        }
    } else if constexpr (THREADS == 256) {
        if (a.cols - n0 <= BN / 2) {
            rows_tile<T, LB, BR, BN / 2, THREADS, DIRECT>(a, it, r0, n0, s0, s1);
            return;
        }
    }
    rows_tile<T, LB, BR, BN, THREADS, DIRECT>(a, it, r0, n0, s0, s1);
}

// The same for few rows a group, where the time goes into reading the weights: tiles of 32 rows and 64
// columns, and the WAVES waves of a workgroup split c, each with a stage of its own and two more in
// its registers on their way from memory, so that no wave waits for another before the end.
template <typename T, Layout LB, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void grouped_few_rows_kernel(GroupedArgs a) {
    constexpr int BR = 32, BN = 64, NR = BR / 16, NN = BN / 16, P = Stage<T>::planes, BK = Stage<T>::bk;
    typedef typename Stage<T>::elem E;
    typedef Tile<T, ALONG, BR, BK, 64> TR;
    typedef Tile<T, LB, BN, BK, 64> TB;
    constexpr int stage = P * (TR::plane + TB::plane);
    __shared__ __attribute__((aligned(16))) E lds[WAVES * stage];
    static_assert(sizeof(E) * stage >= BR * BN * sizeof(float), "a wave's results fit its stage");
    const Item it = find_item<WAVES * 64>(a, blockIdx.x / a.col_tiles, BR, 0, true);
    if (it.group < 0) return;
    const int64_t n0 = (int64_t)(blockIdx.x % a.col_tiles) * BN;
    const int64_t r0 = it.lo + (int64_t)it.part * BR;
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const T* r = (const T*)a.r;
    const T* b = (const T*)a.b + (int64_t)it.group * a.b_group;
    E* s = lds + wave * stage;
    f32x4 acc[NR][NN] = {};
    if (it.group < a.groups) {
        const int steps = (a.cc + BK - 1) / BK, share = (steps + WAVES - 1) / WAVES;
        const int64_t c_lo = (int64_t)wave * share * BK;
        const int64_t c_hi = c_lo + (int64_t)share * BK < a.cc ? c_lo + (int64_t)share * BK : a.cc;
        Raw<T> rr[2][TR::chunks], rb[2][TB::chunks];
        auto put = [&](int q) {  // the wave's LDS instructions run in order: no barrier
            TR::store(s, lane, rr[q]);
            TB::store(s + P * TR::plane, lane, rb[q]);
            __builtin_amdgcn_wave_barrier();
        };
        auto use = [&] {
            multiply<T, TR, TB, BK, NR, NN>(s, s + P * TR::plane, 0, 0, acc);
            __builtin_amdgcn_wave_barrier();
        };
        int64_t c = c_lo;
        if (TB::whole(n0, a.cols) && c_lo < c_hi) {
            const int64_t full = (c_hi - c_lo) / BK;
            c = c_lo + full * BK;
            typename TR::Walk wr(lane, r, a.r_pitch, r0, it.hi, c_lo);
            typename TB::Walk wb(lane, b, a.b_pitch, n0, a.cols, c_lo);
            auto get = [&](int q) {
                wr.next(rr[q]);
                wb.next(rb[q]);
            };
            if (full > 0) get(0);
            if (full > 1) get(1);
            int64_t k = 0;
            for (; k + 2 <= full; k += 2) {
                put(0);
                if (k + 2 < full) get(0);
                use();
                put(1);
                if (k + 3 < full) get(1);
                use();
            }
            if (k < full) {
                put(0);
                use();
            }
        }
        for (; c < c_hi; c += BK) {
            TR::load(rr[0], lane, r, a.r_pitch, r0, it.hi, c, c_hi, (const T*)a.r_end);
            TB::load(rb[0], lane, b, a.b_pitch, n0, a.cols, c, c_hi, (const T*)a.b_end);
            put(0);
            use();
        }
    }
    // the waves' parts, added in order
    float* mine = reinterpret_cast<float*>(s);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int j = 0; j < NN; ++j)
            *reinterpret_cast<f32x4*>(mine + (i * 16 + lane % 16) * BN + j * 16 + lane / 16 * 4) = acc[i][j];
    __syncthreads();
    for (int q = threadIdx.x; q < BR * BN / 4; q += WAVES * 64) {
        const int ir = q / (BN / 4), in = q % (BN / 4) * 4;
        f32x4 v = {};
        for (int w = 0; w < WAVES; ++w)
            v += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + w * stage) + ir * BN + in);
        const int64_t row = r0 + ir, col = n0 + in;
        const int valid = valid4(col, a.cols);
        if (row >= it.hi || !valid) continue;
        if constexpr (sizeof(T) == 4) {
            if (it.group < a.groups && !finite(v[0] + v[1] + v[2] + v[3]))
                for (int k = 0; k < valid; ++k)
                    if (!finite(v[k])) v[k] = product_again<T, LB>(a, b, row, col + k);
        }
        store4<T>((T*)a.out + row * a.cols + col, v + bias4<T>(a, it, col), valid);
    }
}

// weight gradient: a workgroup per chunk of a group's rows and tile of the weight. A group of one
// chunk is written as it is; the chunks of a longer one leave fp32 slabs for the kernel below.
// (Through registers a CU holds three workgroups of 168 registers and one stage each: 41k rows, 147 groups, 145 x 203
// fp16 with the bias gradient 48 us at two, 32 at three.)
template <typename T, int BR, int BN, int THREADS, bool DIRECT, bool BIAS>
__global__ __launch_bounds__(THREADS, DIRECT ? 2 : 3) void grouped_wgrad_kernel(GroupedArgs a) {
    typedef Product<T, ACROSS, ACROSS, BR, BN, THREADS, DIRECT> X;
    __shared__ __attribute__((aligned(16))) typename X::E s0[X::stage];
    __shared__ __attribute__((aligned(16))) typename X::E s1[DIRECT ? X::stage : 8];
    const int tiles = a.row_tiles * a.col_tiles;
    const int bid = tile_of(a);
    const int id = bid / tiles, tile = bid % tiles;
    const Item it = find_item<THREADS>(a, id, a.chunk, 1, false);
    if (it.group < 0) return;
    const int64_t r0 = (int64_t)(tile / a.col_tiles) * BR, n0 = (int64_t)(tile % a.col_tiles) * BN;
    const int64_t c_lo = it.lo + (int64_t)it.part * a.chunk;
    const int64_t c_hi = c_lo + a.chunk < it.hi ? c_lo + a.chunk : it.hi;
    f32x4 acc[X::NR][X::NN] = {};
    float col_sum[8] = {};  // of the columns of this thread's pieces: the same in every piece
    const bool want_b = BIAS && r0 == 0;
    const T* r = (const T*)a.r;
    const T* b = (const T*)a.b;
    X::run(s0, s1, acc, r, a.r_pitch, r0, a.out_rows, (const T*)a.r_end, b, a.b_pitch, n0, a.cols, (const T*)a.b_end, c_lo,
           c_hi, [&](auto* stage) {
        if (!want_b) return;
#pragma unroll
        for (int n = 0; n < X::TB::chunks; ++n) {
            int idx, c;
            X::TB::place(threadIdx.x, n, idx, c);
            typename VecOf<typename X::E, 8>::type e[X::P];
#pragma unroll
            for (int p = 0; p < X::P; ++p)
                e[p] = *reinterpret_cast<const typename VecOf<typename X::E, 8>::type*>(stage + p * X::TB::plane +
                                                                                       X::TB::offset(idx, c));
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if constexpr (X::P == 1) col_sum[k] += (float)e[0][k];
                else col_sum[k] += ((float)e[X::P - 1][k] + (float)e[1][k]) + (float)e[0][k];  // the value, exactly
            }
        }
    });
    const int64_t size = (int64_t)a.out_rows * a.cols;
    const int64_t slab = size + (BIAS ? a.cols : 0);
    // the slab at the part's place: there are a.items of them, and no group, wherever ptr leads, has a place behind them
    float* part = it.parts > 1 ? a.slabs + (place_of(it.lo, a.chunk, it.group) + it.part) * slab : nullptr;
    auto again = [&](int64_t row, int64_t col) {
        float v = 0.0f;
        for (int64_t c = c_lo; c < c_hi; ++c)
            v = __builtin_fmaf((float)r[c * a.r_pitch + row], (float)b[c * a.b_pitch + col], v);
        return v;
    };
    if constexpr (sizeof(T) == 4) {
        if (any_lost(acc)) {
#pragma unroll
            for (int i = 0; i < X::NR; ++i)
#pragma unroll
                for (int j = 0; j < X::NN; ++j)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (r0 + X::row(i) < a.out_rows && n0 + X::col(j) + k < a.cols && !finite(acc[i][j][k]))
                            acc[i][j][k] = again(r0 + X::row(i), n0 + X::col(j) + k);
        }
    }
#pragma unroll
    for (int i = 0; i < X::NR; ++i) {
        const int64_t row = r0 + X::row(i);
        if (row >= a.out_rows) continue;
#pragma unroll
        for (int j = 0; j < X::NN; ++j) {
            const int64_t col = n0 + X::col(j);
            const int valid = valid4(col, a.cols);
            if (!valid) continue;
            if (part) store4<float>(part + row * a.cols + col, acc[i][j], valid);
            else store4<T>((T*)a.out + (int64_t)it.group * size + row * a.cols + col, acc[i][j], valid);
        }
    }
    if constexpr (!BIAS) return;
    if (!want_b) return;
    // the threads whose pieces have the same columns, in order
    constexpr int teams = THREADS / (BN / 8);
    float* sums = reinterpret_cast<float*>(s0);
    static_assert(sizeof(s0) >= teams * BN * sizeof(float), "the column sums fit the stage");
    __syncthreads();
    const int team = threadIdx.x / (BN / 8), c8 = threadIdx.x % (BN / 8) * 8;
#pragma unroll
    for (int k = 0; k < 8; ++k) sums[team * BN + c8 + k] = col_sum[k];
    __syncthreads();
    for (int c = threadIdx.x; c < BN && n0 + c < a.cols; c += THREADS) {
        float s = sums[c];
        for (int q = 1; q < teams; ++q) s += sums[q * BN + c];
        if constexpr (sizeof(T) == 4) {  // an infinity's pieces are not numbers
            if (!finite(s)) {
                s = 0.0f;
                for (int64_t i = c_lo; i < c_hi; ++i) s += b[i * a.b_pitch + n0 + c];
            }
        }
        if (part) part[size + n0 + c] = s;
        else ((T*)a.dbias)[(int64_t)it.group * a.cols + n0 + c] = (T)s;
    }
}

// dW[g] (and db[g]) of the groups cut in chunks: their slabs added in order
template <typename T>
__global__ __launch_bounds__(kGlThreads) void grouped_slabs_kernel(GroupedArgs a, int pieces) {
    const int g = blockIdx.x / pieces;
    const int64_t lo = ptr_at(a, g), hi = ptr_at(a, g + 1);
    if (hi - lo <= a.chunk) return;
    const int64_t first = place_of(lo, a.chunk, g);
    // (all of them are inside the workspace, wherever ptr leads: first + parts <= hi / chunk + 1 + g <= items)
    const int64_t parts = (hi - lo + a.chunk - 1) / a.chunk;
    const int64_t size = (int64_t)a.out_rows * a.cols, slab = size + (a.dbias ? a.cols : 0);
    const float* p = a.slabs + first * slab;
    for (int64_t e = ((int64_t)(blockIdx.x % pieces) * kGlThreads + threadIdx.x) * 4; e < slab;
         e += (int64_t)pieces * kGlThreads * 4) {
        const int valid = slab - e < 4 ? (int)(slab - e) : 4;
        f32x4 s = {};
        int64_t k = 0;
        if (valid == 4) {
            for (; k + 8 <= parts; k += 8) {  // eight slabs on their way at once, added in order
                f32x4 v[8];
#pragma unroll
                for (int q = 0; q < 8; ++q) __builtin_memcpy(&v[q], p + (k + q) * slab + e, 16);
#pragma unroll
                for (int q = 0; q < 8; ++q) s += v[q];
            }
        }
        for (; k < parts; ++k)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (q < valid) s[q] += p[k * slab + e + q];
        if (e + 4 <= size) {
            store4<T>((T*)a.out + (int64_t)g * size + e, s, 4);
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (q >= valid) break;
                if (e + q < size) ((T*)a.out)[(int64_t)g * size + e + q] = (T)s[q];
                else ((T*)a.dbias)[(int64_t)g * a.cols + e + q - size] = (T)s[q];
            }
        }
    }
}

// ---------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------
constexpr int kTile = 128;
// Tiles of 256 x 256 read half as many bytes a product as tiles of 128 x 128, which the CUs' 64 bytes a
// clock from L2 hold to half the matrix rate; but a CU has one at a time, so that they need rounds
// enough: bf16, us for forward / input / weight gradient with 128 and 256:
//   32768 rows, 32 groups, 2048 x 4096   695 / 657 / 802    535 / 502 / 622
//   24576 rows, 8 groups, 1024 x 1024     73 /  81 /  74     70 /  70 /  74
//   20480 rows, 4 groups, 1024 x 1024     62 /  62 /  86     68 /  67 /  86
constexpr int64_t kBigTiles = 384;
// Up to this many rows a group on average grouped_few_rows_kernel runs, and up to this many of its tiles: larger
// tiles would leave most CUs idle, each with all of c to go through. us with tiles of 128 x 128 and with these, one
// group:
//   bf16, 512 rows, 2048 x 2048    24 / 16       fp32    86 / 45    (512 tiles of 32 x 64)
//   bf16, 2048 rows, 2048 x 256    23 / 11               86 / 28    (256)
//   bf16, 512 rows, 256 x 2048    7.9 / 7.7            16.5 / 11.7  (512)
//   bf16, 8192 rows, 256 x 256      8 / 13               18 / 21    (1024)
constexpr int kFewRows = 32, kFewTiles = 512;

// Rows of a chunk of the weight gradient: whole groups where the weight alone has tiles enough to
// fill the chip, else as many rows as leave two workgroups per CU (more chunks are more slabs to write and
// add: 208k rows, 237 groups, 128 x 128 bf16 39 us, 48 with four), and no fewer than 256 (128 of fp32: 2725 rows, 3
// groups, 216 x 256 16 us, 22 with 256). With many tiles of fp32, whose workgroups
// run longer, uneven groups want four (20k rows, 8 groups, 1024 x 1024: 272 us, 342 with two).
int64_t wgrad_chunk(int64_t rows, int64_t groups, int64_t k, int64_t n, int eb) {
    const int64_t tiles = ((k + kTile - 1) / kTile) * ((n + kTile - 1) / kTile);
    const int64_t want = (eb == 4 && tiles > 4 ? 1024 : 512) / tiles;  // chunks over all groups
    if (want <= groups || rows == 0) return std::max<int64_t>(rows, 1);
    const int64_t c = (rows + want - 1) / want;
    return std::max<int64_t>(eb == 4 ? 128 : 256, (c + 63) / 64 * 64);
}

int64_t wgrad_items(int64_t rows, int64_t groups, int64_t chunk) { return rows / chunk + groups; }

int32_t check_grouped(int64_t rows, int64_t groups, int64_t k, int64_t n, int32_t dtype, int32_t ptr_bits) {
    if (rows < 0 || groups < 1 || k < 1 || n < 1)
        return arg_error("grouped linear: rows < 0, or fewer than one group, input or output column");
    if (!dtype_bytes(dtype)) return arg_error("grouped linear: unknown dtype");
    if (ptr_bits != 32 && ptr_bits != 64) return arg_error("grouped linear: group_ptr is int32 or int64");
    if (k > (1 << 24) || n > (1 << 24) || groups > (1 << 24) || rows > (int64_t{1} << 40))
        return unsupported("grouped linear: more than 2^24 columns or groups, or 2^40 rows");
    return MPGNN_OK;
}

// operands that go straight to LDS: 16-bit, their rows and groups at multiples of 16 bytes
template <typename T>
bool direct_ok(const GroupedArgs& a) {
    constexpr int64_t reach = 1 << 20;  // a lane's offset within a tile of 256 rows fits 32 bits
    return sizeof(T) == 2 && aligned16(a.r) && aligned16(a.b) && a.r_pitch % 8 == 0 && a.b_pitch % 8 == 0 &&
           a.b_group % 8 == 0 && a.r_pitch <= reach && a.b_pitch <= reach;
}

// A launch has at most 2^32 - 1 threads in a dimension.
constexpr char kTooMany[] = "grouped linear: more tiles (rows / 32 to 256 + groups, times column tiles) than a launch has "
                            "workgroups";
bool fits_launch(int64_t blocks, int threads) { return blocks <= (int64_t)UINT32_MAX / threads; }

template <typename T, Layout LB, int WAVES>
void launch_few(GroupedArgs a, unsigned blocks, hipStream_t strm) {
    hipLaunchKernelGGL((grouped_few_rows_kernel<T, LB, WAVES>), dim3(blocks), dim3(WAVES * 64), 0, strm, a);
}

template <typename T, Layout LB, int TILE, int THREADS, bool DIRECT>
void launch_rows(GroupedArgs a, unsigned blocks, hipStream_t strm) {
    hipLaunchKernelGGL((grouped_rows_kernel<T, LB, TILE, TILE, THREADS, DIRECT>), dim3(blocks), dim3(THREADS), 0, strm,
                       a);
}

// GroupedArgs::run for `blocks` tiles of which `sharing` in a row read the same rows, but no more than leave each
// XCD eight runs of the `sure` tiles that there are whatever the groups' sizes. Returns the blocks to launch, whole
// turns over the XCDs. Forward / input gradient in us with runs of one tile and with these:
//   24k rows, 1 group, 1041 x 962 fp16     139 / 114    126 /  91
//   56k rows, 32 groups, 3120 x 584 fp16   435 / 388    354 / 351
//   262k rows, 19 groups, 168 x 792 fp16   324 / 184    256 / 184
int64_t set_run(GroupedArgs& a, int64_t blocks, int64_t sharing, int64_t sure) {
    a.run = (int32_t)std::max<int64_t>(1, std::min(sharing, sure / 64));
    const int64_t turn = 8 * (int64_t)a.run;
    return (blocks + turn - 1) / turn * turn;
}

// columns that tiles of 256 cover without much more padding than tiles of 128
bool big_cols(int64_t n) { return n % 256 == 0 || n % 256 > 128 || n >= 1024; }

template <typename T, Layout LB>
int32_t rows_product(GroupedArgs a, hipStream_t strm) {
    const bool few = a.rows <= (int64_t)kFewRows * a.groups ||
                     (a.rows / 32 * ((a.cols + 63) / 64) <= kFewTiles && (sizeof(T) == 4 || a.cc > 128));
    bool direct = false, big = false;
    if constexpr (sizeof(T) == 2) {
        direct = !few && direct_ok<T>(a);
        big = direct && big_cols(a.cols) && a.rows >= 256 * (int64_t)a.groups &&
              a.rows / 256 * ((a.cols + 255) / 256) >= kBigTiles;
    }
    const int br = few ? 32 : big ? 256 : kTile, bn = few ? 64 : big ? 256 : kTile;
    a.col_tiles = (a.cols + bn - 1) / bn;
    int64_t blocks = (a.rows / br + a.groups + 2) * a.col_tiles;
    if (!few) blocks = set_run(a, blocks, 2 * a.col_tiles, a.rows / br * a.col_tiles);
    // workgroups that find rows: at most one per row and column tile. Up to one per CU a workgroup of the few-rows
    // kernel takes eight waves, to have as many bytes on their way (of which a CU holds one workgroup, two of four)
    const int64_t busy = std::min<int64_t>(a.rows, a.rows / br + a.groups) * a.col_tiles;
    const bool wide = few ? busy <= 256 : big || sizeof(T) == 4;
    if (!fits_launch(blocks, wide ? 512 : 256)) return unsupported(kTooMany);
    if (few) {
        if (wide) launch_few<T, LB, 8>(a, (unsigned)blocks, strm);
        else launch_few<T, LB, 4>(a, (unsigned)blocks, strm);
    } else if constexpr (sizeof(T) == 2) {
        if (big) launch_rows<T, LB, 256, 512, true>(a, (unsigned)blocks, strm);
        else if (direct) launch_rows<T, LB, kTile, 256, true>(a, (unsigned)blocks, strm);
        else launch_rows<T, LB, kTile, 256, false>(a, (unsigned)blocks, strm);
    } else {
        launch_rows<T, LB, kTile, 512, false>(a, (unsigned)blocks, strm);
    }
    return launch_status("grouped linear: the launch failed");
}

template <typename T>
int32_t rows_either(const GroupedArgs& a, bool dgrad, hipStream_t strm) {
    return dgrad ? rows_product<T, ALONG>(a, strm) : rows_product<T, ACROSS>(a, strm);
}

const void* end_of(const void* p, int64_t rows, int64_t pitch, int64_t width, int32_t dtype) {
    return rows < 1 ? p : (const char*)p + ((rows - 1) * pitch + width) * dtype_bytes(dtype);
}

int32_t rows_by_type(const GroupedArgs& a, int32_t dtype, bool dgrad, hipStream_t strm) {
    if (a.rows == 0) return MPGNN_OK;
    if (dtype == MPGNN_F32) return rows_either<float>(a, dgrad, strm);
    return dtype == MPGNN_BF16 ? rows_either<__bf16>(a, dgrad, strm) : rows_either<_Float16>(a, dgrad, strm);
}

template <typename T, int TILE, int THREADS, bool DIRECT>
int32_t launch_wgrad(GroupedArgs a, hipStream_t strm) {
    a.row_tiles = (a.out_rows + TILE - 1) / TILE;
    a.col_tiles = (a.cols + TILE - 1) / TILE;
    const int64_t tiles = (int64_t)a.row_tiles * a.col_tiles;
    const int64_t sure = std::max<int64_t>(a.rows / a.chunk, a.groups) * tiles;
    // Not for a few tiles, which gain nothing and need an even spread over the XCDs more (a chunk for each place
    // there is: 36k rows, 6 groups, 602 x 51 fp16 43 us, in runs 52), and not where an XCD gets whole columns of
    // tiles anyway but could not have all of a chunk's (8k rows, 8 groups, 512 x 2048 bf16 27 us, in runs 31).
    const bool spread = tiles <= 8 || (a.col_tiles % 8 == 0 && sure / 64 < tiles);
    const int64_t blocks = set_run(a, a.items * tiles, spread ? 1 : tiles, sure);
    if (!fits_launch(blocks, THREADS)) return unsupported(kTooMany);
    const dim3 grid((unsigned)blocks), block(THREADS);
    if constexpr (TILE == kTile) {
        if (a.dbias) {
            hipLaunchKernelGGL((grouped_wgrad_kernel<T, TILE, TILE, THREADS, DIRECT, true>), grid, block, 0, strm, a);
            return MPGNN_OK;
        }
    }
    hipLaunchKernelGGL((grouped_wgrad_kernel<T, TILE, TILE, THREADS, DIRECT, false>), grid, block, 0, strm, a);
    return MPGNN_OK;
}

template <typename T>
int32_t wgrad_product(GroupedArgs a, hipStream_t strm) {
    a.items = wgrad_items(a.rows, a.groups, a.chunk);
    int32_t st;
    if constexpr (sizeof(T) == 2) {
        const bool direct = direct_ok<T>(a);
        const int64_t tiles = (int64_t)((a.out_rows + 255) / 256) * ((a.cols + 255) / 256) * a.groups;
        // (with column sums the large tile has no registers left)
        if (direct && !a.dbias && big_cols(a.out_rows) && big_cols(a.cols) && a.rows >= 256 * (int64_t)a.groups && tiles >= kBigTiles)
            st = launch_wgrad<T, 256, 512, true>(a, strm);
        else if (direct) st = launch_wgrad<T, kTile, 256, true>(a, strm);
        else st = launch_wgrad<T, kTile, 256, false>(a, strm);
    } else {
        st = launch_wgrad<T, kTile, 512, false>(a, strm);
    }
    if (st != MPGNN_OK) return st;
    if (a.rows > a.chunk) {
        const int64_t slab = (int64_t)a.out_rows * a.cols + (a.dbias ? a.cols : 0);
        const int pieces = (int)std::min<int64_t>(256, (slab + kGlThreads * 4 - 1) / (kGlThreads * 4));
        hipLaunchKernelGGL(grouped_slabs_kernel<T>, dim3((unsigned)a.groups * pieces), dim3(kGlThreads), 0, strm, a,
                           pieces);
    }
    return launch_status("grouped linear: a launch failed");
}

}  // namespace
}  // namespace mpgnn

extern "C" int32_t mpgnn_grouped_linear_fwd(const void* x, int64_t rows, int64_t x_pitch, int32_t dtype,
                                            const void* weight, int64_t groups, int64_t k, int64_t n, const void* bias,
                                            const void* group_ptr, int32_t ptr_bits, void* out, void* stream) {
    using namespace mpgnn;
    int32_t st = check_grouped(rows, groups, k, n, dtype, ptr_bits);
    if (st != MPGNN_OK) return st;
    if (!weight || !group_ptr || (rows > 0 && (!x || !out)) || (rows > 1 && x_pitch < k))
        return arg_error("mpgnn_grouped_linear_fwd: a null pointer, or x's row pitch is below its width");
    GroupedArgs a{};
    a.r = x; a.r_pitch = x_pitch; a.b = weight; a.b_pitch = n; a.b_group = k * n; a.out = out; a.bias = bias;
    a.ptr = group_ptr; a.ptr64 = ptr_bits == 64; a.rows = rows; a.groups = (int32_t)groups; a.cc = (int32_t)k;
    a.cols = (int32_t)n;
    a.r_end = end_of(x, rows, x_pitch, k, dtype);
    a.b_end = end_of(weight, groups * k, n, n, dtype);
    return rows_by_type(a, dtype, false, static_cast<hipStream_t>(stream));
}

extern "C" int32_t mpgnn_grouped_linear_dgrad(const void* dy, int64_t rows, int64_t dy_pitch, int32_t dtype,
                                              const void* weight, int64_t groups, int64_t k, int64_t n,
                                              const void* group_ptr, int32_t ptr_bits, void* dx, void* stream) {
    using namespace mpgnn;
    int32_t st = check_grouped(rows, groups, k, n, dtype, ptr_bits);
    if (st != MPGNN_OK) return st;
    if (!weight || !group_ptr || (rows > 0 && (!dy || !dx)) || (rows > 1 && dy_pitch < n))
        return arg_error("mpgnn_grouped_linear_dgrad: a null pointer, or dy's row pitch is below its width");
    GroupedArgs a{};
    a.r = dy; a.r_pitch = dy_pitch; a.b = weight; a.b_pitch = n; a.b_group = k * n; a.out = dx;
    a.ptr = group_ptr; a.ptr64 = ptr_bits == 64; a.rows = rows; a.groups = (int32_t)groups; a.cc = (int32_t)n;
    a.cols = (int32_t)k;
    a.r_end = end_of(dy, rows, dy_pitch, n, dtype);
    a.b_end = end_of(weight, groups * k, n, n, dtype);
    return rows_by_type(a, dtype, true, static_cast<hipStream_t>(stream));
}

extern "C" int32_t mpgnn_grouped_linear_wgrad_workspace_bytes(int64_t rows, int64_t groups, int64_t k, int64_t n,
                                                              int64_t* bytes) {
    using namespace mpgnn;
    int32_t st = check_grouped(rows, groups, k, n, MPGNN_F32, 64);
    if (st != MPGNN_OK) return st;
    if (!bytes) return arg_error("mpgnn_grouped_linear_wgrad_workspace_bytes: bytes is null");
    *bytes = 0;
    for (int eb : {2, 4}) {
        const int64_t chunk = wgrad_chunk(rows, groups, k, n, eb);
        if (rows > chunk)
            *bytes = std::max(*bytes, wgrad_items(rows, groups, chunk) * (k * n + n) * (int64_t)sizeof(float));
    }
    return MPGNN_OK;
}

extern "C" int32_t mpgnn_grouped_linear_wgrad(const void* x, int64_t x_pitch, const void* dy, int64_t dy_pitch,
                                              int64_t rows, int32_t dtype, int64_t groups, int64_t k, int64_t n,
                                              const void* group_ptr, int32_t ptr_bits, void* dweight, void* dbias,
                                              void* workspace, void* stream) {
    using namespace mpgnn;
    int32_t st = check_grouped(rows, groups, k, n, dtype, ptr_bits);
    if (st != MPGNN_OK) return st;
    if (!dweight || !group_ptr || (rows > 0 && (!x || !dy)) || (rows > 1 && (x_pitch < k || dy_pitch < n)))
        return arg_error("mpgnn_grouped_linear_wgrad: a null pointer, or a row pitch below the width");
    const int64_t chunk = wgrad_chunk(rows, groups, k, n, dtype_bytes(dtype));
    if (rows > chunk && !workspace) return arg_error("mpgnn_grouped_linear_wgrad: no workspace");
    if (chunk > INT32_MAX) return unsupported("mpgnn_grouped_linear_wgrad: over 2^31 rows");
    GroupedArgs a{};
    a.r = x; a.r_pitch = x_pitch; a.b = dy; a.b_pitch = dy_pitch; a.out = dweight; a.dbias = dbias;
    a.slabs = static_cast<float*>(workspace); a.ptr = group_ptr; a.ptr64 = ptr_bits == 64; a.rows = rows;
    a.groups = (int32_t)groups; a.out_rows = (int32_t)k; a.cols = (int32_t)n; a.chunk = (int32_t)chunk;
    a.r_end = end_of(x, rows, x_pitch, k, dtype);
    a.b_end = end_of(dy, rows, dy_pitch, n, dtype);
    hipStream_t strm = static_cast<hipStream_t>(stream);
    if (dtype == MPGNN_F32) return wgrad_product<float>(a, strm);
    return dtype == MPGNN_BF16 ? wgrad_product<__bf16>(a, strm) : wgrad_product<_Float16>(a, strm);
}
