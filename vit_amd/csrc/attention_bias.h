// Shared device code of the biased / capped / masked attention kernels (attention_bias*.hip).
//
//   s = q k^T * scale;  z = cap * tanh(s / cap) (or s) + bias(kpos - qpos);  p = softmax over the visible keys (z);  out = p v
//   dv = p^T dout;  dp = dout v^T;  dz = p o (dp - delta), delta = rowsum(dout o out);  ds = dz * (1 - tanh^2) * scale
//
// Everything after the matrix products is float32.  Scores are kept in units of log2: the scale, cap, table and slopes are
// multiplied by log2(e) once, so a probability is one v_exp_f32.
//
// Tiles: a workgroup of four waves owns 128 rows of one head (queries in the forward and dQ kernels, keys in the dK/dV
// kernel), 32 rows a wave, and walks tiles of 64 rows of the other side through LDS.  All products are 32 x 32 tiles with the
// wave's own row on the lane (mfma_f32_32x32x16_bf16, or 32x32x2_f32 for float32): the softmax statistics of a row then live
// in one lane pair (one shuffle), and the probabilities leave the accumulators as the second product's operand without
// crossing a lane.  32 own rows instead of 16 halve the LDS reads a score costs; at head size 64 the vector ALU (mask, bias,
// exponent) is what bounds these kernels, not the matrix cores.
#pragma once

#include "vitk_common.h"

#include <cfloat>

namespace abias {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int QB = 128;   // own rows of a workgroup
constexpr int TB = 64;    // rows of a streamed tile
constexpr int WIN = 1024; // largest range of distances of one tile pair whose biases are staged in LDS

enum { BIAS_NONE = 0, BIAS_SLOPE = 1, BIAS_TABLE = 2 };

struct Args {
	const void *q, *k, *v, *dout, *out;
	void* out_w;
	bf16_t* rest;    // [B, Sq, H * dh] out before its rounding minus out, or null
	float* lse_rest; // [B, H, Sq] the same of lse (float32 with slopes), or null
	float* lse;    // [B, H, Sq] log2 of the normaliser, +inf for a row that sees no key
	void *dq, *dk, *dv;
	float* delta;  // [B, H, Sq]
	int B, H, G, Hkv, Sq, Skv, dh;  // G = H / Hkv
	int64_t ldq, ldk, ldv, ldo, lddo, lddq, lddk, lddv;
	int64_t bq, bk, bv, bo, bdo, bdq, bdk, bdv;
	int gran;        // bytes one load may move from q, k, v, dout, out: 16, 8, or the element size
	int ovec;        // results may be stored 4 elements at a time (1), bfloat16 ones 8 (2)
	float c;         // scale * log2(e)
	float scale;
	float cap_l2;    // cap * log2(e)
	float inv_cap;   // scale / cap
	int causal, off; // off = Skv - Sq
	const int* prefix;
	const int *qseg, *kseg;
	const int *qpos, *kpos;
	int64_t bqp, bkp;         // batch strides of the positions (0: shared)
	const float* slopes;
	const float* expand;      // [H][n_lookup] table value of every distance index, in log2 units
	const int* lookup;
	int n_lookup, lookup_lo;
	int n_bucket;
	const int4 *qr, *kr;      // per 64 rows: {least (complemented if a row is padding), greatest segment, least, greatest position}; null without either
	int nq64, nk64;
	int split, per_split;     // the streamed side in `split` parts of `per_split` tiles
	float* part;              // partial results of a split launch
	float* row_part;          // and its row sums {sum dz, sum p} (dQ kernel, SUMS)
	int nblk;                 // blocks of 128 own rows
};

// ---- element types ----------------------------------------------------------------------------------------------------
template <typename T> struct Tr;
template <> struct Tr<bf16_t> {
	typedef bf16x8 frag;
	static constexpr int CH = 8;  // elements of a 16-byte chunk
	static __device__ __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Tr<float> {
	typedef f32x4 frag;
	static constexpr int CH = 4;
	static __device__ __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) {
#pragma unroll
		for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
		return c;
	}
};

// ---- LDS image of a tile: rows of DHP elements, 16-byte chunks permuted within a row so that 8 lanes reading one chunk of 8
// rows (row_frag) and the transposing reads (col_frag) touch all banks
template <typename T, int DHP> struct Img {
	static constexpr int RB = DHP * (int)sizeof(T);
	static constexpr int NC = RB / 16;       // chunks of a row
	static constexpr int STEPS = NC / 2;     // contraction steps of a product over the head size
	static constexpr int ND = DHP / 32;      // 32-column tiles of an output
	static constexpr int BYTES = TB * RB;
	static constexpr int NIT = TB * NC / 256;  // chunks a thread stages
	static __device__ __forceinline__ int off(int row, int chunk) { return row * RB + ((chunk ^ (RB == 64 ? ((row >> 1) & 3) : (row & 7))) << 4); }
};

template <typename T, int DHP> __device__ __forceinline__ typename Tr<T>::frag row_frag(const char* img, int row0, int s, int lane) {
	return *reinterpret_cast<const typename Tr<T>::frag*>(img + Img<T, DHP>::off(row0 + (lane & 31), 2 * s + (lane >> 5)));
}

// element j of the lane = img[row0 + 4 (lane >> 5) + (j & 3) + 8 (j >> 2)][d0 + (lane & 31)]
template <int DHP> __device__ __forceinline__ bf16x8 col_frag(const char* img, int row0, int d0, int lane) {
	typedef s16x4 __attribute__((address_space(3))) * lds_ptr_t;
	const int g = lane >> 4, i = lane & 15, q = i >> 2, p = i & 3;
	const int row = row0 + 4 * (g >> 1) + q;
	const int chunk = (d0 >> 3) + 2 * (g & 1) + (p >> 1), sub = (p & 1) << 3;
	s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr_t)(img + Img<bf16_t, DHP>::off(row, chunk) + sub));
	s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr_t)(img + Img<bf16_t, DHP>::off(row + 8, chunk) + sub));
	union {
		s16x4 h[2];
		bf16x8 v;
	} u;
	u.h[0] = lo;
	u.h[1] = hi;
	return u.v;
}

__device__ __forceinline__ bf16x8 pack_half(const f32x16& p, int s) {
	bf16x8 r;
#pragma unroll
	for (int j = 0; j < 8; ++j) r[j] = (bf16_t)p[8 * s + j];
	return r;
}

// acc[dt][d][own] += sum over the 32 tile rows r of img[row0 + r][32 dt + d] * w[r][own], w an accumulator tile (own row on the
// lane).  With bf16 operands w is rounded to bf16 (at most 2^-9 of each term, of either sign).
template <typename T, int DHP>
__device__ __forceinline__ void outer(f32x16 (&acc)[DHP / 32], const char* img, int row0, const f32x16& w, int lane) {
	if constexpr (sizeof(T) == 2) {
#pragma unroll
		for (int s = 0; s < 2; ++s) {
			const bf16x8 pf = pack_half(w, s);
#pragma unroll
			for (int dt = 0; dt < DHP / 32; ++dt) acc[dt] = Tr<bf16_t>::mma(col_frag<DHP>(img, row0 + 16 * s, 32 * dt, lane), pf, acc[dt]);
		}
	} else {
		const int hi = lane >> 5, i = lane & 31;
#pragma unroll
		for (int r = 0; r < 16; ++r) {
			const int row = row0 + (r & 3) + 8 * (r >> 2) + 4 * hi;
#pragma unroll
			for (int dt = 0; dt < DHP / 32; ++dt) {
				const float a = *reinterpret_cast<const float*>(img + Img<float, DHP>::off(row, 8 * dt + (i >> 2)) + ((i & 3) << 2));
				acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, w[r], acc[dt], 0, 0, 0);
			}
		}
	}
}

// ---- loads ------------------------------------------------------------------------------------------------------------
// Rows of one head through a buffer descriptor that ends with the last row there is: a row past the end, and a chunk that is told to be out
// (offset OUT), reads as zero without a branch, and a tile's loads differ from the previous tile's in the descriptor alone: the offsets
// stay in registers.  (Guarded 64-bit loads with their branches made the forward kernel 2600 instructions long.)
constexpr int OUT = (int)0x80000000u;
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

struct Rows {
	__amdgpu_buffer_rsrc_t r;
};
// rows row0 .. of a head whose first row starts at `base` (uniform); `total` rows in all, at most `span` of them are looked at
template <typename T> __device__ __forceinline__ Rows rows_of(const T* base, int64_t ld, int row0, int total, int span, int dh) {
	const uint64_t p = reinterpret_cast<uint64_t>(base + (int64_t)row0 * ld);
	const int n = min(total - row0, span);
	const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)p), hi = __builtin_amdgcn_readfirstlane((uint32_t)(p >> 32));
	const int bytes = __builtin_amdgcn_readfirstlane(n > 0 ? (int)(((int64_t)(n - 1) * ld + dh) * (int)sizeof(T)) : 0);
	Rows x;
	x.r = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>((uint64_t)hi << 32 | lo), 0, bytes, 0x00020000);
	return x;
}
// byte offset of chunk `ch` of row `row`, OUT past the head
template <typename T> __device__ __forceinline__ int chunk_off(int row, int64_t ld, int ch, int dh) {
	return ch * (16 / (int)sizeof(T)) < dh ? row * (int)ld * (int)sizeof(T) + ch * 16 : OUT;
}
// 16 bytes at `off`, the columns past the head zero; ch: which chunk of the row.  GR = 16: alignment allows whole chunks; else gran (uniform) says
// how many bytes one load may move, 8 or one element
template <typename T, int GR> __device__ __forceinline__ u32x4 load_chunk(const Rows& x, int off, int ch, int dh, int gran) {
	if constexpr (GR == 16) return __builtin_amdgcn_raw_buffer_load_b128(x.r, off, 0, 0);
	constexpr int CH = 16 / (int)sizeof(T);
	const int c0 = ch * CH;
	u32x4 v = {0, 0, 0, 0};
	if (gran == 8) {
		const u32x2 a = __builtin_amdgcn_raw_buffer_load_b64(x.r, off, 0, 0);
		const u32x2 b = __builtin_amdgcn_raw_buffer_load_b64(x.r, c0 + CH / 2 < dh ? off + 8 : OUT, 0, 0);
		v = u32x4{a[0], a[1], b[0], b[1]};
	} else if constexpr (sizeof(T) == 2) {
#pragma unroll
		for (int e = 0; e < 4; ++e) {
			const uint32_t a = __builtin_amdgcn_raw_buffer_load_b16(x.r, c0 + 2 * e < dh ? off + 4 * e : OUT, 0, 0);
			const uint32_t b = __builtin_amdgcn_raw_buffer_load_b16(x.r, c0 + 2 * e + 1 < dh ? off + 4 * e + 2 : OUT, 0, 0);
			v[e] = a | b << 16;
		}
	} else {
#pragma unroll
		for (int e = 0; e < 4; ++e) v[e] = __builtin_amdgcn_raw_buffer_load_b32(x.r, c0 + e < dh ? off + 4 * e : OUT, 0, 0);
	}
	return v;
}

// fragment of the wave's own row `row` (of the descriptor) straight from memory; zero where !ok
template <typename T, int GR> __device__ __forceinline__ typename Tr<T>::frag own_frag(const Rows& x, int row, int64_t ld, int s, int dh, int gran, bool ok, int lane) {
	const int ch = 2 * s + (lane >> 5);
	return __builtin_bit_cast(typename Tr<T>::frag, load_chunk<T, GR>(x, ok ? chunk_off<T>(row, ld, ch, dh) : OUT, ch, dh, gran));
}

// The staging of 64-row tiles: a thread's chunks, the same ones of every tile
template <typename T, int DHP, int GR> struct Stage {
	typedef Img<T, DHP> I;
	int off[I::NIT];
	u32x4 r[I::NIT];
	__device__ __forceinline__ void init(int64_t ld, int dh) {
#pragma unroll
		for (int i = 0; i < I::NIT; ++i) {
			const int idx = threadIdx.x + 256 * i;
			off[i] = chunk_off<T>(idx / I::NC, ld, idx % I::NC, dh);
		}
	}
	// which of the thread's chunks belong to rows of a negative segment (bits): they read as zero.  n: rows there are.  All loads before the first use
	static __device__ __forceinline__ uint32_t hidden(const int* seg, int n) {
		int sg[I::NIT];
#pragma unroll
		for (int i = 0; i < I::NIT; ++i) sg[i] = seg[min((int)(threadIdx.x + 256 * i) / I::NC, n - 1)];
		uint32_t m = 0;
#pragma unroll
		for (int i = 0; i < I::NIT; ++i) m |= (uint32_t)sg[i] >> 31 << i;
		return m;
	}
	__device__ __forceinline__ void fetch(const Rows& x, int dh, int gran, uint32_t hidden) {
#pragma unroll
		for (int i = 0; i < I::NIT; ++i) {
			const int idx = threadIdx.x + 256 * i;
			r[i] = load_chunk<T, GR>(x, hidden >> i & 1 ? OUT : off[i], idx % I::NC, dh, gran);
		}
	}
	// nonzero: an infinity or a NaN in the chunk: an exponent of ones, found by the carry that one more would give it
	static __device__ __forceinline__ uint32_t special(const u32x4& v) {
		uint32_t c = 0;
#pragma unroll
		for (int e = 0; e < 4; ++e) c |= sizeof(T) == 2 ? ((v[e] & 0x7f807f80u) + 0x00800080u) & 0x80008000u : ((v[e] & 0x7f800000u) + 0x00800000u) & 0x80000000u;
		return c;
	}
	__device__ __forceinline__ uint32_t special() const {
		uint32_t c = 0;
#pragma unroll
		for (int i = 0; i < I::NIT; ++i) c |= special(r[i]);
		return c;
	}
	// such chunks of the committed tile to zero, their rows marked (rare: read back from the tile in a loop, which holds no registers elsewhere)
	static __device__ __forceinline__ void clear_special(char* img, int* bad) {
#pragma unroll 1
		for (int i = 0; i < I::NIT; ++i) {
			const int idx = threadIdx.x + 256 * i;
			u32x4* at = reinterpret_cast<u32x4*>(img + I::off(idx / I::NC, idx % I::NC));
			if (special(*at) != 0) {
				*at = u32x4{0, 0, 0, 0};
				bad[idx / I::NC] = 1;
			}
		}
	}
	__device__ __forceinline__ void commit(char* img) const {
#pragma unroll
		for (int i = 0; i < I::NIT; ++i) {
			const int idx = threadIdx.x + 256 * i;
			*reinterpret_cast<u32x4*>(img + I::off(idx / I::NC, idx % I::NC)) = r[i];
		}
	}
};

// Infinities and NaN behind a mask.  A matrix product multiplies a hidden pair's weight 0 with whatever its row holds, and 0 * NaN would reach rows that do
// not see it.  In a partly visible tile that holds one (all threads look at what they have staged) such chunks are zeroed and their rows marked; an own
// row that sees a marked row becomes NaN as a whole (sees_marked), where the definition may have single columns; the others are as if it were not there.
// (Column by column -- the product without the special elements, and a second one that counts the infinities of either sign for the rows that see them -- the
// registers of that path spilled all over the loops: 16 x 32 x 784^2 training 1235 -> 1420 us, 2 x 16 x 2048^2 x 128 640 -> 1474, one query 160 -> 368.)
// Uniform; true: rows are marked.  tile: a number that says which of the tiles with one was the last (a flag in LDS that needs no clearing; 12 heads x 8192
// tokens of documents, training: 363 us, with __syncthreads_or 378).
template <typename S> __device__ __forceinline__ bool settle_tile(bool full, int tile, const S& x, char* ximg, const S& y, char* yimg, int* bad) {
	if (full) {
		__syncthreads();
		return false;
	}
	if (threadIdx.x < TB) bad[threadIdx.x] = 0;
	if ((x.special() | y.special()) != 0) bad[TB] = tile;  // (the last writer's number is the tile's own: a barrier lies between this and the reads before)
	__syncthreads();
	if (__builtin_amdgcn_readfirstlane(bad[TB]) != tile) return false;
	x.clear_special(ximg, bad);
	y.clear_special(yimg, bad);
	__syncthreads();
	return true;
}
// ---- scores -----------------------------------------------------------------------------------------------------------
// tanh(x) to about 1e-7: below 0.6 an odd polynomial (fitted to tanh(x) / x over x^2 at Chebyshev nodes), above it
// 1 - 2 / (1 + e^2x).  The two meet where the second has lost no digits; a capped score is cap * tanh, so an absolute error would
// be multiplied by the cap.
__device__ __forceinline__ float tanh_small(float x) {
	const float u = x * x;
	float r = fmaf(-5.856427829712629e-03f, u, 2.075747586786747e-02f);
	r = fmaf(r, u, -5.376992002129555e-02f);
	r = fmaf(r, u, 1.3331705331802368e-01f);
	r = fmaf(r, u, -3.333328366279602e-01f);
	r = fmaf(r, u, 1.0f);
	return x * r;
}
__device__ __forceinline__ float tanh_large(float x) {
	const float e = __builtin_amdgcn_exp2f(fabsf(x) * (2.0f * LOG2E));
	return copysignf(1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + e), x);
}
// t[r] = tanh(s[r] * inv_cap); the exponential form only where a value of the wave needs it
__device__ __forceinline__ void cap_tile(f32x16& t, const f32x16& s, float inv_cap) {
	float big = 0.f;
#pragma unroll
	for (int r = 0; r < 16; ++r) big = fmaxf(big, fabsf(s[r]));
	const bool any = __any(!(big * inv_cap <= 0.6f));
#pragma unroll
	for (int r = 0; r < 16; ++r) {
		const float x = s[r] * inv_cap;
		float y = tanh_small(x);
		if (any) y = fabsf(x) <= 0.6f ? y : tanh_large(x);
		t[r] = y;
	}
}

// ---- which tiles of the streamed side a workgroup visits ------------------------------------------------------------------
// Segments of 64 rows: least and greatest number, padding left out (it would stretch the range down to every other segment: the one block
// at the seam of the last sequence and a padded tail then walked all keys, and the launch waited for it).  A range with padding in it has
// its least number complemented; one of padding alone is {~INT_MAX, -1}, which meets nothing.
template <typename R> __device__ __forceinline__ int seg_least(const R& r) { return r.x < 0 ? ~r.x : r.x; }
struct Span {  // of the own rows of a workgroup
	int smin, smax, pmin, pmax;
	bool pad;
};
// A value at an address that is the same in every lane, through the scalar unit.  The compiler takes a vector load where it cannot show that; vector loads
// return in order, so the wait for one in front of a tile's scores also waited for the whole next tile (16 x 12 heads, one query, 16384 keys: 198 us, so 160).
// T is a power-of-two number of 32-bit words; the data is written by earlier launches only.
template <typename T> __device__ __forceinline__ T uniform_load(const T* p) {
	const uint64_t u = (uint64_t)p;
	const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u), hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
	return *(const __attribute__((address_space(4))) T*)((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ i32x4 range_at(const int4* r, int64_t i) { return uniform_load(reinterpret_cast<const i32x4*>(r) + i); }
__device__ __forceinline__ Span span_of(const int4* r, int i0, int n, bool pos, int lo, int hi) {
	Span s{0, 0, lo, hi, false};
	if (r != nullptr) {
		i32x4 x = range_at(r, i0);
		s.pad = x.x < 0;
		x.x = seg_least(x);
		if (i0 + 1 < n) {
			const i32x4 y = range_at(r, i0 + 1);
			s.pad |= y.x < 0;
			x.x = min(x.x, seg_least(y));
			x.y = max(x.y, y.y);
			x.z = min(x.z, y.z);
			x.w = max(x.w, y.w);
		}
		s.smin = x.x;
		s.smax = x.y;
		if (pos) {
			s.pmin = x.z;
			s.pmax = x.w;
		}
	}
	return s;
}

// The tiles t0 <= t < t1 that hold a visible pair, 64 looked at in one go (a lane each).  full(): every pair is visible.
template <bool KEYS>  // KEYS: own rows are queries and the tiles keys; else the other way round
struct Walk {
	uint64_t act, ful;
	int base, t1;
	bool any_full;  // among the tiles so far one was
	__device__ __forceinline__ void group(const Args& a, int own0, int own1, const Span& own, const int4* tr, int prefix, int lane) {
		const int t = base + lane;
		bool vis = t < t1, all = vis;
		const int r0 = t * TB, r1 = r0 + TB - 1;
		if constexpr (KEYS) all = all && r1 < a.Skv;
		if (a.causal) {
			const int q0 = KEYS ? own0 : r0, q1 = KEYS ? own1 : min(r1, a.Sq - 1), k0 = KEYS ? r0 : own0, k1 = KEYS ? r1 : own1;
			vis = vis && (k0 < prefix || k0 <= q1 + a.off);
			all = all && (k1 < prefix || k1 <= q0 + a.off);
		}
		if (a.kseg != nullptr && vis) {
			const int4 r = tr[t];
			vis = max(seg_least(r), own.smin) <= min(r.y, own.smax);
			all = all && !own.pad && r.x == r.y && own.smin == own.smax && r.x == own.smin;  // (a complemented r.x equals no r.y)
		}
		act = __ballot(vis);
		ful = __ballot(all) & act;
		any_full |= ful != 0;
	}
	__device__ __forceinline__ int next(const Args& a, int own0, int own1, const Span& own, const int4* tr, int prefix, int lane, bool& full) {
		while (act == 0) {
			base += 64;
			if (base >= t1) return -1;
			group(a, own0, own1, own, tr, prefix, lane);
		}
		const int i = __builtin_ctzll(act);
		full = (ful >> i) & 1;
		act &= act - 1;
		return base + i;
	}
	__device__ __forceinline__ void start(const Args& a, int t0, int t1_, int own0, int own1, const Span& own, const int4* tr, int prefix, int lane) {
		base = t0;
		t1 = t1_;
		act = ful = 0;
		any_full = false;
		if (base < t1) group(a, own0, own1, own, tr, prefix, lane);
	}
};

// ---- biases of a tile pair ------------------------------------------------------------------------------------------------
// The distances d = kpos - qpos of a pair of blocks lie in [lo, hi]; the bias is a function of d alone, so what a tile needs is
// the stretch of `expand` between them (128 queries x 64 keys in a row of tokens: 191 values instead of 8192 gathers).
enum { WIN_LDS = 0, WIN_ONE = 1, WIN_MEM = 2 };  // staged in LDS / one value for all pairs / too wide: read from memory
struct Window {
	int lo, mode;
};
__device__ __forceinline__ Window window_of(const Args& a, int lo, int hi) {
	Window w;
	w.lo = lo;
	const bool one = (hi <= a.lookup_lo || lo >= a.lookup_lo + a.n_lookup - 1) && a.slopes == nullptr;
	w.mode = one ? WIN_ONE : ((unsigned)hi - (unsigned)lo < (unsigned)WIN ? WIN_LDS : WIN_MEM);
	return w;
}
__device__ __forceinline__ int lookup_index(const Args& a, int d) {
	return min(max(d, a.lookup_lo), a.lookup_lo + a.n_lookup - 1) - a.lookup_lo;  // (saturating; clamped first, so nothing overflows)
}
__device__ __forceinline__ float bias_at(const Args& a, const float* ex, float slope, int d) {
	return fmaf(-slope, fabsf((float)d), ex[lookup_index(a, d)]);
}

// The lane number as something to work out anew: addresses that a tile derives from it are then not kept in registers over the whole loop (with
// a table there are a hundred of them, more than the registers of the third wave of a SIMD)
__device__ __forceinline__ int anew(int lane) {
	asm volatile("" : "+v"(lane));
	return lane;
}
__device__ __forceinline__ float pair_max(float v) { return fmaxf(v, __shfl_xor(v, 32, 64)); }
__device__ __forceinline__ float pair_sum(float v) { return v + __shfl_xor(v, 32, 64); }

// What a tile pair's scores need besides the products: biases, positions, segments and limits of the streamed rows (LDS, one
// entry a row), and of the wave's own row (registers).
struct Own {
	int pos, seg, lim;  // lim: keys at or past it are hidden from this query (own rows = queries)
	int idx;            // own rows = keys: the key's index
	float slope;        // slope of the head, log2 units
	const float* ex;    // the head's row of `expand`
};
struct TileSide {
	const float* win;
	const int *pos, *seg, *lim;
};

// A score is kept as z with p = 2^(z * score_scale - m): without cap and bias z stays the raw product, and the scale rides in the exponent's
// multiply-add; otherwise it is in log2 units already.
template <bool CAP, int BIAS> __device__ __forceinline__ float score_exp(const Args& a, float z, float m) {
	return __builtin_amdgcn_exp2f(!CAP && BIAS == BIAS_NONE ? fmaf(z, a.c, -m) : z - m);
}
// The backward's weight of a score: `rest` is what rounding took from lse, which with slopes may be thousands large (float32 alone: a step of lse is as much of
// every weight of the row; z - lse is exact where the weight counts)
template <typename T, bool CAP, int BIAS> __device__ __forceinline__ float weight_of(const Args& a, float z, float lse, float rest) {
	if constexpr (sizeof(T) == 4 && BIAS != BIAS_NONE) return __builtin_amdgcn_exp2f(z - lse - rest);
	return score_exp<CAP, BIAS>(a, z, lse);
}
// log2 of the normaliser of a row with maximum m and sum l
__device__ __forceinline__ void store_lse(const Args& a, int64_t row, float m, float l) {
	const float b = __builtin_amdgcn_logf(l), s = m + b;
	a.lse[row] = l == 0.f ? INFINITY : s;
	if (a.lse_rest != nullptr) a.lse_rest[row] = l == 0.f ? 0.f : b - (s - m);
}
// z: in the raw product of 32 streamed rows (row0 .. row0 + 31 of the tile) with the wave's own rows, out the score; tn: tanh(s / cap).
// rpos: position of the tile's row 0 where positions are indices.  The positions in LDS are multiplied by 4 with a table (a window's byte offsets).
template <bool KEYS, bool CAP, int BIAS>
__device__ __forceinline__ void modify(f32x16& z, f32x16& tn, const Args& a, const Window& w, const TileSide& ts, const Own& o, bool pos, int rpos, int row0, int lane) {
	const int h4 = 4 * (lane >> 5);
	float mul = a.c;
	if constexpr (CAP) {
		cap_tile(tn, z, a.inv_cap);
		z = tn;
		mul = a.cap_l2;
	}
	if constexpr (BIAS == BIAS_NONE) {
		if constexpr (CAP) {
#pragma unroll
			for (int r = 0; r < 16; ++r) z[r] *= mul;
		}
	}
	if constexpr (BIAS == BIAS_SLOPE) {
		if (!pos) {
			const float d0 = (float)(rpos + row0 + h4 - o.pos);
#pragma unroll
			for (int r = 0; r < 16; ++r) z[r] = fmaf(-o.slope, fabsf(d0 + (float)((r & 3) + 8 * (r >> 2))), z[r] * mul);
		} else {
#pragma unroll
			for (int g = 0; g < 4; ++g) {
				const int4 p = *reinterpret_cast<const int4*>(ts.pos + row0 + h4 + 8 * g);
				const int rp[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
				for (int e = 0; e < 4; ++e) z[4 * g + e] = fmaf(-o.slope, fabsf((float)(rp[e] - o.pos)), z[4 * g + e] * mul);
			}
		}
	}
	if constexpr (BIAS == BIAS_TABLE) {
		if (w.mode == WIN_ONE) {
			const float b = o.ex[lookup_index(a, w.lo)];
#pragma unroll
			for (int r = 0; r < 16; ++r) z[r] = fmaf(z[r], mul, b);
		} else if (w.mode == WIN_LDS) {
			if (!pos) {  // consecutive positions: one address a lane, the rows as offsets of the load
				if constexpr (KEYS) {
					const float* b = ts.win + (rpos + row0 + h4 - o.pos - w.lo);
#pragma unroll
					for (int r = 0; r < 16; ++r) z[r] = fmaf(z[r], mul, b[(r & 3) + 8 * (r >> 2)]);
				} else {
					const float* b = ts.win + (o.pos - rpos - row0 - h4 - 27 - w.lo);
#pragma unroll
					for (int r = 0; r < 16; ++r) z[r] = fmaf(z[r], mul, b[27 - (r & 3) - 8 * (r >> 2)]);
				}
			} else {
				const int base = 4 * (KEYS ? -o.pos - w.lo : o.pos - w.lo);
#pragma unroll
				for (int g = 0; g < 4; ++g) {
					const int4 p = *reinterpret_cast<const int4*>(ts.pos + row0 + h4 + 8 * g);
					const int rp[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
					for (int e = 0; e < 4; ++e)
						z[4 * g + e] = fmaf(z[4 * g + e], mul, *reinterpret_cast<const float*>(reinterpret_cast<const char*>(ts.win) + (KEYS ? base + rp[e] : base - rp[e])));
				}
			}
		} else {
#pragma unroll
			for (int r = 0; r < 16; ++r) {
				const int row = row0 + h4 + (r & 3) + 8 * (r >> 2);
				const int rp = pos ? ts.pos[row] >> 2 : rpos + row;
				z[r] = fmaf(z[r], mul, bias_at(a, o.ex, o.slope, KEYS ? rp - o.pos : o.pos - rp));
				if ((r & 3) == 3) __builtin_amdgcn_sched_barrier(0);  // (4 loads at a time: this path is rare, its registers are not)
			}
		}
	}
}

// hidden pairs of a tile that is not wholly visible: score -inf.  k0: index of the tile's row 0 (own rows = queries)
template <bool KEYS>
__device__ __forceinline__ void hide(f32x16& z, const Args& a, const TileSide& ts, const Own& o, int k0, int row0, int lane) {
	const int h4 = 4 * (lane >> 5), left = o.lim - k0 - row0 - h4;
	if constexpr (KEYS) {
#pragma unroll
		for (int r = 0; r < 16; ++r) z[r] = (r & 3) + 8 * (r >> 2) < left ? z[r] : -INFINITY;
	} else {
#pragma unroll
		for (int g = 0; g < 4; ++g) {
			const int4 l = *reinterpret_cast<const int4*>(ts.lim + row0 + h4 + 8 * g);
			z[4 * g] = o.idx < l.x ? z[4 * g] : -INFINITY;
			z[4 * g + 1] = o.idx < l.y ? z[4 * g + 1] : -INFINITY;
			z[4 * g + 2] = o.idx < l.z ? z[4 * g + 2] : -INFINITY;
			z[4 * g + 3] = o.idx < l.w ? z[4 * g + 3] : -INFINITY;
		}
	}
	if (a.kseg != nullptr) {
#pragma unroll
		for (int g = 0; g < 4; ++g) {
			const int4 s = *reinterpret_cast<const int4*>(ts.seg + row0 + h4 + 8 * g);
			z[4 * g] = s.x == o.seg ? z[4 * g] : -INFINITY;
			z[4 * g + 1] = s.y == o.seg ? z[4 * g + 1] : -INFINITY;
			z[4 * g + 2] = s.z == o.seg ? z[4 * g + 2] : -INFINITY;
			z[4 * g + 3] = s.w == o.seg ? z[4 * g + 3] : -INFINITY;
		}
	}
}

// NaN for an own row that sees a marked row of the tile (settle_tile), else 0: what it sees is worked out anew, apart from the scores, so that the
// tiles without a marked row pay no registers for it
template <bool KEYS> __device__ __forceinline__ float sees_marked(const Args& a, const TileSide& ts, const Own& o, int k0, const int* bad, int lane) {
	float poison = 0.f;
	lane = anew(lane);
#pragma unroll 1
	for (int row0 = 0; row0 < TB; row0 += 32) {
		f32x16 z;
#pragma unroll
		for (int r = 0; r < 16; ++r) z[r] = 0.f;
		hide<KEYS>(z, a, ts, o, k0, row0, lane);
#pragma unroll
		for (int r = 0; r < 16; ++r) poison = bad[row0 + 4 * (lane >> 5) + (r & 3) + 8 * (r >> 2)] != 0 && z[r] == 0.f ? __builtin_nanf("") : poison;
	}
	return poison;
}

// keys at or past it are hidden from query qi (segment `seg`)
__device__ __forceinline__ int limit_of(const Args& a, int qi, int seg, int prefix) {
	if (qi >= a.Sq || seg < 0) return 0;
	return a.causal ? min(a.Skv, max(prefix, qi + a.off + 1)) : a.Skv;
}

// What rounding to bfloat16 takes from a value of out; 0 where that is near what its sums leave: of a row that sees one key out is that key's value, and its
// rest none, though the weight in the normaliser, unlike that in the product, is 1 only to the rounding of the scores (2^-14: scores to 2^10)
__device__ __forceinline__ float rest_of(float v) {
	const float r = v - (float)(bf16_t)v;
	return fabsf(r) <= fabsf(v) * 0x1p-14f ? 0.f : r;
}

// 4 consecutive columns d0 .. d0 + 3 of a head's row
template <typename T> __device__ __forceinline__ void store4(T* row, int d0, int dh, int vec, const float (&v)[4]) {
	if (vec) {
		if (d0 < dh) store_vec<T, 4>(row + d0, v);
	} else {
#pragma unroll
		for (int i = 0; i < 4; ++i)
			if (d0 + i < dh) row[d0 + i] = from_f32<T>(v[i]);
	}
}

// A lane's row from accumulator tiles: value(dt, r) is column 32 dt + (r & 3) + 8 (r >> 2) + 4 (lane >> 5).  vec as Args::ovec: with 2 the two lanes of a row
// exchange halves, so that each has 8 consecutive columns and half as many stores go out (64 x 12 x 196^2 x 64, forward with rest: 53 us by 4, 50 by 8).
template <typename T, int ND, typename F> __device__ __forceinline__ void store_tiles(T* row, int dh, int vec, int lane, const F& value) {
	if constexpr (sizeof(T) == 2) {
		if (vec == 2) {
			auto pack = [&](int dt, int r) {
				const bf16_t lo = (bf16_t)value(dt, r), hi = (bf16_t)value(dt, r + 1);
				return (uint32_t)__builtin_bit_cast(uint16_t, lo) | (uint32_t)__builtin_bit_cast(uint16_t, hi) << 16;
			};
#pragma unroll
			for (int dt = 0; dt < ND; ++dt)
#pragma unroll
				for (int g = 0; g < 4; g += 2) {
					const auto a = __builtin_amdgcn_permlane32_swap(pack(dt, 4 * g), pack(dt, 4 * g + 4), false, false);
					const auto b = __builtin_amdgcn_permlane32_swap(pack(dt, 4 * g + 2), pack(dt, 4 * g + 6), false, false);
					const int d0 = 32 * dt + 8 * (g + (lane >> 5));
					if (d0 < dh) *reinterpret_cast<u32x4*>(row + d0) = u32x4{a[0], b[0], a[1], b[1]};
				}
			return;
		}
	}
#pragma unroll
	for (int dt = 0; dt < ND; ++dt)
#pragma unroll
		for (int g = 0; g < 4; ++g) {
			const float v[4] = {value(dt, 4 * g), value(dt, 4 * g + 1), value(dt, 4 * g + 2), value(dt, 4 * g + 3)};
			store4<T>(row, 32 * dt + 8 * g + 4 * (lane >> 5), dh, vec, v);
		}
}

// Workgroup -> (batch x head, block of own rows, part of the streamed side).  Consecutive workgroups go to the 8 dies in turn; the blocks of
// one head should share its rows in one die's L2.  With many heads die x takes heads x, x + 8, ... (sequences of different lengths are
// then spread over the dies: 16 padded sequences of 12 heads, one query each, 387 us against 527 with whole sequences to a die); with few, which 8 does
// not divide, the x-th eighth of all (head, block, part) in order, so that every die gets the same number (12 heads to 8 dies one by one: 2 to some, 1 to others).
// Behind a causal mask a head's blocks are taken from both ends in turn: any stretch of them is then about average work.
__host__ __device__ inline bool place_by_head(int nhead) { return nhead % 8 == 0 || nhead >= 64; }
__device__ __forceinline__ bool place(int nblk, int nhead, int split, int& bh, int& blk, int& part, bool both_ends) {
	const int per = nblk * split, x = blockIdx.x & 7, y = blockIdx.x >> 3;
	int rest;
	if (place_by_head(nhead)) {
		bh = y / per;
		rest = y - bh * per;
		bh = bh * 8 + x;
		if (bh >= nhead) return false;
	} else {
		const int all = nhead * per, each = (all + 7) >> 3, i = x * each + y;
		if (i >= all || y >= each) return false;
		bh = i / per;
		rest = i - bh * per;
	}
	blk = rest / split;
	part = rest - blk * split;
	if (both_ends) blk = blk & 1 ? blk >> 1 : nblk - 1 - (blk >> 1);
	return true;
}
inline int64_t placed_blocks(int64_t nblk, int64_t nhead, int64_t split) { return place_by_head((int)nhead) ? vitk_cdiv(nhead, 8) * 8 * nblk * split : vitk_cdiv(nblk * nhead * split, 8) * 8; }

// A forward over a divided axis leaves split * rows rows of dh sums and behind them {maximum, sum of the weights} of each; this is where those begin, in
// floats: even, so that a pair is one aligned load with odd head sizes too
__host__ __device__ inline int64_t part_pairs(int64_t split, int64_t rows, int64_t dh) { return (split * rows * dh + 1) & ~(int64_t)1; }
inline int64_t part_bytes(int64_t split, int64_t rows, int64_t dh) { return 4 * (part_pairs(split, rows, dh) + 2 * split * rows); }

// The table-gradient kernel's division of work: a workgroup = one head, one block of 128 queries, `chunk` tiles of keys, `images` batch entries
struct TablePlan {
	int chunk, nchunk, images, nimages;
};

}  // namespace abias

int vitk_abias_fwd_bf16(const abias::Args& a, hipStream_t st);
int vitk_abias_fwd_f32(const abias::Args& a, hipStream_t st);
int vitk_abias_dq_bf16(const abias::Args& a, bool sums, hipStream_t st);
int vitk_abias_dq_f32(const abias::Args& a, bool sums, hipStream_t st);
int vitk_abias_dkv_bf16(const abias::Args& a, hipStream_t st);
int vitk_abias_dkv_f32(const abias::Args& a, hipStream_t st);
// sums: [H][blocks of 128 queries][nchunk][nimages][n_bucket]
int vitk_abias_table_bf16(const abias::Args& a, const abias::TablePlan& p, float* sums, hipStream_t st);
int vitk_abias_table_f32(const abias::Args& a, const abias::TablePlan& p, float* sums, hipStream_t st);
