// Group normalisation with an activation over token-major (channels-last) activations x [B, S, C], C channels in G groups:
//
//   mean, var over the S * C / G values of an image's group;  xhat = (x - mean) * rstd;  z = xhat * gamma + beta;  y = act(z)
//   dz = dy * act'(z);  dgamma_c = sum dz xhat;  dbeta_c = sum dz;  with h = dz * gamma:
//   dx = rstd * (h - avg_g(h) - xhat * avg_g(h xhat))
//
// All of it is bandwidth: a forward must read x and write y, a backward read dy and x and write dx.  Two forms:
//  * fused: a workgroup of up to 512 threads holds all S rows of some whole groups of one image in registers (x and dy as the words they
//    came in; dz is worked out twice, its floats would be twice the registers), so every tensor crosses memory once.  Slices of one image may be narrower than a cache line: they go to
//    one die, whose L2 then serves the rest of the line to the neighbours.
//  * two passes for images whose narrowest slice does not fit: row slabs leave their sums, a second launch reads them in its prologue
//    and applies.  Images are taken in runs that the 256 MB last-level cache holds, so the second read of x (and dy) stays on the die.
// Statistics are float32: a thread's few rows about the first of them, and what threads and workgroups leave joined about means (sum_moments), so neither a
// mean far larger than the deviation nor outlying rows cost digits (128 x 28 x 28 x 768, training: 254 us; with one shift for all, which loses 1e-4 of the
// deviation to an outlier there, 251).  All sums are joined in a fixed order: the same bits from run to run.
#include "vitk_common.h"

namespace {

// fused kernels: threads of a workgroup, and vectors of a tensor that a thread holds at most.  128 x 28 x 28 x 768, forward and backward: 254 us with
// 512 threads both ways (5 rows a thread); 8 more with 256 threads and 10 rows in the forward, 69 more with 256 in the backward.  7 rows: the backward,
// which holds x and dy, has 128 registers for two workgroups to a CU, and spills with 8.  Instances for 2 and 5 rows keep images of fewer rows from
// loading rows that they do not have (forward and backward in us, own instance and that of 7 rows): 128 x 784 x 768 (5 rows) 86 + 177 and 92 + 190,
// 256 x 196 x 768 (5) 45 + 92 and 54 + 103, 128 x 400 x 384 in 8 groups (5) 24 + 42 and 27 + 47, 256 x 49 x 1536 (2) 46 + 63 and 57 + 111.
constexpr int FUSED_THREADS = 512, MOST_ROWS = 7;
constexpr int64_t CACHED_BYTES = 200ll << 20;     // of the tensors that are read twice, per run of images
constexpr int MAX_SLABS = 512;

// ---- activations: none, two with exponentials, and the clamps (relu, relu6) as one
enum { ACT_CLAMP = 0, ACT_SILU = 1, ACT_GELU = 2, ACT_NONE = 3 };
struct Shape {
	int S, C, G, cpg;
	float eps;
	float lo, hi;  // ACT_CLAMP: y = min(max(z, lo), hi)
};
// Normal distribution function of float32 activations: Phi(-|z|) = exp(-z^2 / 2) t Q(t), t = 1 / (1 + x / 2), x = |z| / sqrt 2, Q of degree 8 fitted to
// exp(x^2) erfc(x) / (2 t) over x in [0, 9.5] at Chebyshev nodes (relative error 4e-8, with float32 arithmetic 3e-7 and what the exponential's argument
// adds).  act_apply's 7.1.26 is good to 1.5e-7 absolute, enough for a result that is rounded to bfloat16, but to no digits of Phi(-5).  16 x 12544 x 256,
// training: 350 us, with 7.1.26 347, with erfcf 417.  `e` returns exp(-z^2 / 2).
__device__ __forceinline__ float normal_cdf(float z, float& e) {
	const float x = fabsf(z) * 0.70710678118654752f;
	const float t = __builtin_amdgcn_rcpf(fmaf(0.5f, x, 1.0f));
	e = __expf(-x * x);
	float q = fmaf(-2.944620830e-02f, t, 1.418548746e-01f);
	q = fmaf(q, t, -2.426996493e-01f);
	q = fmaf(q, t, 1.379976596e-01f);
	q = fmaf(q, t, -1.259449427e-02f);
	q = fmaf(q, t, 1.010371873e-01f);
	q = fmaf(q, t, 1.216299633e-01f);
	q = fmaf(q, t, 1.411768115e-01f);
	q = fmaf(q, t, 1.410438345e-01f);
	const float tail = q * t * e;
	return z >= 0.f ? 1.0f - tail : tail;
}
template <typename T, int ACT> __device__ __forceinline__ float act_of(float z, const Shape& s) {
	if constexpr (ACT == ACT_SILU) return act_apply(z, VITK_ACT_SILU);
	if constexpr (ACT == ACT_GELU && sizeof(T) == 4) {
		float e;
		return z * normal_cdf(z, e);
	}
	if constexpr (ACT == ACT_GELU) return act_apply(z, VITK_ACT_GELU);
	if constexpr (ACT == ACT_NONE) return z;
	return z < s.lo ? s.lo : (z > s.hi ? s.hi : z);  // (NaN stays NaN)
}
template <typename T, int ACT> __device__ __forceinline__ float slope_of(float z, const Shape& s) {
	if constexpr (ACT == ACT_SILU) return act_deriv(z, VITK_ACT_SILU);
	if constexpr (ACT == ACT_GELU && sizeof(T) == 4) {
		float e;
		const float cdf = normal_cdf(z, e);
		return fmaf(z * 0.39894228040143268f, e, cdf);
	}
	if constexpr (ACT == ACT_GELU) return act_deriv(z, VITK_ACT_GELU);
	if constexpr (ACT == ACT_NONE) return 1.f;
	return z <= s.lo || z >= s.hi ? 0.f : 1.f;
}

// dy * act'(z), the same bits wherever it is worked out
template <typename T, int ACT> __device__ __forceinline__ float dz_of(float dy, float xh, float w, float sh, const Shape& s) {
#pragma clang fp contract(off)
	return dy * slope_of<T, ACT>(fmaf(xh, w, sh), s);
}

// Rows are worked out one after another: the scheduler would interleave them, and keep the floats of all of them in registers
__device__ __forceinline__ void row_fence() { __builtin_amdgcn_sched_barrier(0); }

// V values of a tensor as the words they came in: kept as such, and taken apart where a row is worked out
template <typename T, int V> struct Raw {
	static constexpr int NW = sizeof(T) * V >= 4 ? (int)sizeof(T) * V / 4 : 1;
	uint32_t w[NW];
	__device__ __forceinline__ float get(int i) const {
		if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
		return __uint_as_float(i % 2 == 0 ? w[i / 2] << 16 : w[i / 2] & 0xffff0000u);
	}
	// Makes the compiler forget what it derived from the words: without it the converted floats are kept beside them, three times the registers
	__device__ __forceinline__ void reread() {
#pragma unroll
		for (int i = 0; i < NW; ++i) asm volatile("" : "+v"(w[i]));
	}
};
template <typename T, int V> __device__ __forceinline__ Raw<T, V> load_raw(const T* p) {
	Raw<T, V> r;
	if constexpr (sizeof(T) * V == 16) {
		const uint4 t = *reinterpret_cast<const uint4*>(p);
		r.w[0] = t.x;
		r.w[1] = t.y;
		r.w[2] = t.z;
		r.w[3] = t.w;
	} else if constexpr (sizeof(T) * V == 8) {
		const uint2 t = *reinterpret_cast<const uint2*>(p);
		r.w[0] = t.x;
		r.w[1] = t.y;
	} else if constexpr (sizeof(T) * V == 4) {
		r.w[0] = *reinterpret_cast<const uint32_t*>(p);
	} else {
		r.w[0] = *reinterpret_cast<const uint16_t*>(p);
	}
	return r;
}

// Division of numbers below 2^16 by a divisor d < 2^16: mulhi(n, ceil(2^32 / d)), exact since n * (the reciprocal's excess) < 2^32.  The
// integer division that the compiler writes is some 30 instructions, and the kernels below have a dozen of them per thread: at 10
// vectors a thread they were half of all vector instructions.
struct Div {
	uint32_t m, d;
	__host__ __device__ __forceinline__ explicit Div(int d_) : m(d_ == 1 ? 0u : 0xffffffffu / (uint32_t)d_ + 1u), d((uint32_t)d_) {}
	__device__ __forceinline__ int operator()(int n) const { return d == 1u ? n : (int)__umulhi((uint32_t)n, m); }
};

// red: [2][rows][width] partial sums -> red[0 .. width) and red[rows * width ..) the totals over the rows, in a fixed order
__device__ __forceinline__ void sum_rows(float* red, int rows, int width) {
	const Div dw(width);
	const int parts = max(1, min(rows, dw(blockDim.x)));
	__syncthreads();
	for (int i = threadIdx.x; i < parts * width; i += blockDim.x) {  // (one pass unless width > threads, where parts = 1)
		const int p = dw(i), c = i - p * width;
		float a = 0.f, b = 0.f;
		for (int r = p; r < rows; r += parts) {
			a += red[r * width + c];
			b += red[(rows + r) * width + c];
		}
		red[p * width + c] = a;  // (row p of column c is read by this thread alone)
		red[(rows + p) * width + c] = b;
	}
	__syncthreads();
	for (int c = threadIdx.x; c < width; c += blockDim.x) {
		float a = red[c], b = red[rows * width + c];
		for (int p = 1; p < parts; ++p) {
			a += red[p * width + c];
			b += red[(rows + p) * width + c];
		}
		red[c] = a;
		red[rows * width + c] = b;
	}
	__syncthreads();
}

// The same for {sum of n values, sum of their squared deviations from their own mean}: row r of red stands for values r, r + rows, ... of `total`.  What is
// joined is taken about the mean of the first that is: the square of its distance from the joint mean, which comes off again, is then smaller than the result
// where that first one holds an outlier (about a single value it would be n times the result, and its digits lost).
__device__ __forceinline__ void sum_moments(float* red, int rows, int width, int total) {
	const Div dw(width);
	const int parts = max(1, min(rows, dw(blockDim.x)));
	const int least = total / rows, more = total - least * rows;  // row r: least values, and one more if r < more
	const float n0 = (float)least, n1 = n0 + 1.f, inv0 = least > 0 ? 1.f / n0 : 0.f, inv1 = 1.f / n1;
	__syncthreads();
	for (int i = threadIdx.x; i < parts * width; i += blockDim.x) {  // (as in sum_rows)
		const int p = dw(i), c = i - p * width;
		const float mid = red[p * width + c] * (p < more ? inv1 : inv0);
		float a = 0.f, b = 0.f, n = 0.f;
		for (int r = p; r < rows; r += parts) {
			const float nr = r < more ? n1 : n0, d = fmaf(-nr, mid, red[r * width + c]);
			a += d;
			b += fmaf(d * d, r < more ? inv1 : inv0, red[(rows + r) * width + c]);
			n += nr;
		}
		red[p * width + c] = fmaf(n, mid, a);
		red[(rows + p) * width + c] = n > 0.f ? fmaf(-a * __builtin_amdgcn_rcpf(n), a, b) : 0.f;
	}
	__syncthreads();
	for (int c = threadIdx.x; c < width; c += blockDim.x) {
		const int q = rows / parts, over = rows - q * parts, mq = more / parts, mover = more - mq * parts;  // rows of a part, and those with one value more
		auto values = [&](int p) { return (float)((q + (p < over)) * least + mq + (p < mover)); };
		const float mid = red[c] / values(0);
		float a = 0.f, b = 0.f;
		for (int p = 0; p < parts; ++p) {
			const float n = values(p), d = fmaf(-n, mid, red[p * width + c]);
			a += d;
			b += fmaf(d * d, n > 0.f ? __builtin_amdgcn_rcpf(n) : 0.f, red[(rows + p) * width + c]);
		}
		const float n = (float)total;
		red[c] = fmaf(n, mid, a);
		red[rows * width + c] = fmaxf(fmaf(-a / n, a, b), 0.f);
	}
	__syncthreads();
}

// lanes that share a group's sums over n items: a power of two (its logarithm), 4 items or so a lane, no more than there are threads
__device__ __forceinline__ int lanes_for(int n) {
	int l = 0;
	while (l < 6 && (4 << l) < n && (2 << l) <= (int)blockDim.x) ++l;
	return l;
}
__device__ __forceinline__ float lane_sum(float v, int lanes) {
	for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
	return v;
}

// rs * (dz * w - p - xh * q) with dz * w rounded as the sum behind p rounds it: a group of one value then has the gradient 0 that it should
__device__ __forceinline__ float dx_of(float dz, float w, float xh, float p, float q, float rs) {
#pragma clang fp contract(off)
	const float h = dz * w - p;
	return rs * (h - xh * q);
}

// mean and sum of squared deviations of a group from its channels' sums s1 about x0[c] and squared deviations m2c (n values a channel): all lanes of the group
// get them.  Channels have equal counts: mean = average of their means, M2 = their M2 + n * squared deviations of their means.
__device__ __forceinline__ void group_moments(const float* s1, const float* m2c, const float* x0, int c0, int cpg, float n, int lanes, int l, float& mean, float& m2) {
	const float inv = 1.f / n;
	float m = 0.f;
	for (int c = c0 + l; c < c0 + cpg; c += lanes) m += fmaf(s1[c], inv, x0[c]);
	mean = lane_sum(m, lanes) / cpg;
	float q = 0.f;
	for (int c = c0 + l; c < c0 + cpg; c += lanes) {
		const float e = x0[c] + s1[c] * inv - mean;
		q += m2c[c] + n * e * e;
	}
	m2 = lane_sum(q, lanes);
}
__device__ __forceinline__ void group_dots(const float* s1, const float* s2, const float* gamma, int c0, int cpg, int lanes, int l, float& p, float& q) {
	float a = 0.f, b = 0.f;
	for (int c = c0 + l; c < c0 + cpg; c += lanes) {
		const float w = gamma[c];
		a = fmaf(w, s1[c], a);
		b = fmaf(w, s2[c], b);
	}
	p = lane_sum(a, lanes);
	q = lane_sum(b, lanes);
}

// A thread needs some numbers for each of its V channels (scale, shift, statistics of the group).  Read one by one from memory they are two dozen
// loads in a row, several microseconds of a workgroup's life, so the workgroup brings them to LDS together: op[j * width + c].
template <int V> __device__ __forceinline__ void operands(const float* op, int v, float (&o)[V]) {
#pragma unroll
	for (int i = 0; i < V; ++i) o[i] = op[v * V + i];
}

// ---- fused: one workgroup = all rows of channels [c0, c0 + cw) of one image ------------------------------------------------------
// thread = (row lane r, vector column v); rows r, r + k, r + 2k, ... in registers.  Workgroup id: slices of one image 8 apart (one die).
struct Slice {
	int b, c0, cw;
};
__device__ __forceinline__ Slice slice_of(int B, int C, int width, int n) {
	const int id = blockIdx.x, y = id >> 3;
	Slice s;
	s.b = y / n * 8 + (id & 7);
	s.c0 = y % n * width;
	s.cw = min(width, C - s.c0);
	return s;
}

template <typename T, int V, int ROWS, int ACT>
__global__ __launch_bounds__(FUSED_THREADS) void gn_fused_fwd_kernel(const T* __restrict__ x, const float* __restrict__ gamma, const float* __restrict__ beta, T* __restrict__ y,
	float* __restrict__ mean, float* __restrict__ rstd, Shape s, int B, int width, int slices) {
	extern __shared__ float red[];  // [2][k][cw] moments, [3][cw] operands, mean and rstd of the groups
	const Slice sl = slice_of(B, s.C, width, slices);
	if (sl.b >= B) return;
	const int c0 = sl.c0, cw = sl.cw, tpr = cw / V, b = sl.b;
	const Div dt(tpr), dc(s.cpg);
	const int k = min(dt(blockDim.x), s.S), r0 = dt(threadIdx.x), v = threadIdx.x - r0 * tpr;  // (a narrow last slice has more row lanes than rows)
	const bool on = r0 < k;
	const T* xb = x + (int64_t)b * s.S * s.C + c0;
	float* op = red + 2 * k * cw;
	Raw<T, V> xr[ROWS];
	const int64_t at = (int64_t)r0 * s.C + v * V, step = (int64_t)k * s.C;
	Raw<T, V> first;
	if (on) {
		first = load_raw<T, V>(xb + v * V);
#pragma unroll
		for (int j = 0; j < ROWS; ++j) xr[j] = load_raw<T, V>(xb + (r0 + j * k < s.S ? at + j * step : at));  // (past the end the thread's first row, the shift: adds nothing)
	}
	// (all threads: in a narrow last slice of an image of fewer rows than a vector has values those with rows are fewer than its channels)
	for (int c = threadIdx.x; c < cw; c += blockDim.x) {
		op[c] = gamma != nullptr ? gamma[c0 + c] : 1.f;
		op[cw + c] = beta != nullptr ? beta[c0 + c] : 0.f;
		op[2 * cw + c] = to_f32<T>(xb[c]);
	}
	if (on) {
		const Raw<T, V> own = xr[0];
		float s1[V], s2[V];
#pragma unroll
		for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.f;
#pragma unroll
		for (int j = 0; j < ROWS; ++j) {
			xr[j].reread();
#pragma unroll
			for (int i = 0; i < V; ++i) {
				const float d = xr[j].get(i) - own.get(i);
				s1[i] += d;
				s2[i] = fmaf(d, d, s2[i]);
			}
			row_fence();
		}
		const float n = (float)Div(k)(s.S - r0 + k - 1), inv = 1.f / n;  // values of the thread
#pragma unroll
		for (int i = 0; i < V; ++i) {
			red[r0 * cw + v * V + i] = fmaf(n, own.get(i) - first.get(i), s1[i]);
			red[(k + r0) * cw + v * V + i] = fmaxf(fmaf(-s1[i] * inv, s1[i], s2[i]), 0.f);
		}
	}
	sum_moments(red, k, cw, s.S);
	float* gm = op + 3 * cw;
	const int ng = dc(cw), lg = lanes_for(s.cpg), lanes = 1 << lg, per = blockDim.x >> lg;
	for (int g0 = 0; g0 < ng; g0 += per) {  // (every thread takes part in the shuffles; those past the last whole lane group write nothing)
		const int g = g0 + (int)(threadIdx.x >> lg);
		const bool mine = (threadIdx.x & (lanes - 1)) == 0 && (int)threadIdx.x < per * lanes && g < ng;
		float m, m2;
		group_moments(red, red + k * cw, op + 2 * cw, min(g, ng - 1) * s.cpg, s.cpg, (float)s.S, lanes, (threadIdx.x & (lanes - 1)), m, m2);
		if (mine) {
			const float rs = 1.f / sqrtf(m2 / ((float)s.S * s.cpg) + s.eps);
			gm[g] = m;
			gm[ng + g] = rs;
			if (mean != nullptr) {
				mean[(int64_t)b * s.G + dc(c0) + g] = m;
				rstd[(int64_t)b * s.G + dc(c0) + g] = rs;
			}
		}
	}
	__syncthreads();
	if (!on) return;
#pragma unroll
	for (int j = 0; j < ROWS; ++j) xr[j].reread();
	float mu[V], a[V], sh[V];
#pragma unroll
	for (int i = 0; i < V; ++i) {
		const int c = v * V + i, g = dc(c);
		mu[i] = gm[g];
		a[i] = gm[ng + g] * op[c];
		sh[i] = op[cw + c];
	}
	T* yb = y + (int64_t)b * s.S * s.C + c0 + at;
#pragma unroll
	for (int j = 0; j < ROWS; ++j) {
		if (r0 + j * k < s.S) {
			float o[V];
#pragma unroll
			for (int i = 0; i < V; ++i) o[i] = act_of<T, ACT>(fmaf(xr[j].get(i) - mu[i], a[i], sh[i]), s);
			store_vec<T, V>(yb + j * step, o);
		}
		row_fence();
	}
}

// part [B][C] {sum dz, sum dz xhat} for the parameter gradients
template <typename T, int V, int ROWS, int ACT>
__global__ __launch_bounds__(FUSED_THREADS, 4) void gn_fused_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x, const float* __restrict__ gamma, const float* __restrict__ beta,
	const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx, float2* __restrict__ part, Shape s, int B, int width, int slices) {
	extern __shared__ float red[];
	const Slice sl = slice_of(B, s.C, width, slices);
	if (sl.b >= B) return;
	const int c0 = sl.c0, cw = sl.cw, tpr = cw / V, b = sl.b;
	const Div dt(tpr), dc(s.cpg);
	const int k = min(dt(blockDim.x), s.S), r0 = dt(threadIdx.x), v = threadIdx.x - r0 * tpr;  // (a narrow last slice has more row lanes than rows)
	const bool on = r0 < k;
	const int64_t base = ((int64_t)b * s.S + r0) * s.C + c0 + v * V, step = (int64_t)k * s.C;
	float* op = red + 2 * k * cw;  // [4][cw]: mean, rstd, gamma, beta
	Raw<T, V> xr[ROWS], gr[ROWS];
	float mu[V], rs[V], w[V], sh[V];
	// (the operands' loads go out in front of the tensors', which then fly over the barrier)
	auto operand = [&](int c, float (&o)[4]) {
		const int64_t g = (int64_t)b * s.G + dc(c0 + c);
		o[0] = mean[g];
		o[1] = rstd[g];
		o[2] = gamma != nullptr ? gamma[c0 + c] : 1.f;
		o[3] = beta != nullptr ? beta[c0 + c] : 0.f;
	};
	float mine_op[4] = {0.f, 0.f, 0.f, 0.f};
	if ((int)threadIdx.x < cw) operand(threadIdx.x, mine_op);
	if (on) {
#pragma unroll
		for (int j = 0; j < ROWS; ++j) {
			const int64_t o = r0 + j * k < s.S ? j * step : 0;
			xr[j] = load_raw<T, V>(x + base + o);
			gr[j] = load_raw<T, V>(dy + base + o);
		}
	}
	for (int c = threadIdx.x; c < cw; c += blockDim.x) {
		if (c != (int)threadIdx.x) operand(c, mine_op);
#pragma unroll
		for (int i = 0; i < 4; ++i) op[i * cw + c] = mine_op[i];
	}
	__syncthreads();
	if (on) {
		operands<V>(op, v, mu);
		operands<V>(op + cw, v, rs);
		operands<V>(op + 2 * cw, v, w);
		operands<V>(op + 3 * cw, v, sh);
		float s1[V], s2[V];
#pragma unroll
		for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.f;
#pragma unroll
		for (int j = 0; j < ROWS; ++j) {
			const bool ok = r0 + j * k < s.S;
			xr[j].reread();
			gr[j].reread();
#pragma unroll
			for (int i = 0; i < V; ++i) {
				const float xh = (xr[j].get(i) - mu[i]) * rs[i];
				const float d = dz_of<T, ACT>(gr[j].get(i), xh, w[i], sh[i], s);
				s1[i] += ok ? d : 0.f;
				s2[i] = ok ? fmaf(d, xh, s2[i]) : s2[i];
			}
			row_fence();
		}
#pragma unroll
		for (int i = 0; i < V; ++i) {
			red[r0 * cw + v * V + i] = s1[i];
			red[(k + r0) * cw + v * V + i] = s2[i];
		}
	}
	sum_rows(red, k, cw);
	float* ga = op + 4 * cw;
	const int ng = dc(cw), lg = lanes_for(s.cpg), lanes = 1 << lg, per = blockDim.x >> lg;
	const float inv = 1.f / ((float)s.S * s.cpg);
	for (int c = threadIdx.x; c < cw; c += blockDim.x) part[(int64_t)b * s.C + c0 + c] = make_float2(red[c], red[k * cw + c]);
	for (int g0 = 0; g0 < ng; g0 += per) {  // (every thread takes part in the shuffles; those past the last whole lane group write nothing)
		const int g = g0 + (int)(threadIdx.x >> lg);
		const bool mine = (threadIdx.x & (lanes - 1)) == 0 && (int)threadIdx.x < per * lanes && g < ng;
		float p, q;
		group_dots(red, red + k * cw, op + 2 * cw, min(g, ng - 1) * s.cpg, s.cpg, lanes, (threadIdx.x & (lanes - 1)), p, q);
		if (mine) {
			ga[g] = p * inv;
			ga[ng + g] = q * inv;
		}
	}
	__syncthreads();
	if (!on) return;
#pragma unroll
	for (int j = 0; j < ROWS; ++j) {
		xr[j].reread();
		gr[j].reread();
	}
	float p[V], q[V];
	operands<V>(op, v, mu);
	operands<V>(op + cw, v, rs);
	operands<V>(op + 2 * cw, v, w);
	operands<V>(op + 3 * cw, v, sh);
#pragma unroll
	for (int i = 0; i < V; ++i) {
		const int g = dc(v * V + i);
		p[i] = ga[g];
		q[i] = ga[ng + g];
	}
#pragma unroll
	for (int j = 0; j < ROWS; ++j) {
		if (r0 + j * k < s.S) {
			float o[V];
#pragma unroll
			for (int i = 0; i < V; ++i) {
				const float xh = (xr[j].get(i) - mu[i]) * rs[i];
				o[i] = dx_of(dz_of<T, ACT>(gr[j].get(i), xh, w[i], sh[i], s), w[i], xh, p[i], q[i], rs[i]);
			}
			store_vec<T, V>(dx + base + j * step, o);
		}
		row_fence();
	}
}

// ---- two passes: one workgroup = a slab of rows of one image, all channels ---------------------------------------------------------
// thread = (row lane, vector column) as above; more than `tpr` vectors in a row are taken in column blocks
template <typename T, int V>
__global__ __launch_bounds__(256) void gn_stats_kernel(const T* __restrict__ x, float2* __restrict__ part, Shape s, int rows_per, int tpr) {
	extern __shared__ float red[];  // [2][k][tpr * V], then [3][C]: the channels' sums and shifts
	const Div dt(tpr);
	const int k = dt(blockDim.x), b = blockIdx.y, r0 = dt(threadIdx.x), v = threadIdx.x - r0 * tpr;
	const int first = blockIdx.x * rows_per, last = min(s.S, first + rows_per);
	const T* xb = x + (int64_t)b * s.S * s.C;
	float* tot = red + 2 * k * tpr * V;
	for (int cb = 0; cb < s.C; cb += tpr * V) {
		const int c = cb + v * V, cw = min(tpr * V, s.C - cb);
		if (r0 < k && c < s.C) {
			const Raw<T, V> top = load_raw<T, V>(xb + (int64_t)first * s.C + c);
			if (r0 == 0) {
#pragma unroll
				for (int i = 0; i < V; ++i) tot[2 * s.C + c + i] = top.get(i);
			}
			float mean[V], m2[V], n = 0.f;  // of the thread's rows so far
#pragma unroll
			for (int i = 0; i < V; ++i) mean[i] = m2[i] = 0.f;
			const int64_t step = (int64_t)k * s.C;
			int64_t at = (int64_t)(first + r0) * s.C + c;
			for (int r = first + r0; r < last; r += 8 * k, at += 8 * step) {  // 8 rows in flight
				Raw<T, V> f[8];
				float s1[V], s2[V];
#pragma unroll
				for (int u = 0; u < 8; ++u) f[u] = load_raw<T, V>(xb + at + (r + u * k < last ? u * step : 0));
#pragma unroll
				for (int i = 0; i < V; ++i) {
					s1[i] = s2[i] = 0.f;
					if (n == 0.f) mean[i] = f[0].get(i);
				}
				// sums about the mean so far (of the first rows: about the first), then about the new one
#pragma unroll
				for (int u = 0; u < 8; ++u) {
					const bool ok = r + u * k < last;
					f[u].reread();
#pragma unroll
					for (int i = 0; i < V; ++i) {
						const float d = ok ? f[u].get(i) - mean[i] : 0.f;
						s1[i] += d;
						s2[i] = fmaf(d, d, s2[i]);
					}
					row_fence();
				}
				n += (float)min(8, (last - r + k - 1) / k);
				const float inv = 1.f / n;
#pragma unroll
				for (int i = 0; i < V; ++i) {
					const float d = s1[i] * inv;
					m2[i] += fmaxf(fmaf(-s1[i], d, s2[i]), 0.f);
					mean[i] += d;
				}
			}
#pragma unroll
			for (int i = 0; i < V; ++i) {
				red[r0 * cw + v * V + i] = n * (mean[i] - top.get(i));
				red[(k + r0) * cw + v * V + i] = m2[i];
			}
		}
		sum_moments(red, k, cw, last - first);
		for (int i = threadIdx.x; i < cw; i += blockDim.x) {
			tot[cb + i] = red[i];
			tot[s.C + cb + i] = red[k * cw + i];
		}
		__syncthreads();
	}
	const int lg = lanes_for(s.cpg), lanes = 1 << lg, per = blockDim.x >> lg;
	for (int g0 = 0; g0 < s.G; g0 += per) {  // (every thread takes part in the shuffles; those past the last whole lane group write nothing)
		const int g = g0 + (int)(threadIdx.x >> lg);
		const bool mine = (threadIdx.x & (lanes - 1)) == 0 && (int)threadIdx.x < per * lanes && g < s.G;
		float m, m2;
		group_moments(tot, tot + s.C, tot + 2 * s.C, min(g, s.G - 1) * s.cpg, s.cpg, (float)(last - first), lanes, (threadIdx.x & (lanes - 1)), m, m2);
		if (mine) part[((int64_t)b * s.G + g) * gridDim.x + blockIdx.x] = make_float2(m, m2);
	}
}

// one wave = one group of one image: the slabs' {mean, M2} -> mean, rstd; or {sum h, sum h xhat} -> their averages (out)
template <bool BWD>
__global__ __launch_bounds__(256) void gn_final_kernel(const float2* __restrict__ part, float* __restrict__ mean, float* __restrict__ rstd, float2* __restrict__ out, Shape s, int n, int slabs,
	int slab_rows) {
	const int i = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
	if (i >= n) return;
	const float2* p = part + (int64_t)i * slabs;
	float a = 0.f, b = 0.f;
	if constexpr (BWD) {
		for (int j = lane; j < slabs; j += 64) {
			a += p[j].x;
			b += p[j].y;
		}
		a = wave_sum(a);
		b = wave_sum(b);
		const float inv = 1.f / ((float)s.S * s.cpg);
		if (lane == 0) out[i] = make_float2(a * inv, b * inv);
	} else {
		for (int j = lane; j < slabs; j += 64) a = fmaf((float)(min(s.S, (j + 1) * slab_rows) - j * slab_rows), p[j].x, a);
		a = wave_sum(a) / s.S;
		for (int j = lane; j < slabs; j += 64) b += p[j].y + (float)(min(s.S, (j + 1) * slab_rows) - j * slab_rows) * s.cpg * (p[j].x - a) * (p[j].x - a);
		b = wave_sum(b);
		if (lane == 0) {
			mean[i] = a;
			rstd[i] = 1.f / sqrtf(b / ((float)s.S * s.cpg) + s.eps);
		}
	}
}

template <typename T, int V, int ACT>
__global__ __launch_bounds__(256) void gn_apply_kernel(const T* __restrict__ x, const float* __restrict__ gamma, const float* __restrict__ beta, const float* __restrict__ mean,
	const float* __restrict__ rstd, T* __restrict__ y, Shape s, int rows_per, int tpr) {
	const Div dt(tpr), dc(s.cpg);
	const int k = dt(blockDim.x), b = blockIdx.y, r0 = dt(threadIdx.x), v = threadIdx.x - r0 * tpr;
	extern __shared__ float op[];  // [3][tpr * V]: mean, rstd * gamma, beta
	const int first = blockIdx.x * rows_per, last = min(s.S, first + rows_per), w = tpr * V;
	for (int cb = 0; cb < s.C; cb += w) {
		if (cb != 0) __syncthreads();
		for (int i = threadIdx.x; i < min(w, s.C - cb); i += blockDim.x) {
			const int64_t g = (int64_t)b * s.G + dc(cb + i);
			op[i] = mean[g];
			op[w + i] = rstd[g] * (gamma != nullptr ? gamma[cb + i] : 1.f);
			op[2 * w + i] = beta != nullptr ? beta[cb + i] : 0.f;
		}
		__syncthreads();
		const int c = cb + v * V;
		if (r0 >= k || c >= s.C) continue;
		float mu[V], a[V], sh[V];
		operands<V>(op, v, mu);
		operands<V>(op + w, v, a);
		operands<V>(op + 2 * w, v, sh);
		const int64_t step = (int64_t)k * s.C;
		int64_t at = ((int64_t)b * s.S + first + r0) * s.C + c;
		for (int r = first + r0; r < last; r += 4 * k, at += 4 * step) {
			Raw<T, V> f[4];
#pragma unroll
			for (int u = 0; u < 4; ++u) f[u] = load_raw<T, V>(x + at + (r + u * k < last ? u * step : 0));
#pragma unroll
			for (int u = 0; u < 4; ++u) {
				float o[V];
#pragma unroll
				for (int i = 0; i < V; ++i) o[i] = act_of<T, ACT>(fmaf(f[u].get(i) - mu[i], a[i], sh[i]), s);
				if (r + u * k < last) store_vec<T, V>(y + at + u * step, o);
			}
		}
	}
}

// chan [B][slabs][C] {sum dz, sum dz xhat};  part [B][G][slabs] the same weighted by gamma and summed over the group
template <typename T, int V, int ACT>
__global__ __launch_bounds__(256) void gn_bwd_stats_kernel(const T* __restrict__ dy, const T* __restrict__ x, const float* __restrict__ gamma, const float* __restrict__ beta,
	const float* __restrict__ mean, const float* __restrict__ rstd, float2* __restrict__ chan, float2* __restrict__ part, Shape s, int rows_per, int tpr) {
	extern __shared__ float red[];  // [2][k][tpr * V], [4][tpr * V]: mean, rstd, gamma, beta; then [3][C]: the channels' sums, gamma
	const Div dt(tpr), dc(s.cpg);
	const int k = dt(blockDim.x), b = blockIdx.y, r0 = dt(threadIdx.x), v = threadIdx.x - r0 * tpr;
	const int first = blockIdx.x * rows_per, last = min(s.S, first + rows_per);
	const int wd = tpr * V;
	float *op = red + 2 * k * wd, *tot = op + 4 * wd;
	const int64_t slab = (int64_t)b * gridDim.x + blockIdx.x;
	for (int cb = 0; cb < s.C; cb += tpr * V) {
		const int c = cb + v * V, cw = min(tpr * V, s.C - cb);
		if (cb != 0) __syncthreads();
		for (int j = threadIdx.x; j < cw; j += blockDim.x) {
			const int64_t g = (int64_t)b * s.G + dc(cb + j);
			op[j] = mean[g];
			op[wd + j] = rstd[g];
			op[2 * wd + j] = tot[2 * s.C + cb + j] = gamma != nullptr ? gamma[cb + j] : 1.f;
			op[3 * wd + j] = beta != nullptr ? beta[cb + j] : 0.f;
		}
		__syncthreads();
		if (r0 < k && c < s.C) {
			float mu[V], rs[V], w[V], sh[V], s1[V], s2[V];
			operands<V>(op, v, mu);
			operands<V>(op + wd, v, rs);
			operands<V>(op + 2 * wd, v, w);
			operands<V>(op + 3 * wd, v, sh);
#pragma unroll
			for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.f;
			const int64_t step = (int64_t)k * s.C;
			int64_t at = ((int64_t)b * s.S + first + r0) * s.C + c;
			for (int r = first + r0; r < last; r += 4 * k, at += 4 * step) {
				Raw<T, V> f[4], d[4];
#pragma unroll
				for (int u = 0; u < 4; ++u) {
					const int64_t o = r + u * k < last ? u * step : 0;
					f[u] = load_raw<T, V>(x + at + o);
					d[u] = load_raw<T, V>(dy + at + o);
				}
#pragma unroll
				for (int u = 0; u < 4; ++u) {
					const bool ok = r + u * k < last;
					f[u].reread();
					d[u].reread();
#pragma unroll
					for (int i = 0; i < V; ++i) {
						const float xh = (f[u].get(i) - mu[i]) * rs[i];
						const float dz = dz_of<T, ACT>(d[u].get(i), xh, w[i], sh[i], s);
						s1[i] += ok ? dz : 0.f;
						s2[i] = ok ? fmaf(dz, xh, s2[i]) : s2[i];
					}
					row_fence();
				}
			}
#pragma unroll
			for (int i = 0; i < V; ++i) {
				red[r0 * cw + v * V + i] = s1[i];
				red[(k + r0) * cw + v * V + i] = s2[i];
			}
		}
		sum_rows(red, k, cw);
		for (int i = threadIdx.x; i < cw; i += blockDim.x) {
			tot[cb + i] = red[i];
			tot[s.C + cb + i] = red[k * cw + i];
			chan[slab * s.C + cb + i] = make_float2(red[i], red[k * cw + i]);
		}
		__syncthreads();
	}
	const int lg = lanes_for(s.cpg), lanes = 1 << lg, per = blockDim.x >> lg;
	for (int g0 = 0; g0 < s.G; g0 += per) {  // (every thread takes part in the shuffles; those past the last whole lane group write nothing)
		const int g = g0 + (int)(threadIdx.x >> lg);
		const bool mine = (threadIdx.x & (lanes - 1)) == 0 && (int)threadIdx.x < per * lanes && g < s.G;
		float p, q;
		group_dots(tot, tot + s.C, tot + 2 * s.C, min(g, s.G - 1) * s.cpg, s.cpg, lanes, (threadIdx.x & (lanes - 1)), p, q);
		if (mine) part[((int64_t)b * s.G + g) * gridDim.x + blockIdx.x] = make_float2(p, q);
	}
}

template <typename T, int V, int ACT>
__global__ __launch_bounds__(256) void gn_bwd_apply_kernel(const T* __restrict__ dy, const T* __restrict__ x, const float* __restrict__ gamma, const float* __restrict__ beta,
	const float* __restrict__ mean, const float* __restrict__ rstd, const float2* __restrict__ avg, T* __restrict__ dx, Shape s, int rows_per, int tpr) {
	const Div dt(tpr), dc(s.cpg);
	const int k = dt(blockDim.x), b = blockIdx.y, r0 = dt(threadIdx.x), v = threadIdx.x - r0 * tpr;
	extern __shared__ float op[];  // [6][tpr * V]: mean, rstd, gamma, beta, and the two averages
	const int first = blockIdx.x * rows_per, last = min(s.S, first + rows_per), wd = tpr * V;
	for (int cb = 0; cb < s.C; cb += wd) {
		if (cb != 0) __syncthreads();
		for (int i = threadIdx.x; i < min(wd, s.C - cb); i += blockDim.x) {
			const int64_t g = (int64_t)b * s.G + dc(cb + i);
			const float2 t = avg[g];
			op[i] = mean[g];
			op[wd + i] = rstd[g];
			op[2 * wd + i] = gamma != nullptr ? gamma[cb + i] : 1.f;
			op[3 * wd + i] = beta != nullptr ? beta[cb + i] : 0.f;
			op[4 * wd + i] = t.x;
			op[5 * wd + i] = t.y;
		}
		__syncthreads();
		const int c = cb + v * V;
		if (r0 >= k || c >= s.C) continue;
		float mu[V], rs[V], w[V], sh[V], p[V], q[V];
		operands<V>(op, v, mu);
		operands<V>(op + wd, v, rs);
		operands<V>(op + 2 * wd, v, w);
		operands<V>(op + 3 * wd, v, sh);
		operands<V>(op + 4 * wd, v, p);
		operands<V>(op + 5 * wd, v, q);
		const int64_t step = (int64_t)k * s.C;
		int64_t at = ((int64_t)b * s.S + first + r0) * s.C + c;
		for (int r = first + r0; r < last; r += 4 * k, at += 4 * step) {
			Raw<T, V> f[4], d[4];
#pragma unroll
			for (int u = 0; u < 4; ++u) {
				const int64_t o = r + u * k < last ? u * step : 0;
				f[u] = load_raw<T, V>(x + at + o);
				d[u] = load_raw<T, V>(dy + at + o);
			}
#pragma unroll
			for (int u = 0; u < 4; ++u) {
				float o[V];
#pragma unroll
				for (int i = 0; i < V; ++i) {
					const float xh = (f[u].get(i) - mu[i]) * rs[i];
					o[i] = dx_of(dz_of<T, ACT>(d[u].get(i), xh, w[i], sh[i], s), w[i], xh, p[i], q[i], rs[i]);
				}
				if (r + u * k < last) store_vec<T, V>(dx + at + u * step, o);
				row_fence();
			}
		}
	}
}

// rows [n][C] summed in runs of `run` rows -> out [ceil(n / run)][C]; the last step (one run) writes dgamma and dbeta
__global__ __launch_bounds__(256) void gn_param_kernel(const float2* __restrict__ in, float2* __restrict__ out, float* __restrict__ dgamma, float* __restrict__ dbeta, int64_t n, int run,
	int C, int accumulate) {
	__shared__ float2 red[8][32];
	const int c = blockIdx.x * 32 + (threadIdx.x & 31), g = threadIdx.x >> 5;
	const int64_t first = (int64_t)blockIdx.y * run, last = min(n, first + run);
	float a = 0.f, b = 0.f;
	if (c < C) {
		for (int64_t r = first + g; r < last; r += 8) {
			const float2 t = in[r * C + c];
			a += t.x;
			b += t.y;
		}
	}
	red[g][threadIdx.x & 31] = make_float2(a, b);
	__syncthreads();
	if (g == 0 && c < C) {
		for (int i = 1; i < 8; ++i) {
			a += red[i][threadIdx.x].x;
			b += red[i][threadIdx.x].y;
		}
		if (out != nullptr) {
			out[(int64_t)blockIdx.y * C + c] = make_float2(a, b);
		} else {
			if (dbeta != nullptr) dbeta[c] = accumulate ? dbeta[c] + a : a;
			if (dgamma != nullptr) dgamma[c] = accumulate ? dgamma[c] + b : b;
		}
	}
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------
struct Plan {
	int V;                       // channels a thread loads at once
	int width, slices, threads;  // fused: channels of a workgroup (0: two passes), slices of an image, threads
	int rows;                    // fused: vectors a thread holds (2, 5 or the most)
	int tpr, k;                  // two passes: threads a row, row lanes
	int slabs, slab_rows;        // two passes
	int64_t run;                 // two passes: images of a run
	int64_t n_part;              // rows of [C] channel sums the backward leaves
};

int64_t gcd64(int64_t a, int64_t b) { return b == 0 ? a : gcd64(b, a % b); }

Plan plan_of(int64_t B, int64_t S, int64_t C, int64_t G, int es, bool aligned, bool bwd) {
	Plan p{};
	const int64_t cpg = C / G;
	p.V = aligned && C % (16 / es) == 0 ? 16 / es : (aligned && C % 2 == 0 ? 2 : 1);
	const int64_t unit = cpg / gcd64(cpg, p.V) * p.V;  // whole groups and whole vectors
	const int threads = FUSED_THREADS, most = MOST_ROWS;
	// the widest slice of up to about 128 bytes whose rows fit the registers of the workgroup
	for (int64_t w = std::min(C, vitk_cdiv(128 / es, unit) * unit); w >= unit; w -= unit) {
		const int64_t tpr = w / p.V;
		if (tpr > threads) continue;
		const int64_t k = std::min<int64_t>(S, threads / tpr), rows = vitk_cdiv(S, k);
		if (rows > most) continue;
		p.width = (int)w;
		p.slices = (int)vitk_cdiv(C, w);
		p.threads = (int)(tpr * k);
		p.rows = rows <= 2 ? 2 : (rows <= 5 ? 5 : most);
		p.n_part = B;
		return p;
	}
	const int64_t cv = C / p.V;
	p.tpr = (int)std::min<int64_t>(cv, 256);
	p.k = 256 / p.tpr;
	const int64_t bytes = S * C * es * (bwd ? 2 : 1);
	p.run = std::max<int64_t>(1, std::min<int64_t>(B, CACHED_BYTES / std::max<int64_t>(bytes, 1)));
	// up to 8192 workgroups a launch, each at least 8 rows a lane
	p.slabs = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(MAX_SLABS, vitk_cdiv(8192, p.run)), S / (8 * p.k)));
	p.slab_rows = (int)vitk_cdiv(S, p.slabs);
	p.slabs = (int)vitk_cdiv(S, p.slab_rows);
	p.n_part = B * p.slabs;
	return p;
}

constexpr int PARAM_RUN = 128;

int check(int64_t B, int64_t S, int64_t C, int64_t G, int act, int dtype) {
	VITK_REQUIRE(dtype == VITK_F32 || dtype == VITK_BF16, VITK_ERR_DTYPE);
	VITK_REQUIRE(B > 0 && S > 0 && C > 0 && G > 0 && C % G == 0, VITK_ERR_SHAPE);
	VITK_REQUIRE(B <= 65535 && S <= (1 << 30) && C <= 4096, VITK_ERR_SHAPE);
	VITK_REQUIRE(act >= VITK_ACT_NONE && act <= VITK_ACT_RELU6, VITK_ERR_UNSUPPORTED);
	return VITK_OK;
}

Shape shape_of(int64_t S, int64_t C, int64_t G, float eps, int act) {
	Shape s{(int)S, (int)C, (int)G, (int)(C / G), eps, -INFINITY, INFINITY};
	if (act == VITK_ACT_RELU || act == VITK_ACT_RELU6) s.lo = 0.f;
	if (act == VITK_ACT_RELU6) s.hi = 6.f;
	return s;
}

inline size_t fused_lds(const Plan& p, int64_t cpg) { return sizeof(float) * ((size_t)2 * p.threads * p.V + 4 * p.width + 2 * (p.width / cpg)); }
inline size_t slab_lds(const Plan& p, int64_t C) { return sizeof(float) * ((size_t)(2 * p.k + 4) * p.tpr * p.V + 3 * C); }
inline size_t apply_lds(const Plan& p) { return sizeof(float) * 6 * p.tpr * p.V; }

template <typename T, int V, int ACT>
int forward(const T* x, const float* gamma, const float* beta, T* y, float* mean, float* rstd, int64_t B, const Shape& s, const Plan& p, float2* ws, hipStream_t st) {
	if (p.width != 0) {
		const dim3 grid((unsigned)(vitk_cdiv(B, 8) * 8 * p.slices)), block(p.threads);
		const size_t lds = fused_lds(p, s.cpg);
		if (p.rows == 2) hipLaunchKernelGGL((gn_fused_fwd_kernel<T, V, 2, ACT>), grid, block, lds, st, x, gamma, beta, y, mean, rstd, s, (int)B, p.width, p.slices);
		else if (p.rows == 5) hipLaunchKernelGGL((gn_fused_fwd_kernel<T, V, 5, ACT>), grid, block, lds, st, x, gamma, beta, y, mean, rstd, s, (int)B, p.width, p.slices);
		else hipLaunchKernelGGL((gn_fused_fwd_kernel<T, V, MOST_ROWS, ACT>), grid, block, lds, st, x, gamma, beta, y, mean, rstd, s, (int)B, p.width, p.slices);
		VITK_CHECK_LAUNCH();
		return VITK_OK;
	}
	for (int64_t b = 0; b < B; b += p.run) {
		const int64_t n = std::min(p.run, B - b), at = b * s.S * s.C;
		const dim3 grid((unsigned)p.slabs, (unsigned)n), block(p.tpr * p.k);
		hipLaunchKernelGGL((gn_stats_kernel<T, V>), grid, block, slab_lds(p, s.C), st, x + at, ws, s, p.slab_rows, p.tpr);
		VITK_CHECK_LAUNCH();
		float* mu = mean != nullptr ? mean + b * s.G : reinterpret_cast<float*>(ws + p.run * p.slabs * s.G);
		float* rs = mean != nullptr ? rstd + b * s.G : mu + p.run * s.G;
		hipLaunchKernelGGL((gn_final_kernel<false>), dim3((unsigned)vitk_cdiv(n * s.G, 4)), dim3(256), 0, st, ws, mu, rs, nullptr, s, (int)(n * s.G), p.slabs, p.slab_rows);
		VITK_CHECK_LAUNCH();
		hipLaunchKernelGGL((gn_apply_kernel<T, V, ACT>), grid, block, apply_lds(p), st, x + at, gamma, beta, mu, rs, y + at, s, p.slab_rows, p.tpr);
		VITK_CHECK_LAUNCH();
	}
	return VITK_OK;
}

template <typename T, int V, int ACT>
int backward(const T* dy, const T* x, const float* gamma, const float* beta, const float* mean, const float* rstd, T* dx, float* dgamma, float* dbeta, int accumulate, int64_t B,
	const Shape& s, const Plan& p, float2* ws, hipStream_t st) {
	float2* chan = ws;                             // [n_part][C]
	float2* part = chan + p.n_part * s.C;          // two passes: [run][G][slabs], then [run][G] averages;  at the end the runs of the parameter sums
	if (p.width != 0) {
		const dim3 grid((unsigned)(vitk_cdiv(B, 8) * 8 * p.slices)), block(p.threads);
		const size_t lds = fused_lds(p, s.cpg);
		if (p.rows == 2) hipLaunchKernelGGL((gn_fused_bwd_kernel<T, V, 2, ACT>), grid, block, lds, st, dy, x, gamma, beta, mean, rstd, dx, chan, s, (int)B, p.width, p.slices);
		else if (p.rows == 5) hipLaunchKernelGGL((gn_fused_bwd_kernel<T, V, 5, ACT>), grid, block, lds, st, dy, x, gamma, beta, mean, rstd, dx, chan, s, (int)B, p.width, p.slices);
		else hipLaunchKernelGGL((gn_fused_bwd_kernel<T, V, MOST_ROWS, ACT>), grid, block, lds, st, dy, x, gamma, beta, mean, rstd, dx, chan, s, (int)B, p.width, p.slices);
		VITK_CHECK_LAUNCH();
	} else {
		for (int64_t b = 0; b < B; b += p.run) {
			const int64_t n = std::min(p.run, B - b), at = b * s.S * s.C;
			const dim3 grid((unsigned)p.slabs, (unsigned)n), block(p.tpr * p.k);
			hipLaunchKernelGGL((gn_bwd_stats_kernel<T, V, ACT>), grid, block, slab_lds(p, s.C), st, dy + at, x + at, gamma, beta, mean + b * s.G, rstd + b * s.G, chan + b * p.slabs * s.C, part,
				s, p.slab_rows, p.tpr);
			VITK_CHECK_LAUNCH();
			float2* avg = part + p.run * p.slabs * s.G;
			hipLaunchKernelGGL((gn_final_kernel<true>), dim3((unsigned)vitk_cdiv(n * s.G, 4)), dim3(256), 0, st, part, nullptr, nullptr, avg, s, (int)(n * s.G), p.slabs, p.slab_rows);
			VITK_CHECK_LAUNCH();
			hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V, ACT>), grid, block, apply_lds(p), st, dy + at, x + at, gamma, beta, mean + b * s.G, rstd + b * s.G, avg, dx + at, s, p.slab_rows, p.tpr);
			VITK_CHECK_LAUNCH();
		}
	}
	if (dgamma == nullptr && dbeta == nullptr) return VITK_OK;
	const unsigned cols = (unsigned)vitk_cdiv(s.C, 32);
	int64_t n = p.n_part;
	const float2* in = chan;
	if (n > PARAM_RUN) {  // (more than 128 rows: in two steps, so that more than C / 32 workgroups read them)
		const int64_t runs = vitk_cdiv(n, PARAM_RUN);
		VITK_REQUIRE(runs <= 65535, VITK_ERR_SHAPE);
		hipLaunchKernelGGL(gn_param_kernel, dim3(cols, (unsigned)runs), dim3(256), 0, st, in, part, nullptr, nullptr, n, PARAM_RUN, s.C, 0);
		VITK_CHECK_LAUNCH();
		in = part;
		n = runs;
	}
	hipLaunchKernelGGL(gn_param_kernel, dim3(cols, 1), dim3(256), 0, st, in, nullptr, dgamma, dbeta, n, (int)n, s.C, accumulate);
	VITK_CHECK_LAUNCH();
	return VITK_OK;
}

int64_t bytes_of(const Plan& p, int64_t C, int64_t G, bool bwd) {
	const int64_t part = p.width != 0 ? 0 : p.run * (p.slabs + 1) * G;
	if (!bwd) return part * 8;
	return (p.n_part * C + std::max(part, vitk_cdiv(p.n_part, PARAM_RUN) * C)) * 8;
}

template <typename T, int V> struct Call {
	template <typename... A> static int fwd(int act, A... args) {
		if (act == VITK_ACT_SILU) return forward<T, V, ACT_SILU>(args...);
		if (act == VITK_ACT_GELU) return forward<T, V, ACT_GELU>(args...);
		if (act == VITK_ACT_NONE) return forward<T, V, ACT_NONE>(args...);
		return forward<T, V, ACT_CLAMP>(args...);
	}
	template <typename... A> static int bwd(int act, A... args) {
		if (act == VITK_ACT_SILU) return backward<T, V, ACT_SILU>(args...);
		if (act == VITK_ACT_GELU) return backward<T, V, ACT_GELU>(args...);
		if (act == VITK_ACT_NONE) return backward<T, V, ACT_NONE>(args...);
		return backward<T, V, ACT_CLAMP>(args...);
	}
};

}  // namespace

extern "C" int64_t vitk_group_norm_workspace_bytes(int64_t B, int64_t S, int64_t C, int64_t G, int dtype) {
	const int rc = check(B, S, C, G, VITK_ACT_NONE, dtype);
	if (rc != VITK_OK) return rc;
	int64_t most = 0;
	for (int bwd = 0; bwd < 2; ++bwd)
		for (int al = 0; al < 2; ++al) most = std::max(most, bytes_of(plan_of(B, S, C, G, dtype == VITK_BF16 ? 2 : 4, al != 0, bwd != 0), C, G, bwd != 0));
	return most;
}

extern "C" int vitk_group_norm_fwd(const void* x, const float* gamma, const float* beta, void* y, float* mean, float* rstd, int64_t B, int64_t S, int64_t C, int64_t G, float eps, int act,
	int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
	VITK_REQUIRE(x && y, VITK_ERR_NULL);
	VITK_REQUIRE((mean == nullptr) == (rstd == nullptr), VITK_ERR_NULL);
	const int rc = check(B, S, C, G, act, dtype);
	if (rc != VITK_OK) return rc;
	const int es = dtype == VITK_BF16 ? 2 : 4;
	VITK_REQUIRE(vitk_aligned(x, es) && vitk_aligned(y, es), VITK_ERR_ALIGN);
	const Plan p = plan_of(B, S, C, G, es, vitk_aligned(x, 16) && vitk_aligned(y, 16), false);
	const int64_t need = bytes_of(p, C, G, false);
	VITK_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need && vitk_aligned(workspace, 8)), VITK_ERR_SCRATCH);
	const Shape s = shape_of(S, C, G, eps, act);
	hipStream_t st = (hipStream_t)stream;
	float2* ws = reinterpret_cast<float2*>(workspace);
	if (dtype == VITK_BF16) {
		const bf16_t* in = reinterpret_cast<const bf16_t*>(x);
		bf16_t* out = reinterpret_cast<bf16_t*>(y);
		if (p.V == 8) return Call<bf16_t, 8>::fwd(act, in, gamma, beta, out, mean, rstd, B, s, p, ws, st);
		if (p.V == 2) return Call<bf16_t, 2>::fwd(act, in, gamma, beta, out, mean, rstd, B, s, p, ws, st);
		return Call<bf16_t, 1>::fwd(act, in, gamma, beta, out, mean, rstd, B, s, p, ws, st);
	}
	const float* in = reinterpret_cast<const float*>(x);
	float* out = reinterpret_cast<float*>(y);
	if (p.V == 4) return Call<float, 4>::fwd(act, in, gamma, beta, out, mean, rstd, B, s, p, ws, st);
	if (p.V == 2) return Call<float, 2>::fwd(act, in, gamma, beta, out, mean, rstd, B, s, p, ws, st);
	return Call<float, 1>::fwd(act, in, gamma, beta, out, mean, rstd, B, s, p, ws, st);
}

extern "C" int vitk_group_norm_bwd(const void* dy, const void* x, const float* gamma, const float* beta, const float* mean, const float* rstd, void* dx, float* dgamma, float* dbeta,
	int accumulate, int64_t B, int64_t S, int64_t C, int64_t G, int act, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
	VITK_REQUIRE(dy && x && mean && rstd && dx, VITK_ERR_NULL);
	const int rc = check(B, S, C, G, act, dtype);
	if (rc != VITK_OK) return rc;
	const int es = dtype == VITK_BF16 ? 2 : 4;
	VITK_REQUIRE(vitk_aligned(x, es) && vitk_aligned(dy, es) && vitk_aligned(dx, es), VITK_ERR_ALIGN);
	const Plan p = plan_of(B, S, C, G, es, vitk_aligned(x, 16) && vitk_aligned(dy, 16) && vitk_aligned(dx, 16), true);
	VITK_REQUIRE(workspace != nullptr && workspace_bytes >= bytes_of(p, C, G, true) && vitk_aligned(workspace, 8), VITK_ERR_SCRATCH);
	const Shape s = shape_of(S, C, G, 0.f, act);
	hipStream_t st = (hipStream_t)stream;
	float2* ws = reinterpret_cast<float2*>(workspace);
	if (dtype == VITK_BF16) {
		const bf16_t *g = reinterpret_cast<const bf16_t*>(dy), *in = reinterpret_cast<const bf16_t*>(x);
		bf16_t* out = reinterpret_cast<bf16_t*>(dx);
		if (p.V == 8) return Call<bf16_t, 8>::bwd(act, g, in, gamma, beta, mean, rstd, out, dgamma, dbeta, accumulate, B, s, p, ws, st);
		if (p.V == 2) return Call<bf16_t, 2>::bwd(act, g, in, gamma, beta, mean, rstd, out, dgamma, dbeta, accumulate, B, s, p, ws, st);
		return Call<bf16_t, 1>::bwd(act, g, in, gamma, beta, mean, rstd, out, dgamma, dbeta, accumulate, B, s, p, ws, st);
	}
	const float *g = reinterpret_cast<const float*>(dy), *in = reinterpret_cast<const float*>(x);
	float* out = reinterpret_cast<float*>(dx);
	if (p.V == 4) return Call<float, 4>::bwd(act, g, in, gamma, beta, mean, rstd, out, dgamma, dbeta, accumulate, B, s, p, ws, st);
	if (p.V == 2) return Call<float, 2>::bwd(act, g, in, gamma, beta, mean, rstd, out, dgamma, dbeta, accumulate, B, s, p, ws, st);
	return Call<float, 1>::bwd(act, g, in, gamma, beta, mean, rstd, out, dgamma, dbeta, accumulate, B, s, p, ws, st);
}
