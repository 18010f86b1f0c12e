// C ABI of the biased / capped / masked attention: argument validation, the preparation of biases and tile ranges, the division of
// long axes among workgroups and the kernels that join its parts.
#include "attention_bias.h"

#include <climits>
#include <cmath>

namespace {

using namespace abias;

// ---- preparation: everything about biases and masks that does not depend on q and k ---------------------------------------------
// expand[h][i] = table[lookup[i]][h] in log2 units (0 where the bucket does not exist); ranges {least, greatest segment, least,
// greatest position} of every 64 rows, by which the attention kernels skip tiles without a visible pair and drop the mask in
// tiles that are wholly visible.
__global__ __launch_bounds__(256) void abias_expand_kernel(const float* __restrict__ table, const int* __restrict__ lookup, float* __restrict__ expand, int n, int n_bucket, int H) {
	for (int i = blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256) {
		const int bucket = lookup[i];
		for (int h = blockIdx.y; h < H; h += gridDim.y)
			expand[(int64_t)h * n + i] = (unsigned)bucket < (unsigned)n_bucket ? table[(int64_t)bucket * H + h] * LOG2E : 0.f;
	}
}

__device__ __forceinline__ void range_row(const int* seg, const int* pos, int64_t pos_stride, int4* out, int b, int g, int n64, int rows, int lane) {
	const int row = g * TB + lane, last = min(row, rows - 1);
	int s1 = seg != nullptr ? seg[(int64_t)b * rows + last] : 0, p0 = pos != nullptr ? pos[b * pos_stride + last] : 0;
	int s0 = s1 < 0 ? INT_MAX : s1, p1 = p0;
	const bool pad = __any(s1 < 0);
#pragma unroll
	for (int o = 32; o > 0; o >>= 1) {
		s0 = min(s0, __shfl_xor(s0, o, 64));
		s1 = max(s1, __shfl_xor(s1, o, 64));
		p0 = min(p0, __shfl_xor(p0, o, 64));
		p1 = max(p1, __shfl_xor(p1, o, 64));
	}
	if (lane == 0) out[(int64_t)b * n64 + g] = make_int4(pad ? ~s0 : s0, max(s1, -1), p0, p1);
}
__global__ __launch_bounds__(256) void abias_range_kernel(const int* qseg, const int* kseg, const int* qpos, const int* kpos, int64_t bqp, int64_t bkp, int4* qr, int4* kr, int B, int nq64,
	int nk64, int Sq, int Skv) {
	const int lane = threadIdx.x & 63;
	const int64_t n = (int64_t)B * (nq64 + nk64);
	for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < n; i += (int64_t)gridDim.x * 4) {
		const int b = (int)(i / (nq64 + nk64)), g = (int)(i % (nq64 + nk64));
		if (g < nq64) range_row(qseg, qpos, bqp, qr, b, g, nq64, Sq, lane);
		else range_row(kseg, kpos, bkp, kr, b, g - nq64, nk64, Skv, lane);
	}
}

// ---- joining the parts of a divided axis ------------------------------------------------------------------------------------------
// 16 lanes = one query row of a head, 8 columns each: out = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s
template <typename T>
__global__ __launch_bounds__(256) void abias_join_kernel(Args a) {
	const int64_t rows = (int64_t)a.B * a.H * a.Sq, row = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
	if (row >= rows) return;
	const int c0 = 8 * (threadIdx.x & 15);
	const float2* ml = reinterpret_cast<const float2*>(a.part + part_pairs(a.split, rows, a.dh));
	float m = -INFINITY;
	for (int s = 0; s < a.split; ++s) m = fmaxf(m, ml[s * rows + row].x);
	const float ms = m == -INFINITY ? 0.f : m;
	float l = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
	const bool vec = a.dh % 4 == 0;
	for (int s = 0; s < a.split; ++s) {
		const float2 x = ml[s * rows + row];
		const float w = __builtin_amdgcn_exp2f(x.x - ms);
		const float* po = a.part + (s * rows + row) * a.dh + c0;
		l = fmaf(w, x.y, l);
		float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
		if (vec) {
#pragma unroll
			for (int i = 0; i < 2; ++i)
				if (c0 + 4 * i < a.dh) {
					const f32x4 t = *reinterpret_cast<const f32x4*>(po + 4 * i);
#pragma unroll
					for (int e = 0; e < 4; ++e) v[4 * i + e] = t[e];
				}
		} else {
#pragma unroll
			for (int e = 0; e < 8; ++e)
				if (c0 + e < a.dh) v[e] = po[e];
		}
#pragma unroll
		for (int e = 0; e < 8; ++e) o[e] = fmaf(w, v[e], o[e]);
	}
	if (l == 0.f && m != -INFINITY) l = __builtin_nanf("");  // (scores of -inf alone: see the forward kernel)
	const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
	const int64_t bh = row / a.Sq, b = bh / a.H, h = bh % a.H, qi = row % a.Sq;
	T* op = reinterpret_cast<T*>(a.out_w) + b * a.bo + qi * a.ldo + h * a.dh;
#pragma unroll
	for (int i = 0; i < 2; ++i) {
		float v[4];
#pragma unroll
		for (int e = 0; e < 4; ++e) v[e] = o[4 * i + e] * inv;
		store4<T>(op, c0 + 4 * i, a.dh, a.ovec, v);
		if constexpr (sizeof(T) == 2) {
			if (a.rest != nullptr) {
#pragma unroll
				for (int e = 0; e < 4; ++e) v[e] = rest_of(v[e]);
				store4<bf16_t>(a.rest + (b * a.Sq + qi) * a.H * a.dh + h * a.dh, c0 + 4 * i, a.dh, a.dh % 4 == 0, v);
			}
		}
	}
	if (c0 == 0 && a.lse != nullptr) store_lse(a, row, m, l);
}

// delta += sum of the parts' sums of dz over the sum of their sums of p (see attention_bias_dq.h)
__global__ __launch_bounds__(256) void abias_delta_join_kernel(const float* __restrict__ part, float* __restrict__ delta, int split, int64_t rows) {
	for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows; i += (int64_t)gridDim.x * 256) {
		float s = 0.f, t = 0.f;
		for (int p = 0; p < split; ++p) {
			s += part[(p * rows + i) * 2];
			t += part[(p * rows + i) * 2 + 1];
		}
		delta[i] = t == 0.f ? 0.f : delta[i] + s / t;
	}
}

// out[b][row][head * dh + d] = sum over the parts, in their order; V columns a thread
template <typename T, int V>
__global__ __launch_bounds__(256) void abias_sum_kernel(const float* __restrict__ part, T* __restrict__ out, int split, int heads, int rows, int dh, int64_t n, int64_t ld, int64_t batch) {
	for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V; i < n; i += (int64_t)gridDim.x * 256 * V) {
		float s[V], v[V];
		load_vec<float, V>(part + i, s);
		for (int p = 1; p < split; ++p) {
			load_vec<float, V>(part + p * n + i, v);
#pragma unroll
			for (int e = 0; e < V; ++e) s[e] += v[e];
		}
		const int64_t r = i / dh, d = i % dh, bh = r / rows;
		store_vec<T, V>(out + bh / heads * batch + r % rows * ld + bh % heads * dh + d, s);
	}
}

// dtable[bucket][h] (+)= sum of the n workgroups' sums, in a fixed order: 32 buckets a workgroup, 8 runs of partial rows, joined in LDS
__global__ __launch_bounds__(256) void abias_table_sum_kernel(const float* __restrict__ part, float* __restrict__ dtable, int n, int n_bucket, int H, int accumulate) {
	__shared__ float red[8][32];
	const int h = blockIdx.y, i = blockIdx.x * 32 + (threadIdx.x & 31), g = threadIdx.x >> 5;
	float s = 0.f;
	if (i < n_bucket) {
		const float* p = part + (int64_t)h * n * n_bucket + i;
		for (int w = g; w < n; w += 8) s += p[(int64_t)w * n_bucket];
	}
	red[g][threadIdx.x & 31] = s;
	__syncthreads();
	if (g == 0 && i < n_bucket) {
		for (int c = 1; c < 8; ++c) s += red[c][threadIdx.x];
		float* out = dtable + (int64_t)i * H + h;
		*out = accumulate ? *out + s : s;
	}
}

// ---- host -------------------------------------------------------------------------------------------------------------------------
constexpr int64_t MAX_ROWS = 1 << 30;
constexpr int64_t MAX_LD = 1 << 21;  // elements: 128 rows stay below 2^31 bytes, the reach of a buffer load's offset
constexpr int TABLE_GRAD_BUCKETS = 8192;  // 32 KB of bucket sums beside the tiles

inline int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }
inline bool needs_ranges(const vitk_biased_attention_desc& d) { return d.q_seg != nullptr || (d.q_pos != nullptr && (d.table != nullptr || d.slopes != nullptr)); }

inline bool keeps_rest(const vitk_biased_attention_desc& d) { return d.keep_rest != 0 && d.dtype == VITK_BF16; }
inline bool keeps_lse_rest(const vitk_biased_attention_desc& d) { return d.keep_rest != 0 && d.dtype == VITK_F32 && d.slopes != nullptr; }

struct Prep {
	int64_t expand, qr, kr, rest, total;
};
Prep prep_layout(const vitk_biased_attention_desc& d) {
	Prep p{};
	p.expand = 0;
	p.qr = d.table != nullptr ? up256(d.n_head * d.n_lookup * 4) : 0;
	p.kr = p.qr;
	p.total = p.qr;
	if (needs_ranges(d)) {
		p.kr = p.qr + up256(d.B * vitk_cdiv(d.Sq, TB) * 16);
		p.total = p.kr + up256(d.B * vitk_cdiv(d.Skv, TB) * 16);
	}
	p.rest = p.total;
	if (keeps_rest(d)) p.total += up256(d.B * d.Sq * d.n_head * d.dh * 2);
	if (keeps_lse_rest(d)) p.total += up256(d.B * d.Sq * d.n_head * 4);
	return p;
}

// Parts of a divided axis: with fewer than 512 workgroups (two for each of the 256 CUs) and at least 8 tiles to walk, as many parts as bring
// 1024 workgroups, of 4 tiles or more each.  One query of 12 heads over 16384 keys, batch 16: 192 workgroups undivided.
int split_of(int64_t workgroups, int64_t tiles) {
	if (workgroups >= 512 || tiles < 8) return 1;
	const int64_t s = std::min(vitk_cdiv(1024, workgroups), vitk_cdiv(tiles, 4));
	return (int)std::max<int64_t>(1, std::min<int64_t>(s, 256));
}
void set_split(Args& a, int64_t own_rows, int64_t heads, int64_t tiles) {
	a.nblk = (int)vitk_cdiv(own_rows, QB);
	a.split = split_of((int64_t)a.B * heads * a.nblk, tiles);
	a.per_split = (int)vitk_cdiv(tiles, a.split);
	a.split = (int)vitk_cdiv(tiles, a.per_split);
}
// Table gradient: at most about 2048 workgroups by tiles of keys; where tile pairs are fewer than 1024, the batch is divided too, 4 images or more to
// a workgroup (a scatter costs about as much as the scores of 2 images).
TablePlan table_plan(const Args& a) {
	const int64_t rows = (int64_t)a.H * vitk_cdiv(a.Sq, QB);
	TablePlan p{};
	const int64_t want = std::max<int64_t>(1, std::min<int64_t>(a.nk64, vitk_cdiv(2048, rows)));
	p.chunk = (int)vitk_cdiv(a.nk64, want);
	p.nchunk = (int)vitk_cdiv(a.nk64, p.chunk);
	const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(vitk_cdiv(1024, rows * p.nchunk), a.B / 4));
	p.images = (int)vitk_cdiv(a.B, parts);
	p.nimages = (int)vitk_cdiv(a.B, p.images);
	return p;
}

int check(const vitk_biased_attention_desc& d) {
	VITK_REQUIRE(d.dtype == VITK_F32 || d.dtype == VITK_BF16, VITK_ERR_DTYPE);
	VITK_REQUIRE(d.B > 0 && d.n_head > 0 && d.n_kv_head > 0 && d.Sq > 0 && d.Skv > 0 && d.dh > 0, VITK_ERR_SHAPE);
	VITK_REQUIRE(d.dh <= 128 && d.B <= (1 << 20) && d.n_head <= (1 << 16) && d.Sq <= MAX_ROWS && d.Skv <= MAX_ROWS, VITK_ERR_SHAPE);
	VITK_REQUIRE(d.n_head % d.n_kv_head == 0, VITK_ERR_SHAPE);
	const int64_t hq = d.n_head * d.dh, hk = d.n_kv_head * d.dh;
	VITK_REQUIRE(d.ldq >= hq && d.ldo >= hq && d.ldk >= hk && d.ldv >= hk, VITK_ERR_SHAPE);
	VITK_REQUIRE(d.ldq <= MAX_LD && d.ldk <= MAX_LD && d.ldv <= MAX_LD && d.ldo <= MAX_LD && d.lddo <= MAX_LD, VITK_ERR_SHAPE);
	VITK_REQUIRE(d.batch_q >= 0 && d.batch_k >= 0 && d.batch_v >= 0 && d.batch_o >= 0, VITK_ERR_SHAPE);
	VITK_REQUIRE(std::isfinite(d.scale) && std::isfinite(d.softcap) && d.softcap >= 0.f, VITK_ERR_SHAPE);
	VITK_REQUIRE((d.q_seg == nullptr) == (d.k_seg == nullptr), VITK_ERR_NULL);
	VITK_REQUIRE((d.q_pos == nullptr) == (d.k_pos == nullptr), VITK_ERR_NULL);
	VITK_REQUIRE(d.batch_qpos >= 0 && d.batch_kpos >= 0, VITK_ERR_SHAPE);
	VITK_REQUIRE(d.prefix == nullptr || d.causal, VITK_ERR_UNSUPPORTED);
	if (d.table != nullptr) {
		VITK_REQUIRE(d.lookup != nullptr, VITK_ERR_NULL);
		VITK_REQUIRE(d.n_lookup > 0 && d.n_lookup <= MAX_ROWS && d.n_bucket > 0 && d.n_bucket <= MAX_ROWS, VITK_ERR_SHAPE);
		VITK_REQUIRE(d.lookup_lo >= -MAX_ROWS && d.lookup_lo <= MAX_ROWS && d.lookup_lo + d.n_lookup <= 2 * MAX_ROWS - 1, VITK_ERR_SHAPE);
	}
	return VITK_OK;
}

struct Aligner {  // the widest loads / stores that every pointer and stride allows
	int64_t bits = 0;
	void add(const void* p, int64_t ld, int64_t batch, int es) { bits |= (int64_t)reinterpret_cast<uintptr_t>(p) | ld * es | batch * es; }
	bool ok(int64_t n) const { return (bits & (n - 1)) == 0; }
};

Args make_args(const vitk_biased_attention_desc& d) {
	Args a{};
	a.q = d.q; a.k = d.k; a.v = d.v; a.out = d.out; a.out_w = d.out; a.lse = d.lse;
	a.dout = d.dout; a.dq = d.dq; a.dk = d.dk; a.dv = d.dv;
	a.B = (int)d.B; a.H = (int)d.n_head; a.Hkv = (int)d.n_kv_head; a.G = a.H / a.Hkv; a.Sq = (int)d.Sq; a.Skv = (int)d.Skv; a.dh = (int)d.dh;
	a.ldq = d.ldq; a.ldk = d.ldk; a.ldv = d.ldv; a.ldo = d.ldo; a.lddo = d.lddo; a.lddq = d.lddq; a.lddk = d.lddk; a.lddv = d.lddv;
	a.bq = d.batch_q; a.bk = d.batch_k; a.bv = d.batch_v; a.bo = d.batch_o; a.bdo = d.batch_do; a.bdq = d.batch_dq; a.bdk = d.batch_dk; a.bdv = d.batch_dv;
	a.scale = d.scale > 0.f ? d.scale : 1.0f / sqrtf((float)d.dh);
	a.c = a.scale * LOG2E;
	a.cap_l2 = d.softcap * LOG2E;
	a.inv_cap = d.softcap > 0.f ? a.scale / d.softcap : 0.f;
	a.causal = d.causal != 0;
	a.off = a.Skv - a.Sq;
	a.prefix = d.prefix;
	a.qseg = d.q_seg; a.kseg = d.k_seg;
	a.slopes = d.slopes;
	if (d.table != nullptr || d.slopes != nullptr) {
		a.qpos = d.q_pos; a.kpos = d.k_pos;
		a.bqp = d.batch_qpos; a.bkp = d.batch_kpos;
	}
	if (d.table != nullptr) {
		a.lookup = d.lookup; a.n_lookup = (int)d.n_lookup; a.lookup_lo = (int)d.lookup_lo; a.n_bucket = (int)d.n_bucket;
	}
	a.nq64 = (int)vitk_cdiv(d.Sq, TB);
	a.nk64 = (int)vitk_cdiv(d.Skv, TB);
	const int es = d.dtype == VITK_BF16 ? 2 : 4;
	Aligner in, out;
	in.add(d.q, d.ldq, d.batch_q, es);
	in.add(d.k, d.ldk, d.batch_k, es);
	in.add(d.v, d.ldv, d.batch_v, es);
	in.add(nullptr, d.dh, 0, es);
	out.add(nullptr, d.dh, 0, es);
	out.add(d.out, d.ldo, d.batch_o, es);
	if (d.dout != nullptr) {
		in.add(d.dout, d.lddo, d.batch_do, es);
		in.add(d.out, d.ldo, d.batch_o, es);
		out.add(d.dq, d.lddq, d.batch_dq, es);
		out.add(d.dk, d.lddk, d.batch_dk, es);
		out.add(d.dv, d.lddv, d.batch_dv, es);
	}
	a.gran = in.ok(16) ? 16 : (in.ok(8) ? 8 : es);
	a.ovec = es == 2 && out.ok(16) ? 2 : out.ok(4 * es);
	return a;
}

void use_prep(Args& a, const vitk_biased_attention_desc& d) {
	const Prep p = prep_layout(d);
	char* base = reinterpret_cast<char*>(d.prep);
	if (d.table != nullptr) a.expand = reinterpret_cast<const float*>(base + p.expand);
	if (keeps_rest(d)) a.rest = reinterpret_cast<bf16_t*>(base + p.rest);
	if (keeps_lse_rest(d)) a.lse_rest = reinterpret_cast<float*>(base + p.rest);
	if (needs_ranges(d)) {
		a.qr = reinterpret_cast<const int4*>(base + p.qr);
		a.kr = reinterpret_cast<const int4*>(base + p.kr);
	}
}

struct BwdSpace {
	int64_t delta, table, rows, part, total;
};
BwdSpace bwd_layout(const vitk_biased_attention_desc& d) {
	Args a = make_args(d);
	BwdSpace s{};
	const int64_t qrows = d.B * d.n_head * d.Sq, krows = d.B * d.n_kv_head * d.Skv;
	int64_t part = 0, table = 0, rows = 0;
	set_split(a, d.Sq, d.n_head, a.nk64);
	if (a.split > 1) part = a.split * qrows * d.dh * 4;
	if (d.dtable != nullptr) {
		const TablePlan p = table_plan(a);
		table = d.n_head * vitk_cdiv(d.Sq, QB) * p.nchunk * p.nimages * d.n_bucket * 4;
		if (a.split > 1) rows = (int64_t)a.split * qrows * 8;
	}
	set_split(a, d.Skv, d.n_kv_head, a.nq64);
	if (a.split > 1) part = std::max(part, 2 * a.split * krows * d.dh * 4);
	s.delta = 0;
	s.table = up256(qrows * 4);
	s.rows = s.table + up256(table);
	s.part = s.rows + up256(rows);
	s.total = s.part + up256(part);
	return s;
}

}  // namespace

extern "C" int64_t vitk_biased_attention_prep_bytes(const vitk_biased_attention_desc* d) {
	if (d == nullptr) return VITK_ERR_NULL;
	const int rc = check(*d);
	return rc != VITK_OK ? rc : prep_layout(*d).total;
}

extern "C" int64_t vitk_biased_attention_workspace_bytes(const vitk_biased_attention_desc* d, int backward) {
	if (d == nullptr) return VITK_ERR_NULL;
	const int rc = check(*d);
	if (rc != VITK_OK) return rc;
	if (backward) return bwd_layout(*d).total;
	Args a = make_args(*d);
	set_split(a, d->Sq, d->n_head, a.nk64);
	return a.split > 1 ? up256(part_bytes(a.split, d->B * d->n_head * d->Sq, d->dh)) : 0;
}

extern "C" int vitk_biased_attention_fwd(const vitk_biased_attention_desc* dp, void* stream) {
	VITK_REQUIRE(dp != nullptr, VITK_ERR_NULL);
	const vitk_biased_attention_desc& d = *dp;
	VITK_REQUIRE(d.q && d.k && d.v && d.out, VITK_ERR_NULL);
	int rc = check(d);
	if (rc != VITK_OK) return rc;
	hipStream_t st = (hipStream_t)stream;
	Args a = make_args(d);
	a.dout = nullptr;
	const Prep p = prep_layout(d);
	VITK_REQUIRE(p.total == 0 || d.prep != nullptr, VITK_ERR_NULL);
	VITK_REQUIRE(d.prep_bytes >= p.total && vitk_aligned(d.prep, 16), VITK_ERR_SCRATCH);
	set_split(a, d.Sq, d.n_head, a.nk64);
	if (a.split > 1) {
		const int64_t need = part_bytes(a.split, d.B * d.n_head * d.Sq, d.dh);
		VITK_REQUIRE(d.workspace != nullptr, VITK_ERR_NULL);
		VITK_REQUIRE(d.workspace_bytes >= need && vitk_aligned(d.workspace, 16), VITK_ERR_SCRATCH);
		a.part = reinterpret_cast<float*>(d.workspace);
	}
	use_prep(a, d);
	const int64_t rows = d.B * d.n_head * d.Sq;
	VITK_REQUIRE(placed_blocks(a.nblk, d.B * d.n_head, a.split) < (1 << 24) && (a.split == 1 || vitk_cdiv(rows, 16) < (1 << 24)), VITK_ERR_SHAPE);
	if (d.table != nullptr) {
		const dim3 grid((unsigned)std::min<int64_t>(vitk_cdiv(d.n_lookup, 256), 1024), (unsigned)std::min<int64_t>(d.n_head, 64));
		hipLaunchKernelGGL(abias_expand_kernel, grid, dim3(256), 0, st, d.table, d.lookup, const_cast<float*>(a.expand), a.n_lookup, a.n_bucket, a.H);
		VITK_CHECK_LAUNCH();
	}
	if (needs_ranges(d)) {
		const int64_t n = d.B * (a.nq64 + a.nk64);
		hipLaunchKernelGGL(abias_range_kernel, dim3((unsigned)std::min<int64_t>(vitk_cdiv(n, 4), 2048)), dim3(256), 0, st, a.qseg, a.kseg, a.qpos, a.kpos, a.bqp, a.bkp, const_cast<int4*>(a.qr),
			const_cast<int4*>(a.kr), a.B, a.nq64, a.nk64, a.Sq, a.Skv);
		VITK_CHECK_LAUNCH();
	}
	rc = d.dtype == VITK_BF16 ? vitk_abias_fwd_bf16(a, st) : vitk_abias_fwd_f32(a, st);
	if (rc != VITK_OK || a.split == 1) return rc;
	const dim3 grid((unsigned)vitk_cdiv(rows, 16));
	if (d.dtype == VITK_BF16) hipLaunchKernelGGL(abias_join_kernel<bf16_t>, grid, dim3(256), 0, st, a);
	else hipLaunchKernelGGL(abias_join_kernel<float>, grid, dim3(256), 0, st, a);
	VITK_CHECK_LAUNCH();
	return VITK_OK;
}

template <typename T>
static int sum_parts(const float* part, void* out, int vec, int split, int64_t B, int64_t heads, int64_t rows, int64_t dh, int64_t ld, int64_t batch, hipStream_t st) {
	const int64_t n = B * heads * rows * dh;
	const dim3 grid((unsigned)std::min<int64_t>(vitk_cdiv(n, vec ? 1024 : 256), 8192)), block(256);
	if (vec) hipLaunchKernelGGL((abias_sum_kernel<T, 4>), grid, block, 0, st, part, reinterpret_cast<T*>(out), split, (int)heads, (int)rows, (int)dh, n, ld, batch);
	else hipLaunchKernelGGL((abias_sum_kernel<T, 1>), grid, block, 0, st, part, reinterpret_cast<T*>(out), split, (int)heads, (int)rows, (int)dh, n, ld, batch);
	VITK_CHECK_LAUNCH();
	return VITK_OK;
}

extern "C" int vitk_biased_attention_bwd(const vitk_biased_attention_desc* dp, void* stream) {
	VITK_REQUIRE(dp != nullptr, VITK_ERR_NULL);
	const vitk_biased_attention_desc& d = *dp;
	VITK_REQUIRE(d.q && d.k && d.v && d.out && d.lse && d.dout && d.dq && d.dk && d.dv, VITK_ERR_NULL);
	int rc = check(d);
	if (rc != VITK_OK) return rc;
	const int64_t hq = d.n_head * d.dh, hk = d.n_kv_head * d.dh;
	VITK_REQUIRE(d.lddo >= hq && d.lddq >= hq && d.lddk >= hk && d.lddv >= hk, VITK_ERR_SHAPE);
	VITK_REQUIRE(d.batch_do >= 0 && d.batch_dq >= 0 && d.batch_dk >= 0 && d.batch_dv >= 0, VITK_ERR_SHAPE);
	// (a gradient is written once: rows of different images must not meet)
	VITK_REQUIRE(d.B == 1 || (d.batch_dq >= d.lddq && d.batch_dk >= d.lddk && d.batch_dv >= d.lddv), VITK_ERR_SHAPE);
	VITK_REQUIRE(d.dtable == nullptr || d.table != nullptr, VITK_ERR_NULL);
	VITK_REQUIRE(d.dtable == nullptr || d.n_bucket <= TABLE_GRAD_BUCKETS, VITK_ERR_UNSUPPORTED);
	const Prep p = prep_layout(d);
	VITK_REQUIRE(p.total == 0 || d.prep != nullptr, VITK_ERR_NULL);
	VITK_REQUIRE(d.prep_bytes >= p.total && vitk_aligned(d.prep, 16), VITK_ERR_SCRATCH);
	const BwdSpace s = bwd_layout(d);
	VITK_REQUIRE(d.workspace != nullptr, VITK_ERR_NULL);
	VITK_REQUIRE(d.workspace_bytes >= s.total && vitk_aligned(d.workspace, 16), VITK_ERR_SCRATCH);
	hipStream_t st = (hipStream_t)stream;
	Args a = make_args(d);
	use_prep(a, d);
	char* ws = reinterpret_cast<char*>(d.workspace);
	a.delta = reinterpret_cast<float*>(ws + s.delta);
	a.part = reinterpret_cast<float*>(ws + s.part);
	const bool bf = d.dtype == VITK_BF16;
	set_split(a, d.Sq, d.n_head, a.nk64);
	a.row_part = reinterpret_cast<float*>(ws + s.rows);
	rc = bf ? vitk_abias_dq_bf16(a, d.dtable != nullptr, st) : vitk_abias_dq_f32(a, d.dtable != nullptr, st);
	if (rc != VITK_OK) return rc;
	if (d.dtable != nullptr) {
		if (a.split > 1) {
			const int64_t rows = d.B * d.n_head * d.Sq;
			hipLaunchKernelGGL(abias_delta_join_kernel, dim3((unsigned)std::min<int64_t>(vitk_cdiv(rows, 256), 2048)), dim3(256), 0, st, a.row_part, a.delta, a.split, rows);
			VITK_CHECK_LAUNCH();
		}
		float* sums = reinterpret_cast<float*>(ws + s.table);
		const TablePlan tp = table_plan(a);
		rc = bf ? vitk_abias_table_bf16(a, tp, sums, st) : vitk_abias_table_f32(a, tp, sums, st);
		if (rc != VITK_OK) return rc;
		hipLaunchKernelGGL(abias_table_sum_kernel, dim3((unsigned)vitk_cdiv(a.n_bucket, 32), (unsigned)a.H), dim3(256), 0, st, sums, d.dtable, a.nblk * tp.nchunk * tp.nimages, a.n_bucket, a.H,
			d.accumulate_dtable);
		VITK_CHECK_LAUNCH();
	}
	if (a.split > 1) {
		rc = bf ? sum_parts<bf16_t>(a.part, d.dq, a.ovec, a.split, d.B, d.n_head, d.Sq, d.dh, d.lddq, d.batch_dq, st) : sum_parts<float>(a.part, d.dq, a.ovec, a.split, d.B, d.n_head, d.Sq, d.dh, d.lddq, d.batch_dq, st);
		if (rc != VITK_OK) return rc;
	}
	set_split(a, d.Skv, d.n_kv_head, a.nq64);
	rc = bf ? vitk_abias_dkv_bf16(a, st) : vitk_abias_dkv_f32(a, st);
	if (rc != VITK_OK) return rc;
	if (a.split > 1) {
		const float* pv = a.part + (int64_t)a.split * d.B * d.n_kv_head * d.Skv * d.dh;
		rc = bf ? sum_parts<bf16_t>(a.part, d.dk, a.ovec, a.split, d.B, d.n_kv_head, d.Skv, d.dh, d.lddk, d.batch_dk, st) : sum_parts<float>(a.part, d.dk, a.ovec, a.split, d.B, d.n_kv_head, d.Skv, d.dh, d.lddk, d.batch_dk, st);
		if (rc != VITK_OK) return rc;
		rc = bf ? sum_parts<bf16_t>(pv, d.dv, a.ovec, a.split, d.B, d.n_kv_head, d.Skv, d.dh, d.lddv, d.batch_dv, st) : sum_parts<float>(pv, d.dv, a.ovec, a.split, d.B, d.n_kv_head, d.Skv, d.dh, d.lddv, d.batch_dv, st);
		if (rc != VITK_OK) return rc;
	}
	return VITK_OK;
}
