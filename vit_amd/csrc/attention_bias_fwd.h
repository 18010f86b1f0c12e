// Forward of the biased / capped / masked attention (mathematics, tiles and orientation: attention_bias.h).
//
// One workgroup = 128 queries of one head, a wave 32 of them; keys in tiles of 64 with a running maximum and sum.
//   S^T[key][q] = K Q^T (A = K rows from LDS, B = the wave's Q rows in registers);  O^T[d][q] += V^T P^T (A = V columns by the
//   transposing LDS read, B = P^T as it stands in the accumulators)
// The next tile's rows fly to registers while a tile is worked on.  The accumulator is rescaled only in tiles where a maximum
// of the wave grows.  With few blocks of queries the keys are cut into parts (a single query over a long cache), each workgroup
// leaving (maximum, sum, unnormalised output) for attention_bias.hip to join.
#pragma once

#include "attention_bias.h"

namespace {

using namespace abias;

// Waves of a SIMD: three for up to 64 columns of bfloat16 (32 of float32), two for twice that, one for 128 of float32.  With a table three for 32 columns
// of bfloat16 alone: 64 spill 65 registers then (8 heads x 4096^2, training: 680 us with three, 591 with two).  Elsewhere three and two are near each other
// (8 x 12 heads x 1024^2 of 64 columns: 45.8 and 45.4 us, capped 63.2 and 63.9; 16 x 32 heads x 784^2 x 12 with a table: 196 and 192).
template <typename T, int DHP, int GR, bool CAP, int BIAS>
__global__ __launch_bounds__(256, DHP * (int)sizeof(T) >= 512 ? 1 : (DHP * (int)sizeof(T) <= (BIAS == BIAS_TABLE ? 64 : 128) ? 3 : 2)) void abias_fwd_kernel(Args a) {
	typedef Img<T, DHP> I;
	__shared__ __attribute__((aligned(16))) char Ks[I::BYTES];
	__shared__ __attribute__((aligned(16))) char Vs[I::BYTES];
	__shared__ float win[BIAS == BIAS_TABLE ? WIN : 1];
	__shared__ __attribute__((aligned(16))) int kpos_s[TB], kseg_s[TB], bad_s[TB + 1];
	int bh, blk, part;
	if (!place(a.nblk, a.B * a.H, a.split, bh, blk, part, a.causal != 0)) return;
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
	const int b = bh / a.H, h = bh - b * a.H, hk = h / a.G;
	const int q0 = blk * QB, qi = q0 + 32 * wave + (lane & 31);
	Own o{};
	o.seg = a.qseg != nullptr ? (qi < a.Sq ? a.qseg[(int64_t)b * a.Sq + qi] : -1) : 0;
	const bool own_ok = qi < a.Sq && o.seg >= 0;  // (rows of a negative segment are not read: they see no key)
	const T* kb = reinterpret_cast<const T*>(a.k) + b * a.bk + hk * a.dh;
	const T* vb = reinterpret_cast<const T*>(a.v) + b * a.bv + hk * a.dh;
	const Rows qx = rows_of<T>(reinterpret_cast<const T*>(a.q) + b * a.bq + h * a.dh, a.ldq, q0, a.Sq, QB, a.dh);
	typename Tr<T>::frag qf[I::STEPS];
#pragma unroll
	for (int s = 0; s < I::STEPS; ++s) qf[s] = own_frag<T, GR>(qx, qi - q0, a.ldq, s, a.dh, a.gran, own_ok, lane);

	const bool pos = BIAS != BIAS_NONE && a.kpos != nullptr;
	const int prefix = a.prefix != nullptr ? a.prefix[b] : 0;
	const int* kseg = a.kseg != nullptr ? a.kseg + (int64_t)b * a.Skv : nullptr;
	const int* kpos = pos ? a.kpos + b * a.bkp : nullptr;
	const int4* kr = a.kr != nullptr ? a.kr + (int64_t)b * a.nk64 : nullptr;
	const int q1 = min(q0 + QB, a.Sq) - 1;
	const Span own = span_of(a.qr != nullptr ? a.qr + (int64_t)b * a.nq64 : nullptr, 2 * blk, a.nq64, pos, q0 + a.off, q0 + QB - 1 + a.off);
	o.lim = limit_of(a, qi, o.seg, prefix);
	if constexpr (BIAS != BIAS_NONE) {
		o.pos = pos ? (qi < a.Sq ? a.qpos[b * a.bqp + qi] : own.pmin) : qi + a.off;
		o.slope = a.slopes != nullptr ? a.slopes[h] * LOG2E : 0.f;
		o.ex = BIAS == BIAS_TABLE ? a.expand + (int64_t)h * a.n_lookup : nullptr;
	}

	float m = -INFINITY, l = 0.f, poison = 0.f;
	f32x16 acc[I::ND];
#pragma unroll
	for (int dt = 0; dt < I::ND; ++dt)
#pragma unroll
		for (int r = 0; r < 16; ++r) acc[dt][r] = 0.f;

	// float32: the scale in front of the maximum, so that the greatest score's weight is 1 exactly (as the scale of the exponent's multiply-add it is
	// off by the rounding of the maximum), and out of a row that sees one key is that key's value
	constexpr bool SCALE_FIRST = sizeof(T) == 4 && !CAP && BIAS == BIAS_NONE;
	Stage<T, DHP, GR> kst, vst;
	kst.init(a.ldk, a.dh);
	vst.init(a.ldv, a.dh);
	float wreg[WIN / 256];
	int preg = 0, sreg = 0;
	Window wn{0, WIN_ONE};
	bool full_n = false;
	auto fetch_tile = [&](int t) {
		const int k0 = t * TB;
		const int* sg = full_n ? nullptr : kseg;
		const int* sgt = sg != nullptr ? sg + k0 : nullptr;
		const uint32_t hid = sgt != nullptr ? Stage<T, DHP, GR>::hidden(sgt, a.Skv - k0) : 0u;
		kst.fetch(rows_of<T>(kb, a.ldk, k0, a.Skv, TB, a.dh), a.dh, a.gran, hid);
		vst.fetch(rows_of<T>(vb, a.ldv, k0, a.Skv, TB, a.dh), a.dh, a.gran, hid);
		int plo = k0, phi = k0 + TB - 1;
		if (pos) {
			const i32x4 r = range_at(kr, t);
			plo = r.z;
			phi = r.w;
		}
		if (threadIdx.x < TB) {
			const int key = k0 + (int)threadIdx.x;
			if (pos) preg = key < a.Skv ? kpos[key] : plo;
			if (sg != nullptr) sreg = key < a.Skv ? sg[key] : -1;
		}
		if constexpr (BIAS == BIAS_TABLE) {
			wn = window_of(a, plo - own.pmax, phi - own.pmin);
			if (wn.mode == WIN_LDS) {
				const int n = phi - own.pmin - wn.lo + 1;
#pragma unroll
				for (int i = 0; i < WIN / 256; ++i) {
					const int j = (int)threadIdx.x + 256 * i;
					if (j < n) wreg[i] = o.ex[lookup_index(a, wn.lo + j)];
				}
			}
		}
	};

	Walk<true> walk;
	const int t_end = (int)min((int64_t)a.nk64, (int64_t)(part + 1) * a.per_split);
	walk.start(a, part * a.per_split, t_end, q0, q1, own, kr, prefix, lane);
	if (threadIdx.x == 0) bad_s[TB] = -1;
	int t = walk.next(a, q0, q1, own, kr, prefix, lane, full_n);
	if (t >= 0) fetch_tile(t);
	const TileSide ts{win, kpos_s, kseg_s, nullptr};
	while (t >= 0) {
		const int k0 = t * TB;
		const Window w = wn;
		const bool full = full_n;
		__syncthreads();  // every wave is done with the previous tile
		kst.commit(Ks);
		vst.commit(Vs);
		if (threadIdx.x < TB) {
			if (pos) kpos_s[threadIdx.x] = BIAS == BIAS_TABLE ? preg * 4 : preg;
			if (kseg != nullptr) kseg_s[threadIdx.x] = sreg;
		}
		if constexpr (BIAS == BIAS_TABLE) {
			if (w.mode == WIN_LDS) {
#pragma unroll
				for (int i = 0; i < WIN / 256; ++i) win[threadIdx.x + 256 * i] = fmaf(-o.slope, fabsf((float)(w.lo + (int)threadIdx.x + 256 * i)), wreg[i]);
			}
		}
		const bool special = settle_tile(full, t, kst, Ks, vst, Vs, bad_s);
		t = walk.next(a, q0, q1, own, kr, prefix, lane, full_n);
		if (t >= 0) fetch_tile(t);
		if (q0 + 32 * wave >= a.Sq) continue;  // (no row of this wave exists: it only helps with the staging)

		if (special) poison += sees_marked<true>(a, ts, o, k0, bad_s, lane);
		const int lv = anew(lane);
		f32x16 z[2];
		float bm = -INFINITY;
#pragma unroll
		for (int i = 0; i < 2; ++i) {
#pragma unroll
			for (int r = 0; r < 16; ++r) z[i][r] = 0.f;
#pragma unroll
			for (int s = 0; s < I::STEPS; ++s) z[i] = Tr<T>::mma(row_frag<T, DHP>(Ks, 32 * i, s, lane), qf[s], z[i]);
			f32x16 tn;
			modify<true, CAP, BIAS>(z[i], tn, a, w, ts, o, pos, k0, 32 * i, lv);
			if constexpr (SCALE_FIRST) {
#pragma unroll
				for (int r = 0; r < 16; ++r) z[i][r] *= a.c;
			}
			if (!full) hide<true>(z[i], a, ts, o, k0, 32 * i, lv);
#pragma unroll
			for (int r = 0; r < 16; ++r) bm = fmaxf(bm, z[i][r]);
		}
		bm = pair_max(bm);
		if constexpr (!CAP && BIAS == BIAS_NONE && !SCALE_FIRST) bm *= a.c;
		if (__any(bm > m)) {
			const float mn = fmaxf(m, bm);
			const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
			m = mn;
			l *= alpha;
#pragma unroll
			for (int dt = 0; dt < I::ND; ++dt)
#pragma unroll
				for (int r = 0; r < 16; ++r) acc[dt][r] *= alpha;
		}
		const float ms = m == -INFINITY ? 0.f : m;  // (a row that has seen no key yet: all its z are -inf)
		float ls = 0.f;
#pragma unroll
		for (int i = 0; i < 2; ++i)
#pragma unroll
			for (int r = 0; r < 16; ++r) {
				const float p = SCALE_FIRST ? __builtin_amdgcn_exp2f(z[i][r] - ms) : score_exp<CAP, BIAS>(a, z[i][r], ms);
				z[i][r] = p;
				ls += p;
			}
		l += ls;
#pragma unroll
		for (int i = 0; i < 2; ++i) {
			outer<T, DHP>(acc, Vs, 32 * i, z[i], lane);
		}
	}
	l = pair_sum(l) + pair_sum(poison);
	// A row that sees keys and has no weight: its scores are all -inf, which is no softmax, and no row that sees nothing.  Infinities in q reach every key: a
	// look at what the row sees settles it.  Those of k are noticed in partly visible tiles (poison); behind a wholly visible one the row has seen keys, and
	// other parts of the keys may still have weight (a maximum that is finite tells the join).
	if (__any(l == 0.f && o.lim > 0)) {
		uint32_t c = 0;
#pragma unroll
		for (int s = 0; s < I::STEPS; ++s) c |= Stage<T, DHP, GR>::special(__builtin_bit_cast(u32x4, qf[s]));
		c |= __shfl_xor(c, 32, 64);
		bool sees = false;
		if (l == 0.f && c != 0) {
			const int end = min(min(a.Skv, o.lim), t_end * TB);
			for (int j = part * a.per_split * TB; j < end && !sees; ++j) sees = kseg == nullptr || kseg[j] == o.seg;
		}
		if (sees) l = __builtin_nanf("");
		if (l == 0.f && walk.any_full && o.lim > 0) {
			if (a.split > 1) m = -FLT_MAX;
			else l = __builtin_nanf("");
		}
	}
	if (qi >= a.Sq) return;
	if (a.split > 1) {
		const int64_t rows = (int64_t)a.B * a.H * a.Sq, row = (int64_t)bh * a.Sq + qi;
		store_tiles<float, I::ND>(a.part + ((int64_t)part * rows + row) * a.dh, a.dh, a.dh % 4 == 0, lane, [&](int dt, int r) { return acc[dt][r]; });
		if (lane < 32) {
			reinterpret_cast<float2*>(a.part + part_pairs(a.split, rows, a.dh))[part * rows + row] = make_float2(m, l);
		}
		return;
	}
	const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // (a row without a visible key is 0; NaN stays NaN)
	T* op = reinterpret_cast<T*>(a.out_w) + b * a.bo + (int64_t)qi * a.ldo + h * a.dh;
	store_tiles<T, I::ND>(op, a.dh, a.ovec, lane, [&](int dt, int r) { return acc[dt][r] * inv; });
	if constexpr (sizeof(T) == 2) {
		if (a.rest != nullptr) {
			bf16_t* rp = a.rest + ((int64_t)b * a.Sq + qi) * a.H * a.dh + h * a.dh;
			store_tiles<T, I::ND>(rp, a.dh, a.dh % 8 == 0 ? 2 : a.dh % 4 == 0, lane, [&](int dt, int r) { return rest_of(acc[dt][r] * inv); });
		}
	}
	if (lane < 32 && a.lse != nullptr) store_lse(a, (int64_t)bh * a.Sq + qi, m, l);
}

template <typename T, int DHP, int GR, bool CAP> int launch_bias(const Args& a, hipStream_t st) {
	const int64_t blocks = placed_blocks(a.nblk, (int64_t)a.B * a.H, a.split);
	VITK_REQUIRE(blocks < (1 << 24), VITK_ERR_SHAPE);
	const dim3 grid((unsigned)blocks), block(256);
	if (a.expand != nullptr) hipLaunchKernelGGL((abias_fwd_kernel<T, DHP, GR, CAP, BIAS_TABLE>), grid, block, 0, st, a);
	else if (a.slopes != nullptr) hipLaunchKernelGGL((abias_fwd_kernel<T, DHP, GR, CAP, BIAS_SLOPE>), grid, block, 0, st, a);
	else hipLaunchKernelGGL((abias_fwd_kernel<T, DHP, GR, CAP, BIAS_NONE>), grid, block, 0, st, a);
	VITK_CHECK_LAUNCH();
	return VITK_OK;
}
template <typename T, int DHP, int GR> int launch(const Args& a, hipStream_t st) { return a.cap_l2 > 0.f ? launch_bias<T, DHP, GR, true>(a, st) : launch_bias<T, DHP, GR, false>(a, st); }
template <typename T> int fwd_dispatch(const Args& a, hipStream_t st) {
	if (a.gran == 16) {
		if (a.dh <= 32) return launch<T, 32, 16>(a, st);
		if (a.dh <= 64) return launch<T, 64, 16>(a, st);
		return launch<T, 128, 16>(a, st);
	}
	if (a.dh <= 32) return launch<T, 32, 8>(a, st);
	if (a.dh <= 64) return launch<T, 64, 8>(a, st);
	return launch<T, 128, 8>(a, st);
}

}  // namespace
