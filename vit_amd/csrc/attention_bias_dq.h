// Backward of the biased / capped / masked attention: dQ kernel and dK/dV kernel (mathematics, tiles, orientation: attention_bias.h).
//
// Both form the scores again from q, k and the saved normaliser: p = exp2(z - lse).  Two kernels, seven products instead of the five
// of a single pass, so that every gradient is summed by one workgroup in a fixed order (no float atomics on dQ).
//   dQ (own rows = queries):   S^T = K Q^T, dP^T = V dO^T, dQ^T[d][q] += K^T dS^T        (K columns by the transposing LDS read)
//   dK/dV (own rows = keys):   S = Q K^T, dP = dO V^T, dV^T[d][k] += dO^T P, dK^T[d][k] += Q^T dS, over all query heads of the key head
// delta = rowsum(dout o out).  For the gradient of a bias table that is not exact enough: a bucket sums dz over many keys of a row, where
// sum_j p (dp - delta) cancels, and the error that out's rounding to bfloat16 leaves in delta (2^-9 of it; with what the forward kept of it 2^-14, and what the
// rounding of the weights in out makes) would be most of what is left.
// SUMS: the dQ kernel therefore also adds up what is left, r = sum_j dz, and sum_j p of every row, and leaves delta + r / sum p, which makes the
// row's dz sum to zero, for the kernels behind it (two additions a score instead of a pass of two products for delta alone).
#pragma once

#include "attention_bias.h"

namespace {

using namespace abias;

// Waves of a SIMD, by the bytes of a row in LDS: three at 64, although a table then spills 17 registers (16 x 32 heads x 784^2 x 12: 268 us, with two 296); two at
// 128, and at 256 without a table although that spills 21 to 66 (2 x 16 heads x 2048^2 x 128, capped: 206 us, with one 246; uncapped, 8 x 6 x 1024^2: 98 and
// 125); else one.
template <typename T, int DHP, int GR, bool CAP, int BIAS, bool SUMS>
__global__ __launch_bounds__(256, DHP * (int)sizeof(T) >= 256 + 256 * (BIAS != BIAS_TABLE) ? 1 : (DHP * (int)sizeof(T) <= 64 ? 3 : 2)) void abias_dq_kernel(Args a) {
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
	const bool pos = BIAS != BIAS_NONE && a.kpos != nullptr;
	const int prefix = a.prefix != nullptr ? a.prefix[b] : 0;
	const int* kseg = a.kseg != nullptr ? a.kseg + (int64_t)b * a.Skv : nullptr;
	const int* kpos = pos ? a.kpos + b * a.bkp : nullptr;
	const int4* kr = a.kr != nullptr ? a.kr + (int64_t)b * a.nk64 : nullptr;
	const int q1 = min(q0 + QB, a.Sq) - 1;
	const Span own = span_of(a.qr != nullptr ? a.qr + (int64_t)b * a.nq64 : nullptr, 2 * blk, a.nq64, pos, q0 + a.off, q0 + QB - 1 + a.off);
	Own o{};
	o.seg = a.qseg != nullptr ? (qi < a.Sq ? a.qseg[(int64_t)b * a.Sq + qi] : -1) : 0;
	const bool own_ok = qi < a.Sq && o.seg >= 0;  // (rows of a negative segment are not read: they see no key)
	o.lim = limit_of(a, qi, o.seg, prefix);
	if constexpr (BIAS != BIAS_NONE) {
		o.pos = pos ? (qi < a.Sq ? a.qpos[b * a.bqp + qi] : own.pmin) : qi + a.off;
		o.slope = a.slopes != nullptr ? a.slopes[h] * LOG2E : 0.f;
		o.ex = BIAS == BIAS_TABLE ? a.expand + (int64_t)h * a.n_lookup : nullptr;
	}
	const T* kb = reinterpret_cast<const T*>(a.k) + b * a.bk + hk * a.dh;
	const T* vb = reinterpret_cast<const T*>(a.v) + b * a.bv + hk * a.dh;
	const Rows qx = rows_of<T>(reinterpret_cast<const T*>(a.q) + b * a.bq + h * a.dh, a.ldq, q0, a.Sq, QB, a.dh);
	const Rows gx = rows_of<T>(reinterpret_cast<const T*>(a.dout) + b * a.bdo + h * a.dh, a.lddo, q0, a.Sq, QB, a.dh);
	const Rows ox = rows_of<T>(reinterpret_cast<const T*>(a.out) + b * a.bo + h * a.dh, a.ldo, q0, a.Sq, QB, a.dh);
	typename Tr<T>::frag qf[I::STEPS], gf[I::STEPS];
#pragma unroll
	for (int s = 0; s < I::STEPS; ++s) {
		qf[s] = own_frag<T, GR>(qx, qi - q0, a.ldq, s, a.dh, a.gran, own_ok, lane);
		gf[s] = own_frag<T, GR>(gx, qi - q0, a.lddo, s, a.dh, a.gran, own_ok, lane);
	}
	// delta from the diagonal of the product out dout^T, summed as the products of dout and a value row are: of a row that sees one key out is that
	// key's value, and dp - delta is then the 0 that it should be, not a rounding error.  With bfloat16 out's rounding (2^-9 of it) would be most of the
	// error of dq and dk where a weight is near one and dp - delta small (documents of 3 tokens, capped: 0.9 % of dq), so what it took counts too
	float delta = 0.f;
	{
		f32x16 od;
#pragma unroll
		for (int r = 0; r < 16; ++r) od[r] = 0.f;
#pragma unroll
		for (int s = 0; s < I::STEPS; ++s) od = Tr<T>::mma(own_frag<T, GR>(ox, qi - q0, a.ldo, s, a.dh, a.gran, own_ok, lane), gf[s], od);
		if constexpr (sizeof(T) == 2) {  // (no rest: rows that read as zero)
			const Rows rx = rows_of<T>(a.rest + (int64_t)b * a.Sq * a.H * a.dh + h * a.dh, a.H * a.dh, q0, a.rest != nullptr ? a.Sq : 0, QB, a.dh);
#pragma unroll
			for (int s = 0; s < I::STEPS; ++s) od = Tr<T>::mma(own_frag<T, GR>(rx, qi - q0, a.H * a.dh, s, a.dh, a.gran, own_ok, lane), gf[s], od);
		}
#pragma unroll
		for (int r = 0; r < 16; ++r) delta = 4 * (lane >> 5) + (r & 3) + 8 * (r >> 2) == (lane & 31) ? od[r] : delta;
		delta = pair_sum(delta);
	}
	if (part == 0 && qi < a.Sq && lane < 32 && (!SUMS || a.split > 1)) a.delta[(int64_t)bh * a.Sq + qi] = delta;
	float poison = 0.f, rest = 0.f, total = 0.f;  // SUMS: sum of dz, sum of p
	const float lse = own_ok ? a.lse[(int64_t)bh * a.Sq + qi] : INFINITY;
	const float lse_rest = sizeof(T) == 4 && own_ok && a.lse_rest != nullptr ? a.lse_rest[(int64_t)bh * a.Sq + qi] : 0.f;

	f32x16 acc[I::ND];
#pragma unroll
	for (int dt = 0; dt < I::ND; ++dt)
#pragma unroll
		for (int r = 0; r < 16; ++r) acc[dt][r] = 0.f;

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
		__syncthreads();
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
		if (q0 + 32 * wave >= a.Sq) continue;
		if (special) poison += sees_marked<true>(a, ts, o, k0, bad_s, lane);
#pragma unroll
		for (int i = 0; i < 2; ++i) {
			const int lv = anew(lane);
			f32x16 z, dp, tn;
#pragma unroll
			for (int r = 0; r < 16; ++r) z[r] = dp[r] = 0.f;
#pragma unroll
			for (int s = 0; s < I::STEPS; ++s) z = Tr<T>::mma(row_frag<T, DHP>(Ks, 32 * i, s, lane), qf[s], z);
#pragma unroll
			for (int s = 0; s < I::STEPS; ++s) dp = Tr<T>::mma(row_frag<T, DHP>(Vs, 32 * i, s, lane), gf[s], dp);
			modify<true, CAP, BIAS>(z, tn, a, w, ts, o, pos, k0, 32 * i, lv);
			if (!full) hide<true>(z, a, ts, o, k0, 32 * i, lv);
#pragma unroll
			for (int r = 0; r < 16; ++r) {
				const float p = weight_of<T, CAP, BIAS>(a, z[r], lse, lse_rest);
				float ds = p * (dp[r] - delta);
				if constexpr (SUMS) {
					if (!full) ds = p == 0.f ? 0.f : ds;
					total += p;
					rest += ds;
				}
				if constexpr (CAP) ds *= fmaf(-tn[r], tn[r], 1.f);
				if constexpr (CAP || !SUMS) {
					if (!full) ds = p == 0.f ? 0.f : ds;  // (a hidden pair: dp and the tanh may be an infinity or a NaN)
				}
				z[r] = ds;
			}
			outer<T, DHP>(acc, Ks, 32 * i, z, lane);
		}
	}
	poison = pair_sum(poison);
	if (qi >= a.Sq) return;
	const int64_t rows = (int64_t)a.B * a.H * a.Sq, row = (int64_t)bh * a.Sq + qi;
	if constexpr (SUMS) {
		rest = pair_sum(rest);
		total = pair_sum(total);
		if (lane < 32) {
			if (a.split > 1) {
				a.row_part[((int64_t)part * rows + row) * 2] = rest;
				a.row_part[((int64_t)part * rows + row) * 2 + 1] = total;
			} else {
				a.delta[row] = total == 0.f ? 0.f : delta + rest / total;
			}
		}
	}
	const auto value = [&](int dt, int r) { return fmaf(acc[dt][r], a.scale, poison); };
	if (a.split > 1) store_tiles<float, I::ND>(a.part + ((int64_t)part * rows + row) * a.dh, a.dh, a.dh % 4 == 0, lane, value);
	else store_tiles<T, I::ND>(reinterpret_cast<T*>(a.dq) + b * a.bdq + (int64_t)qi * a.lddq + h * a.dh, a.dh, a.ovec, lane, value);
}

template <typename T, int DHP, int GR, bool CAP> int launch_bias(const Args& a, bool sums, hipStream_t st) {
	const int64_t blocks = placed_blocks(a.nblk, (int64_t)a.B * a.H, a.split);
	VITK_REQUIRE(blocks < (1 << 24), VITK_ERR_SHAPE);
	const dim3 grid((unsigned)blocks), block(256);
	if (sums) hipLaunchKernelGGL((abias_dq_kernel<T, DHP, GR, CAP, BIAS_TABLE, true>), grid, block, 0, st, a);
	else if (a.expand != nullptr) hipLaunchKernelGGL((abias_dq_kernel<T, DHP, GR, CAP, BIAS_TABLE, false>), grid, block, 0, st, a);
	else if (a.slopes != nullptr) hipLaunchKernelGGL((abias_dq_kernel<T, DHP, GR, CAP, BIAS_SLOPE, false>), grid, block, 0, st, a);
	else hipLaunchKernelGGL((abias_dq_kernel<T, DHP, GR, CAP, BIAS_NONE, false>), grid, block, 0, st, a);
	VITK_CHECK_LAUNCH();
	return VITK_OK;
}
template <typename T, int DHP, int GR> int launch(const Args& a, bool sums, hipStream_t st) { return a.cap_l2 > 0.f ? launch_bias<T, DHP, GR, true>(a, sums, st) : launch_bias<T, DHP, GR, false>(a, sums, st); }
template <typename T> int dq_dispatch(const Args& a, bool sums, hipStream_t st) {
	if (a.gran == 16) {
		if (a.dh <= 32) return launch<T, 32, 16>(a, sums, st);
		if (a.dh <= 64) return launch<T, 64, 16>(a, sums, st);
		return launch<T, 128, 16>(a, sums, st);
	}
	if (a.dh <= 32) return launch<T, 32, 8>(a, sums, st);
	if (a.dh <= 64) return launch<T, 64, 8>(a, sums, st);
	return launch<T, 128, 8>(a, sums, st);
}

}  // namespace
