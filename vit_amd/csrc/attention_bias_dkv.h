// dK/dV kernel of the biased / capped / masked attention: the other half of the backward (see attention_bias_dq.h).
#pragma once

#include "attention_bias.h"

namespace {

using namespace abias;

// Waves of a SIMD, by the bytes of a row in LDS: three at 64, although up to 25 registers spill (16 x 32 heads x 784^2 x 12 with a table: 342 us, with two 378; 8 x
// 12 x 1024^2 x 32 sloped: 71 and 97); two at 128; one from 256 on, where both accumulators and both own operands take up to 512 registers.
template <typename T, int DHP, int GR, bool CAP, int BIAS>
__global__ __launch_bounds__(256, DHP * (int)sizeof(T) >= 256 ? 1 : (DHP * (int)sizeof(T) <= 64 ? 3 : 2)) void abias_dkv_kernel(Args a) {
	typedef Img<T, DHP> I;
	__shared__ __attribute__((aligned(16))) char Qs[I::BYTES];
	__shared__ __attribute__((aligned(16))) char Gs[I::BYTES];
	__shared__ float win[BIAS == BIAS_TABLE ? WIN : 1];
	__shared__ __attribute__((aligned(16))) int qpos_s[TB], qseg_s[TB], qlim_s[TB], bad_s[TB + 1];
	__shared__ __attribute__((aligned(16))) float lse_s[TB], delta_s[TB], rest_s[sizeof(T) == 4 ? TB : 4];
	int bk, blk, part;
	if (!place(a.nblk, a.B * a.Hkv, a.split, bk, blk, part, false)) return;
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
	const int b = bk / a.Hkv, hk = bk - b * a.Hkv;
	const int k0 = blk * QB, ki = k0 + 32 * wave + (lane & 31);
	const bool pos = BIAS != BIAS_NONE && a.kpos != nullptr;
	const int prefix = a.prefix != nullptr ? a.prefix[b] : 0;
	const int* qseg = a.qseg != nullptr ? a.qseg + (int64_t)b * a.Sq : nullptr;
	const int* qpos = pos ? a.qpos + b * a.bqp : nullptr;
	const int4* qr = a.qr != nullptr ? a.qr + (int64_t)b * a.nq64 : nullptr;
	const int k1 = min(k0 + QB, a.Skv) - 1;
	const Span own = span_of(a.kr != nullptr ? a.kr + (int64_t)b * a.nk64 : nullptr, 2 * blk, a.nk64, pos, k0, k0 + QB - 1);
	Own o{};
	o.idx = ki;
	o.seg = a.kseg != nullptr ? (ki < a.Skv ? a.kseg[(int64_t)b * a.Skv + ki] : -1) : 0;
	const bool own_ok = ki < a.Skv && o.seg >= 0;
	if constexpr (BIAS != BIAS_NONE) o.pos = pos ? (ki < a.Skv ? a.kpos[b * a.bkp + ki] : own.pmin) : ki;
	const Rows kx = rows_of<T>(reinterpret_cast<const T*>(a.k) + b * a.bk + hk * a.dh, a.ldk, k0, a.Skv, QB, a.dh);
	const Rows vx = rows_of<T>(reinterpret_cast<const T*>(a.v) + b * a.bv + hk * a.dh, a.ldv, k0, a.Skv, QB, a.dh);
	typename Tr<T>::frag kf[I::STEPS], vf[I::STEPS];
#pragma unroll
	for (int s = 0; s < I::STEPS; ++s) {
		kf[s] = own_frag<T, GR>(kx, ki - k0, a.ldk, s, a.dh, a.gran, own_ok, lane);
		vf[s] = own_frag<T, GR>(vx, ki - k0, a.ldv, s, a.dh, a.gran, own_ok, lane);
	}
	f32x16 dk[I::ND], dv[I::ND];
#pragma unroll
	for (int dt = 0; dt < I::ND; ++dt)
#pragma unroll
		for (int r = 0; r < 16; ++r) dk[dt][r] = dv[dt][r] = 0.f;

	Stage<T, DHP, GR> qst, gst;
	qst.init(a.ldq, a.dh);
	gst.init(a.lddo, a.dh);
	float wreg[WIN / 256];
	int preg = 0, sreg = 0;
	float lreg = 0.f, dreg = 0.f, rreg = 0.f;
	Window wn{0, WIN_ONE};
	bool full_n = false;
	float poison = 0.f;
	int h = hk * a.G;  // the query head that is walked
	float slope_n = 0.f;
	const float* ex_n = nullptr;
	auto fetch_tile = [&](int t) {
		const int q0 = t * TB;
		const int* sg = full_n ? nullptr : qseg;
		const int* sgt = sg != nullptr ? sg + q0 : nullptr;
		const uint32_t hid = sgt != nullptr ? Stage<T, DHP, GR>::hidden(sgt, a.Sq - q0) : 0u;
		qst.fetch(rows_of<T>(reinterpret_cast<const T*>(a.q) + b * a.bq + h * a.dh, a.ldq, q0, a.Sq, TB, a.dh), a.dh, a.gran, hid);
		gst.fetch(rows_of<T>(reinterpret_cast<const T*>(a.dout) + b * a.bdo + h * a.dh, a.lddo, q0, a.Sq, TB, a.dh), a.dh, a.gran, hid);
		int plo = q0 + a.off, phi = q0 + TB - 1 + a.off;
		if (pos) {
			const i32x4 r = range_at(qr, t);
			plo = r.z;
			phi = r.w;
		}
		if (threadIdx.x < TB) {
			const int qi = q0 + (int)threadIdx.x;
			const bool ok = qi < a.Sq;
			const int64_t row = ((int64_t)b * a.H + h) * a.Sq + qi;
			lreg = ok ? a.lse[row] : INFINITY;
			dreg = ok ? a.delta[row] : 0.f;
			if constexpr (sizeof(T) == 4) rreg = ok && a.lse_rest != nullptr ? a.lse_rest[row] : 0.f;
			if (pos) preg = ok ? qpos[qi] : plo;
			sreg = qseg != nullptr ? (ok ? qseg[qi] : -1) : 0;
		}
		if constexpr (BIAS != BIAS_NONE) {
			slope_n = a.slopes != nullptr ? uniform_load(a.slopes + h) * LOG2E : 0.f;
			if constexpr (BIAS == BIAS_TABLE) {
				ex_n = a.expand + (int64_t)h * a.n_lookup;
				wn = window_of(a, own.pmin - phi, own.pmax - plo);
				if (wn.mode == WIN_LDS) {
					const int n = own.pmax - plo - wn.lo + 1;
#pragma unroll
					for (int i = 0; i < WIN / 256; ++i) {
						const int j = (int)threadIdx.x + 256 * i;
						if (j < n) wreg[i] = ex_n[lookup_index(a, wn.lo + j)];
					}
				}
			}
		}
	};

	Walk<false> walk;
	const int t_beg = part * a.per_split, t_end = (int)min((int64_t)a.nq64, (int64_t)(part + 1) * a.per_split);
	auto advance = [&]() -> int {
		int t = walk.next(a, k0, k1, own, qr, prefix, lane, full_n);
		while (t < 0 && h + 1 < (hk + 1) * a.G) {
			++h;
			walk.start(a, t_beg, t_end, k0, k1, own, qr, prefix, lane);
			t = walk.next(a, k0, k1, own, qr, prefix, lane, full_n);
		}
		return t;
	};
	walk.start(a, t_beg, t_end, k0, k1, own, qr, prefix, lane);
	if (threadIdx.x == 0) bad_s[TB] = -1;
	int t = advance();
	if (t >= 0) fetch_tile(t);
	const TileSide ts{win, qpos_s, qseg_s, qlim_s};
	while (t >= 0) {
		const int q0 = t * TB;
		const Window w = wn;
		const bool full = full_n;
		o.slope = slope_n;
		o.ex = ex_n;
		__syncthreads();
		qst.commit(Qs);
		gst.commit(Gs);
		if (threadIdx.x < TB) {
			qpos_s[threadIdx.x] = BIAS == BIAS_TABLE ? preg * 4 : preg;
			qseg_s[threadIdx.x] = sreg;
			qlim_s[threadIdx.x] = limit_of(a, q0 + (int)threadIdx.x, sreg, prefix);
			lse_s[threadIdx.x] = lreg;
			delta_s[threadIdx.x] = dreg;
			if constexpr (sizeof(T) == 4) rest_s[threadIdx.x] = rreg;
		}
		if constexpr (BIAS == BIAS_TABLE) {
			if (w.mode == WIN_LDS) {
#pragma unroll
				for (int i = 0; i < WIN / 256; ++i) win[threadIdx.x + 256 * i] = fmaf(-o.slope, fabsf((float)(w.lo + (int)threadIdx.x + 256 * i)), wreg[i]);
			}
		}
		const bool special = settle_tile(full, t, qst, Qs, gst, Gs, bad_s);
		t = advance();
		if (t >= 0) fetch_tile(t);
		if (k0 + 32 * wave >= a.Skv) continue;
		if (special) poison += sees_marked<false>(a, ts, o, 0, bad_s, lane);
		const int h4 = 4 * (lane >> 5);
#pragma unroll
		for (int i = 0; i < 2; ++i) {
			const int lv = anew(lane);
			f32x16 z, dp, tn;
#pragma unroll
			for (int r = 0; r < 16; ++r) z[r] = dp[r] = 0.f;
#pragma unroll
			for (int s = 0; s < I::STEPS; ++s) z = Tr<T>::mma(row_frag<T, DHP>(Qs, 32 * i, s, lane), kf[s], z);
#pragma unroll
			for (int s = 0; s < I::STEPS; ++s) dp = Tr<T>::mma(row_frag<T, DHP>(Gs, 32 * i, s, lane), vf[s], dp);
			modify<false, CAP, BIAS>(z, tn, a, w, ts, o, pos, q0 + a.off, 32 * i, lv);
			if (!full) hide<false>(z, a, ts, o, 0, 32 * i, lv);
#pragma unroll
			for (int g = 0; g < 4; ++g) {
				const f32x4 ls = *reinterpret_cast<const f32x4*>(lse_s + 32 * i + h4 + 8 * g), de = *reinterpret_cast<const f32x4*>(delta_s + 32 * i + h4 + 8 * g);
				f32x4 lr = {0.f, 0.f, 0.f, 0.f};
				if constexpr (sizeof(T) == 4) lr = *reinterpret_cast<const f32x4*>(rest_s + 32 * i + h4 + 8 * g);
#pragma unroll
				for (int e = 0; e < 4; ++e) {
					const int r = 4 * g + e;
					float p = weight_of<T, CAP, BIAS>(a, z[r], ls[e], lr[e]);
					if (!full) p = z[r] == -INFINITY ? 0.f : p;  // (a hidden query's normaliser may be a NaN)
					float ds = p * (dp[r] - de[e]);
					if constexpr (CAP) ds *= fmaf(-tn[r], tn[r], 1.f);
					if (!full) ds = p == 0.f ? 0.f : ds;  // (a hidden pair: dp and the tanh may be an infinity or a NaN)
					z[r] = p;
					dp[r] = ds;
				}
			}
			outer<T, DHP>(dv, Gs, 32 * i, z, lane);
			outer<T, DHP>(dk, Qs, 32 * i, dp, lane);
		}
	}
	poison = pair_sum(poison);
	if (ki >= a.Skv) return;
	const int64_t rows = (int64_t)a.B * a.Hkv * a.Skv, row = (int64_t)bk * a.Skv + ki;
	const auto kvalue = [&](int dt, int r) { return own_ok ? fmaf(dk[dt][r], a.scale, poison) : 0.f; };
	const auto vvalue = [&](int dt, int r) { return own_ok ? dv[dt][r] + poison : 0.f; };
	if (a.split > 1) {
		float* pk = a.part + ((int64_t)part * rows + row) * a.dh;
		store_tiles<float, I::ND>(pk, a.dh, a.dh % 4 == 0, lane, kvalue);
		store_tiles<float, I::ND>(pk + (int64_t)a.split * rows * a.dh, a.dh, a.dh % 4 == 0, lane, vvalue);
	} else {
		store_tiles<T, I::ND>(reinterpret_cast<T*>(a.dk) + b * a.bdk + (int64_t)ki * a.lddk + hk * a.dh, a.dh, a.ovec, lane, kvalue);
		store_tiles<T, I::ND>(reinterpret_cast<T*>(a.dv) + b * a.bdv + (int64_t)ki * a.lddv + hk * a.dh, a.dh, a.ovec, lane, vvalue);
	}
}

template <typename T, int DHP, int GR, bool CAP> int launch_bias(const Args& a, hipStream_t st) {
	const int64_t blocks = placed_blocks(a.nblk, (int64_t)a.B * a.Hkv, a.split);
	VITK_REQUIRE(blocks < (1 << 24), VITK_ERR_SHAPE);
	const dim3 grid((unsigned)blocks), block(256);
	if (a.expand != nullptr) hipLaunchKernelGGL((abias_dkv_kernel<T, DHP, GR, CAP, BIAS_TABLE>), grid, block, 0, st, a);
	else if (a.slopes != nullptr) hipLaunchKernelGGL((abias_dkv_kernel<T, DHP, GR, CAP, BIAS_SLOPE>), grid, block, 0, st, a);
	else hipLaunchKernelGGL((abias_dkv_kernel<T, DHP, GR, CAP, BIAS_NONE>), grid, block, 0, st, a);
	VITK_CHECK_LAUNCH();
	return VITK_OK;
}
template <typename T, int DHP, int GR> int launch(const Args& a, hipStream_t st) { return a.cap_l2 > 0.f ? launch_bias<T, DHP, GR, true>(a, st) : launch_bias<T, DHP, GR, false>(a, st); }
template <typename T> int dkv_dispatch(const Args& a, hipStream_t st) {
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
