// Gradient of the bias table: dtable[bucket][h] = sum over batch and pairs with that bucket of dz = p o (dp - delta).
//
// The bucket of a pair depends on (query, key) alone when positions are shared, so a workgroup owns (head, 128 queries, some
// 64-key tiles) and walks the BATCH for each tile pair with dz summed in registers; only that sum goes through the scatter, once per pair
// instead of once per pair and image.  S and dP are formed again (two products more than a scatter inside the dQ kernel would need).
// The scatter adds into bucket sums in LDS in a fixed order: a copy per wave where they fit, else the waves take turns; the workgroups' sums
// go through the scratch buffer and are added in a fixed order by a second kernel.  No global atomics: the gradient is the same
// bits from run to run.
#pragma once

#include "attention_bias.h"

namespace {

using namespace abias;

constexpr int COPY_MAX = 1024;  // bucket counts up to which every wave has its own sums (16 KB of LDS)

template <typename T, int DHP, bool CAP>
__global__ __launch_bounds__(256, DHP * (int)sizeof(T) >= 512 ? 1 : 2) void abias_table_kernel(Args a, float* part, int chunk, int nchunk) {
	typedef Img<T, DHP> I;
	__shared__ __attribute__((aligned(16))) char Ks[I::BYTES];
	__shared__ __attribute__((aligned(16))) char Vs[I::BYTES];
	__shared__ float win[WIN];
	__shared__ __attribute__((aligned(16))) int kpos_s[TB], kseg_s[TB];
	extern __shared__ float sums[];  // [copies][n_bucket]
	int h, blk, ch;
	if (!place(a.nblk, a.H, nchunk, h, blk, ch, false)) return;
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
	const int copies = a.n_bucket <= COPY_MAX ? 4 : 1;
	for (int i = threadIdx.x; i < copies * a.n_bucket; i += 256) sums[i] = 0.f;
	float* mine = sums + (copies == 4 ? wave * a.n_bucket : 0);
	const int hk = h / a.G;
	const int q0 = blk * QB, qi = q0 + 32 * wave + (lane & 31);
	const bool in = qi < a.Sq;
	const int q1 = min(q0 + QB, a.Sq) - 1;
	const bool pos = a.kpos != nullptr;
	const bool per_image = pos && (a.bqp != 0 || a.bkp != 0);  // positions differ from image to image: scatter after each
	Own o{};
	o.slope = a.slopes != nullptr ? a.slopes[h] * LOG2E : 0.f;
	o.ex = a.expand + (int64_t)h * a.n_lookup;
	const int h4 = 4 * (lane >> 5);
	f32x16 dz[2];
#pragma unroll
	for (int i = 0; i < 2; ++i)
#pragma unroll
		for (int r = 0; r < 16; ++r) dz[i][r] = 0.f;
	__syncthreads();

	// dz into the bucket sums; dlo, dhi: range of the distances of this tile pair, k0 its first key
	auto scatter = [&](int dlo, int dhi, int k0) {
		if (dhi <= a.lookup_lo || dlo >= a.lookup_lo + a.n_lookup - 1) {  // one bucket for all pairs
			float s = 0.f;
#pragma unroll
			for (int i = 0; i < 2; ++i)
#pragma unroll
				for (int r = 0; r < 16; ++r) s += dz[i][r];
			s = wave_sum(s);
			const int bucket = a.lookup[lookup_index(a, dlo)];
			for (int turn = 0; turn < (copies == 4 ? 1 : 4); ++turn) {
				if (lane == 0 && (copies == 4 || turn == wave) && (unsigned)bucket < (unsigned)a.n_bucket) mine[bucket] += s;
				if (copies != 4) __syncthreads();
			}
		} else {
			for (int turn = 0; turn < (copies == 4 ? 1 : 4); ++turn) {
				if (copies == 4 || turn == wave) {
#pragma unroll
					for (int i = 0; i < 2; ++i)
#pragma unroll
						for (int r = 0; r < 16; ++r) {
							const int row = 32 * i + h4 + (r & 3) + 8 * (r >> 2);
							if (in && k0 + row < a.Skv) {
								const int bucket = a.lookup[lookup_index(a, (pos ? kpos_s[row] : k0 + row) - o.pos)];
								// (lanes of one instruction that meet in a bucket are added in lane order)
								if ((unsigned)bucket < (unsigned)a.n_bucket) __hip_atomic_fetch_add(mine + bucket, dz[i][r], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
							}
						}
				}
				if (copies != 4) __syncthreads();
			}
		}
#pragma unroll
		for (int i = 0; i < 2; ++i)
#pragma unroll
			for (int r = 0; r < 16; ++r) dz[i][r] = 0.f;
	};

	const int t_end = min(a.nk64, (ch + 1) * chunk);
	for (int t = ch * chunk; t < t_end; ++t) {
		const int k0 = t * TB;
		bool any = false;   // (uniform) something of this tile is in dz
		int dlo = 0, dhi = 0;
		for (int b = 0; b < a.B; ++b) {
			const int prefix = a.prefix != nullptr ? a.prefix[b] : 0;
			const int4* kr = a.kr != nullptr ? a.kr + (int64_t)b * a.nk64 : nullptr;
			const Span own = span_of(a.qr != nullptr ? a.qr + (int64_t)b * a.nq64 : nullptr, 2 * blk, a.nq64, pos, q0 + a.off, q0 + QB - 1 + a.off);
			Walk<true> walk;
			bool full = false;
			walk.start(a, t, t + 1, q0, q1, own, kr, prefix, lane);
			if (walk.act == 0) continue;
			full = (walk.ful & 1) != 0;
			any = true;
			const int* kseg = a.kseg != nullptr && !full ? a.kseg + (int64_t)b * a.Skv : nullptr;
			o.seg = a.qseg != nullptr ? (in ? a.qseg[(int64_t)b * a.Sq + qi] : -1) : 0;
			const bool own_ok = in && o.seg >= 0;
			o.lim = limit_of(a, qi, o.seg, prefix);
			int plo = k0, phi = k0 + TB - 1;
			if (pos) {
				plo = kr[t].z;
				phi = kr[t].w;
				o.pos = in ? a.qpos[b * a.bqp + qi] : own.pmin;
			} else {
				o.pos = qi + a.off;
			}
			dlo = plo - own.pmax;
			dhi = phi - own.pmin;
			const Window w = window_of(a, dlo, dhi);
			uint4 kreg[I::NIT], vreg[I::NIT];
			fetch<T, DHP>(kreg, reinterpret_cast<const T*>(a.k) + b * a.bk + hk * a.dh, a.ldk, k0, a.Skv, a.dh, a.gran, kseg);
			fetch<T, DHP>(vreg, reinterpret_cast<const T*>(a.v) + b * a.bv + hk * a.dh, a.ldv, k0, a.Skv, a.dh, a.gran, kseg);
			const T* qp = reinterpret_cast<const T*>(a.q) + b * a.bq + (int64_t)qi * a.ldq + h * a.dh;
			const T* gp = reinterpret_cast<const T*>(a.dout) + b * a.bdo + (int64_t)qi * a.lddo + h * a.dh;
			typename Tr<T>::frag qf[I::STEPS], gf[I::STEPS];
#pragma unroll
			for (int s = 0; s < I::STEPS; ++s) {
				qf[s] = own_frag<T>(qp, s, a.dh, a.gran, own_ok, lane);
				gf[s] = own_frag<T>(gp, s, a.dh, a.gran, own_ok, lane);
			}
			const int64_t row = ((int64_t)b * a.H + h) * a.Sq + qi;
			const float lse = own_ok ? a.lse[row] : INFINITY, delta = own_ok ? a.delta[row] : 0.f;
			__syncthreads();
			commit<T, DHP>(Ks, kreg);
			commit<T, DHP>(Vs, vreg);
			if (threadIdx.x < TB) {
				const int key = k0 + (int)threadIdx.x;
				if (pos) kpos_s[threadIdx.x] = key < a.Skv ? a.kpos[b * a.bkp + key] : plo;
				if (kseg != nullptr) kseg_s[threadIdx.x] = key < a.Skv ? kseg[key] : -1;
			}
			if (w.mode == WIN_LDS) {
				const int n = phi - own.pmin - w.lo + 1;
				for (int j = threadIdx.x; j < n; j += 256) win[j] = bias_at(a, o.ex, o.slope, w.lo + j);
			}
			__syncthreads();
			const TileSide ts{win, kpos_s, kseg_s, nullptr};
#pragma unroll
			for (int i = 0; i < 2; ++i) {
				f32x16 z, dp, tn;
#pragma unroll
				for (int r = 0; r < 16; ++r) z[r] = dp[r] = 0.f;
#pragma unroll
				for (int s = 0; s < I::STEPS; ++s) z = Tr<T>::mma(row_frag<T, DHP>(Ks, 32 * i, s, lane), qf[s], z);
#pragma unroll
				for (int s = 0; s < I::STEPS; ++s) dp = Tr<T>::mma(row_frag<T, DHP>(Vs, 32 * i, s, lane), gf[s], dp);
				modify<true, CAP, BIAS_TABLE>(z, tn, a, w, ts, o, pos, k0, 32 * i, lane);
				if (!full) hide<true>(z, a, ts, o, k0, 32 * i, lane);
#pragma unroll
				for (int r = 0; r < 16; ++r) dz[i][r] = fmaf(__builtin_amdgcn_exp2f(z[r] - lse), dp[r] - delta, dz[i][r]);
			}
			if (per_image) scatter(dlo, dhi, k0);
		}
		if (any && !per_image) scatter(dlo, dhi, k0);
	}
	__syncthreads();
	float* po = part + (((int64_t)h * a.nblk + blk) * nchunk + ch) * a.n_bucket;
	for (int i = threadIdx.x; i < a.n_bucket; i += 256) {
		float s = sums[i];
		for (int c = 1; c < copies; ++c) s += sums[c * a.n_bucket + i];
		po[i] = s;
	}
}

template <typename T, int DHP> int launch(const Args& a, float* part, int chunk, int nchunk, hipStream_t st) {
	const int64_t blocks = vitk_cdiv(a.H, 8) * 8 * a.nblk * nchunk;
	VITK_REQUIRE(blocks < (1 << 24), VITK_ERR_SHAPE);
	const size_t lds = sizeof(float) * a.n_bucket * (a.n_bucket <= COPY_MAX ? 4 : 1);
	if (a.cap_l2 > 0.f) hipLaunchKernelGGL((abias_table_kernel<T, DHP, true>), dim3((unsigned)blocks), dim3(256), lds, st, a, part, chunk, nchunk);
	else hipLaunchKernelGGL((abias_table_kernel<T, DHP, false>), dim3((unsigned)blocks), dim3(256), lds, st, a, part, chunk, nchunk);
	VITK_CHECK_LAUNCH();
	return VITK_OK;
}
template <typename T> int table_dispatch(const Args& a, float* part, int chunk, int nchunk, hipStream_t st) {
	if (a.dh <= 32) return launch<T, 32>(a, part, chunk, nchunk, st);
	if (a.dh <= 64) return launch<T, 64>(a, part, chunk, nchunk, st);
	return launch<T, 128>(a, part, chunk, nchunk, st);
}

}  // namespace

