// Gradient of the bias table: dtable[bucket][h] = sum over batch and pairs with that bucket of dz = p o (dp - delta).
//
// Scattering dz costs far more than forming it: an LDS float atomic is 193 clocks a wave instruction (measured, whatever the
// addresses), 64 scores; scattering inside the dQ kernel made that kernel seven times slower (16 x 32 heads x 784^2: 338 -> 2417 us).
// The bucket of a pair depends on (query, key) alone where positions are shared, so this kernel owns (head, 128 queries, 64 keys) and walks the
// BATCH for each such tile pair with dz summed in registers: S and dP are formed again, and one scatter serves all images.
// The scatter itself goes by DISTANCE: for one key the queries of a wave have distinct positions, so the 32 lanes of a half wave
// add to distinct slots of a window of distances by an ordinary load, add and store, the two halves (keys 4 apart) in windows of their own, one key after
// another (wave_step);
// then one wave adds the 8 windows up and into the bucket sums, 64 distances at a time.  Where positions repeat within a wave, or a
// window would be wider than 1024 distances, the waves take turns with LDS atomics.  Pairs beyond one end of the lookup share one bucket
// and are summed in registers.  Every order is fixed: the gradient is the same bits from run to run.
#pragma once

#include "attention_bias.h"

namespace {

using namespace abias;

// LDS accesses of the wave's lanes in front of it come before those behind it.  The hardware works a wave's LDS accesses off in order, so it costs no
// instruction; without it the compiler, which looks at one lane, may take a lane's later load ahead of another lane's store to the same place.
__device__ __forceinline__ void wave_step() {
	__builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
	__builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ int bucket_at(const Args& a, int d) {  // n_bucket: none
	const int b = a.lookup[lookup_index(a, d)];
	return (unsigned)b < (unsigned)a.n_bucket ? b : a.n_bucket;
}

template <typename T, int DHP, int GR, bool CAP>
__global__ __launch_bounds__(256, DHP * (int)sizeof(T) >= 256 ? 1 : 2) void abias_table_kernel(Args a, TablePlan tp, float* out) {
	typedef Img<T, DHP> I;
	// the tiles of an image and the windows of the scatter take turns in one piece of LDS
	constexpr int LDS_TILES = 2 * I::BYTES, LDS_WIN = 8 * WIN * (int)sizeof(float);
	__shared__ __attribute__((aligned(16))) char smem[LDS_TILES > LDS_WIN ? LDS_TILES : LDS_WIN];
	char *Ks = smem, *Vs = smem + I::BYTES;
	__shared__ __attribute__((aligned(16))) int kpos_s[TB], kseg_s[TB];
	__shared__ float win[WIN];
	extern __shared__ float sums[];  // [n_bucket + 1]
	int h, blk, part;
	if (!place(a.nblk, a.H, tp.nchunk * tp.nimages, h, blk, part, false)) return;
	const int ch = part / tp.nimages, im = part - ch * tp.nimages;
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, h4 = 4 * half;
	for (int i = threadIdx.x; i <= a.n_bucket; i += 256) sums[i] = 0.f;
	const int hk = h / a.G;
	const int q0 = blk * QB, qi = q0 + 32 * wave + (lane & 31);
	const bool in = qi < a.Sq;
	const int q1 = min(q0 + QB, a.Sq) - 1;
	const bool pos = a.kpos != nullptr;
	const bool per_image = pos && (a.bqp != 0 || a.bkp != 0);  // positions differ from image to image: scatter after each
	const int b0 = im * tp.images, b1 = min(a.B, b0 + tp.images);
	Own o{};
	o.slope = a.slopes != nullptr ? a.slopes[h] * LOG2E : 0.f;
	o.ex = a.expand + (int64_t)h * a.n_lookup;
	f32x16 dz[2];
#pragma unroll
	for (int i = 0; i < 2; ++i)
#pragma unroll
		for (int r = 0; r < 16; ++r) dz[i][r] = 0.f;
	__syncthreads();

	// dz into the bucket sums; dlo .. dhi: the distances of this tile pair, k0 its first key
	auto scatter = [&](int dlo, int dhi, int k0) {
		if (dhi <= a.lookup_lo || dlo >= a.lookup_lo + a.n_lookup - 1) {  // one bucket for all pairs
			float s = 0.f;
#pragma unroll
			for (int i = 0; i < 2; ++i)
#pragma unroll
				for (int r = 0; r < 16; ++r) s += dz[i][r];
			s = wave_sum(s);
			const int bucket = bucket_at(a, dlo);
			for (int turn = 0; turn < 4; ++turn) {
				if (lane == 0 && turn == wave) sums[bucket] += s;
				__syncthreads();
			}
		} else {
			bool twice = false;  // two queries of the wave at one position
#pragma unroll 1
			for (int s = 1; s < 32; ++s) {
				const int other = __shfl(o.pos, (lane & 32) | ((lane + s) & 31), 64), row = (lane + s) & 31;
				twice |= in && q0 + 32 * wave + row < a.Sq && other == o.pos;
			}
			const bool wide = (unsigned)dhi - (unsigned)dlo >= (unsigned)WIN;
			const int n = dhi - dlo + 1;
			if (!__syncthreads_or(twice || wide)) {
				float* all = reinterpret_cast<float*>(smem);
				for (int w = 0; w < 8; ++w)
					for (int i = threadIdx.x; i < n; i += 256) all[w * WIN + i] = 0.f;
				__syncthreads();
				float* mine = all + (2 * wave + half) * WIN;
#pragma unroll
				for (int i = 0; i < 2; ++i)
#pragma unroll
					for (int r = 0; r < 16; ++r) {
						const int row = 32 * i + h4 + (r & 3) + 8 * (r >> 2);
						if (in && k0 + row < a.Skv) mine[(pos ? kpos_s[row] >> 2 : k0 + row) - o.pos - dlo] += dz[i][r];
						wave_step();  // (the slot of this lane's next key was another lane's just now)
					}
				__syncthreads();
				if (wave == 0) {
					for (int i = lane; i < n; i += 64) {
						float s = all[i];
#pragma unroll
						for (int w = 1; w < 8; ++w) s += all[w * WIN + i];
						// (lanes that meet in a bucket are added in lane order)
						__hip_atomic_fetch_add(sums + bucket_at(a, dlo + i), s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
					}
				}
			} else {
				float* mine = reinterpret_cast<float*>(smem) + wave * 2048 + lane;  // (through LDS, so that the loop below need not be unrolled)
#pragma unroll
				for (int i = 0; i < 2; ++i)
#pragma unroll
					for (int r = 0; r < 16; ++r) mine[64 * (16 * i + r)] = dz[i][r];
				for (int turn = 0; turn < 4; ++turn) {
					if (turn == wave) {
#pragma unroll 1
						for (int e = 0; e < 32; ++e) {
							const int row = 32 * (e >> 4) + h4 + (e & 3) + 8 * ((e & 15) >> 2);
							if (in && k0 + row < a.Skv) __hip_atomic_fetch_add(sums + bucket_at(a, (pos ? kpos_s[row] >> 2 : k0 + row) - o.pos), mine[64 * e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
						}
					}
					__syncthreads();
				}
			}
		}
#pragma unroll
		for (int i = 0; i < 2; ++i)
#pragma unroll
			for (int r = 0; r < 16; ++r) dz[i][r] = 0.f;
	};

	// The items (tile, image) in order, the next one's rows on their way while one is worked on
	Stage<T, DHP, GR> kst, vst;
	kst.init(a.ldk, a.dh);
	vst.init(a.ldv, a.dh);
	const int t_end = min(a.nk64, (ch + 1) * tp.chunk);
	int tn_ = ch * tp.chunk, bn = b0 - 1;  // the next item
	bool full_n = false;
	typename Tr<T>::frag qn[I::STEPS], gn[I::STEPS];
	float lse_n = 0.f, delta_n = 0.f, rest_n = 0.f;
	int seg_n = 0, lim_n = 0, ksg_n = 0;
	auto advance = [&]() -> bool {
		for (;;) {
			if (++bn == b1) {
				bn = b0;
				++tn_;
			}
			if (tn_ >= t_end) return false;
			// (the walk asks for segments alone: without them no range is read, a wait for every item less)
			const Span own = span_of(a.kseg != nullptr ? a.qr + (int64_t)bn * a.nq64 : nullptr, 2 * blk, a.nq64, false, 0, 0);
			Walk<true> walk;
			walk.start(a, tn_, tn_ + 1, q0, q1, own, a.kr != nullptr ? a.kr + (int64_t)bn * a.nk64 : nullptr, a.prefix != nullptr ? uniform_load(a.prefix + bn) : 0, lane);
			full_n = (walk.ful & 1) != 0;
			if (walk.act != 0) return true;
		}
	};
	auto fetch_item = [&]() {
		const int k0 = tn_ * TB, b = bn;
		const int* sgt = a.kseg != nullptr && !full_n ? a.kseg + (int64_t)b * a.Skv + k0 : nullptr;
		seg_n = a.qseg != nullptr ? (in ? a.qseg[(int64_t)b * a.Sq + qi] : -1) : 0;  // (in front of the rows: used at once)
		lim_n = limit_of(a, qi, seg_n, a.prefix != nullptr ? uniform_load(a.prefix + b) : 0);
		const bool own_ok = in && seg_n >= 0;
		const uint32_t hid = sgt != nullptr ? Stage<T, DHP, GR>::hidden(sgt, a.Skv - k0) : 0u;
		kst.fetch(rows_of<T>(reinterpret_cast<const T*>(a.k) + b * a.bk + hk * a.dh, a.ldk, k0, a.Skv, TB, a.dh), a.dh, a.gran, hid);
		vst.fetch(rows_of<T>(reinterpret_cast<const T*>(a.v) + b * a.bv + hk * a.dh, a.ldv, k0, a.Skv, TB, a.dh), a.dh, a.gran, hid);
		const Rows qx = rows_of<T>(reinterpret_cast<const T*>(a.q) + b * a.bq + h * a.dh, a.ldq, q0, a.Sq, QB, a.dh);
		const Rows gx = rows_of<T>(reinterpret_cast<const T*>(a.dout) + b * a.bdo + h * a.dh, a.lddo, q0, a.Sq, QB, a.dh);
#pragma unroll
		for (int s = 0; s < I::STEPS; ++s) {
			qn[s] = own_frag<T, GR>(qx, qi - q0, a.ldq, s, a.dh, a.gran, own_ok, lane);
			gn[s] = own_frag<T, GR>(gx, qi - q0, a.lddo, s, a.dh, a.gran, own_ok, lane);
		}
		const int64_t row = ((int64_t)b * a.H + h) * a.Sq + qi;
		lse_n = own_ok ? a.lse[row] : INFINITY;
		if constexpr (sizeof(T) == 4) rest_n = own_ok && a.lse_rest != nullptr ? a.lse_rest[row] : 0.f;
		delta_n = own_ok ? a.delta[row] : 0.f;
		if (threadIdx.x < TB && sgt != nullptr) ksg_n = k0 + (int)threadIdx.x < a.Skv ? sgt[threadIdx.x] : -1;
	};

	int t_of = -1, dlo = 0, dhi = 0;  // the tile that dz, the window and the positions in LDS belong to
	Window w{0, WIN_ONE};
	bool more = advance();
	if (more) fetch_item();
	while (more) {
		const int t = tn_, b = bn, k0 = t * TB;
		const bool full = full_n, first = t != t_of || per_image;
		o.seg = seg_n;
		o.lim = lim_n;
		__syncthreads();  // (the previous item's tiles are done with)
		kst.commit(Ks);
		vst.commit(Vs);
		if (threadIdx.x < TB && a.kseg != nullptr) kseg_s[threadIdx.x] = ksg_n;
		typename Tr<T>::frag qf[I::STEPS], gf[I::STEPS];
#pragma unroll
		for (int s = 0; s < I::STEPS; ++s) {
			qf[s] = qn[s];
			gf[s] = gn[s];
		}
		const float lse = lse_n, delta = delta_n, lse_rest = rest_n;
		if (first) {
			const Span own = span_of(a.qr != nullptr ? a.qr + (int64_t)b * a.nq64 : nullptr, 2 * blk, a.nq64, pos, q0 + a.off, q0 + QB - 1 + a.off);
			int plo = k0, phi = k0 + TB - 1;
			if (pos) {
				const i32x4 r = range_at(a.kr, (int64_t)b * a.nk64 + t);
				plo = r.z;
				phi = r.w;
			}
			o.pos = pos ? (in ? a.qpos[b * a.bqp + qi] : own.pmin) : qi + a.off;
			dlo = plo - own.pmax;
			dhi = phi - own.pmin;
			w = window_of(a, dlo, dhi);
			if (w.mode == WIN_LDS) {
				for (int j = threadIdx.x; j <= dhi - dlo; j += 256) win[j] = bias_at(a, o.ex, o.slope, dlo + j);
			}
			if (threadIdx.x < TB && pos) kpos_s[threadIdx.x] = 4 * (k0 + (int)threadIdx.x < a.Skv ? a.kpos[b * a.bkp + k0 + threadIdx.x] : plo);
			t_of = t;
		}
		__syncthreads();
		more = advance();
		if (more) fetch_item();
		const TileSide ts{win, kpos_s, kseg_s, nullptr};
		if (q0 + 32 * wave < a.Sq) {
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
				modify<true, CAP, BIAS_TABLE>(z, tn, a, w, ts, o, pos, k0, 32 * i, lv);
				if (!full) hide<true>(z, a, ts, o, k0, 32 * i, lv);
#pragma unroll
				for (int r = 0; r < 16; ++r) {
					float p = weight_of<T, CAP, BIAS_TABLE>(a, z[r], lse, lse_rest);
					if (!full) p = z[r] == -INFINITY ? 0.f : p;
					dz[i][r] = fmaf(p, !full && p == 0.f ? 0.f : dp[r] - delta, dz[i][r]);  // (a hidden pair's dp may be an infinity or a NaN)
				}
			}
		}
		if (per_image || !more || tn_ != t) {
			__syncthreads();
			scatter(dlo, dhi, k0);
		}
	}
	__syncthreads();
	float* po = out + (((int64_t)h * a.nblk + blk) * (tp.nchunk * tp.nimages) + part) * a.n_bucket;
	for (int i = threadIdx.x; i < a.n_bucket; i += 256) po[i] = sums[i];
}

template <typename T, int DHP, int GR> int launch(const Args& a, const TablePlan& p, float* sums, hipStream_t st) {
	const int64_t blocks = placed_blocks(a.nblk, a.H, (int64_t)p.nchunk * p.nimages);
	VITK_REQUIRE(blocks < (1 << 24), VITK_ERR_SHAPE);
	const size_t lds = sizeof(float) * (a.n_bucket + 1);
	const void* fn = a.cap_l2 > 0.f ? reinterpret_cast<const void*>(abias_table_kernel<T, DHP, GR, true>) : reinterpret_cast<const void*>(abias_table_kernel<T, DHP, GR, false>);
	if (lds + std::max(2 * Img<T, DHP>::BYTES, 8 * WIN * 4) + 8192 > 64 * 1024) {
		const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
		if (e != hipSuccess) return VITK_ERR_HIP - (int)e;
	}
	if (a.cap_l2 > 0.f) hipLaunchKernelGGL((abias_table_kernel<T, DHP, GR, true>), dim3((unsigned)blocks), dim3(256), lds, st, a, p, sums);
	else hipLaunchKernelGGL((abias_table_kernel<T, DHP, GR, false>), dim3((unsigned)blocks), dim3(256), lds, st, a, p, sums);
	VITK_CHECK_LAUNCH();
	return VITK_OK;
}
template <typename T> int table_dispatch(const Args& a, const TablePlan& p, float* sums, hipStream_t st) {
	if (a.gran == 16) {
		if (a.dh <= 32) return launch<T, 32, 16>(a, p, sums, st);
		if (a.dh <= 64) return launch<T, 64, 16>(a, p, sums, st);
		return launch<T, 128, 16>(a, p, sums, st);
	}
	if (a.dh <= 32) return launch<T, 32, 8>(a, p, sums, st);
	if (a.dh <= 64) return launch<T, 64, 8>(a, p, sums, st);
	return launch<T, 128, 8>(a, p, sums, st);
}

}  // namespace
