// kvattn.cuh — what the kernels of attention over the 4-bit cache share (kvattn.cu: an
// item a warp; kvwide.cu: an item a CTA): a batch's plan, the rounding helpers, the rows as
// they leave.
#pragma once

#include "kv.cuh"

namespace moe {
namespace kva {

constexpr int kAttnTile = 32;      // key rows of a copy
constexpr int kRunMin = 1;         // tiles of a run at least
constexpr int kRunMax = 256;       // where runs are joined
// Key tiles (2 products of 16 rows each) of one chain of sums: the tensor cores cut what they
// add to a sum, always towards zero, so 131072 rows of one sign in one chain came out 6.8e-4
// (mma.sync) and 8.3e-4 (tcgen05) too small.  After kFold tiles the sums move to the item's
// record in fp32 and begin anew: 256 products, below 2^-14 (fp32 rows 1.8e-6 off).  131072 and
// 8192 rows take 0.8 (kvattn.cu) and 2 to 4 (kvwide.cu) % longer so.  Calls whose items are
// shorter by their bounds take kernels without that (FOLD): a 2048-token prompt 127 us, in the
// first form with it 135; 64 sequences 36.7 and 37.3.
constexpr int kFold = 128;
constexpr float kLag = 4.0f;       // exponents of 2 that the running maximum may lag (0: prompt 226 us, 196)
constexpr float kLift = 10.0f;     // weights are held times 2^10
constexpr float kNoMax = 3.0e38f;  // the bias kLift - m before any row was seen

// j / n and j % n for any 31-bit j: the quotient by a rounded-down reciprocal is at
// most one short.  (A division by a runtime value is some twenty dependent
// instructions, which a decode step's few warps wait for.)
struct QuickDiv {
	unsigned n = 1, m = 0;
	QuickDiv() {}
	explicit QuickDiv(unsigned n_) : n(n_), m(n_ > 1 ? (unsigned)(0x100000000ull / n_) : 0) {}
	__device__ __forceinline__ int div(int j) const
	{
		if (n == 1)
			return j;
		const unsigned q = __umulhi((unsigned)j, m);
		return (int)(q + ((unsigned)j - q * n >= n));
	}
};

struct AttnArgs {
	BatchArgs b;
	const void *q;
	void *out;
	int64_t q_ts, q_hs, o_ts, o_hs;
	float *lse;
	const uint8_t *pages;
	int64_t page_bytes;
	int H, KVH, G;
	QuickDiv by_g, by_kvh;
	int causal, window;
	float scale2;        // scale * log2 e
	int q_vec, o_vec;    // 16-byte aligned rows
	int target;          // items wanted (0: one run a tile)
	int64_t items;       // items that the workspace holds
	float *part;         // records [item][row][HL + 4]: sums, bias, weights' sum; NULL: no item has one
	int part_rows;       // rows of an item that can be in use
	int min_rows, max_rows;   // query rows of a KV head in the sequences that are this kernel's
};

// one item of the batch
struct Item {
	int b, kvh, tile;    // sequence, KV head, tile of query rows
	int s0, n, kv;       // its first token, queries, cache rows
	int r0, rows;        // first query row (token * G + head) and rows of the tile
	int lo, hi;          // cache rows that the tile sees
	int t0, t1;          // the item's key tiles
	int run, runs;       // which run of how many
	int first;           // index of the tile's first item
};

__device__ __forceinline__ bool seq_of(const AttnArgs &a, int b, int &s0, int &n, int &kv)
{
	s0 = a.b.q_start[b];
	const int s1 = a.b.q_start[b + 1];
	n = s1 - s0;
	kv = a.b.kv_len[b];
	const bool ok = s0 >= 0 && s1 >= s0 && s1 <= a.b.T && n <= a.b.max_q && kv >= 0 &&
			kv <= a.b.max_kv && (b > 0 || s0 == 0);
	if (!ok) {
		n = 0;
		if (blockIdx.x == 0 && threadIdx.x < 32)
			atomicOr(a.b.err, kKvErrBatch);
	} else if (n * a.G < a.min_rows || n * a.G > a.max_rows) {
		n = 0;
	}
	return n > 0;
}

// key tiles of a sequence, over all of its queries
__device__ __forceinline__ int seq_tiles(const AttnArgs &a, int n, int kv)
{
	const int lo = a.window ? max(0, kv - n - a.window + 1) : 0;
	return (kv + kAttnTile - 1) / kAttnTile - lo / kAttnTile;
}

// sums of v over the lanes up to this one
__device__ __forceinline__ int warp_scan(int v)
{
	const int lane = threadIdx.x % 32;
#pragma unroll
	for (int o = 1; o < 32; o *= 2) {
		const int w = __shfl_up_sync(0xffffffffu, v, o);
		v += lane >= o ? w : 0;
	}
	return v;
}

// Item `index` of the batch (ITEM), or tile `index` of its query tiles with the
// tile's number of runs, by one warp.  Every CTA of both kernels derives the same
// plan from the lengths, 32 sequences at a time: all work in key tiles over the
// items wanted gives the run's length (in fp32: any length is right); sums over the
// sequences before give a sequence's first item.  The sums fit 32 bits where the
// arrays keep to the call's bounds (the host checks those); where q_start does not,
// they may not, and no item is taken that lies outside its sequence.
template <int RPT, bool ITEM>
__device__ __forceinline__ bool find_item(const AttnArgs &a, int index, Item &f)
{
	const int lane = threadIdx.x % 32, B = a.b.B;
	int s0 = 0, n = 0, kv = 0;
	int run = 1 << 30;   // target 0: query tiles enough, one run each
	if (a.target) {
		float all = 0.0f;
		for (int b = lane; b < B; b += 32)
			if (seq_of(a, b, s0, n, kv))
				all += (float)((n * a.G + RPT - 1) / RPT) * (float)seq_tiles(a, n, kv);
		run = (int)fminf(ceilf(warp_sum(all) * a.KVH / a.target), (float)kRunMax);
		run = max(run, kRunMin);
	} else if (blockIdx.x == 0 && threadIdx.x < 32) {
		// the walk below ends at the item: here every sequence is looked at, and those
		// out of range reported
		for (int b = lane; b < B; b += 32)
			seq_of(a, b, s0, n, kv);
		n = 0;
	}
	int item0 = 0, tile0 = 0;
	for (int b0 = 0; b0 < B; b0 += 32) {
		const int b = b0 + lane;
		int tiles = 0, runs = 0;
		if (B > 32 || !a.target) {
			n = 0;
			if (b < B)
				seq_of(a, b, s0, n, kv);
		}
		if (b < B && n > 0) {
			tiles = (n * a.G + RPT - 1) / RPT;
			runs = max(1, (int)((unsigned)(seq_tiles(a, n, kv) + run - 1) / (unsigned)run));
		}
		const int items = tiles * runs * a.KVH;
		const int iend = item0 + warp_scan(items);
		const int tend = ITEM ? iend : tile0 + warp_scan(tiles * a.KVH);
		const unsigned m = __ballot_sync(0xffffffffu, index < (ITEM ? iend : tend));
		if (m) {
			// the first sequence that ends behind it
			const int src = __ffs(m) - 1;
			s0 = __shfl_sync(0xffffffffu, s0, src);
			n = __shfl_sync(0xffffffffu, n, src);
			kv = __shfl_sync(0xffffffffu, kv, src);
			tiles = __shfl_sync(0xffffffffu, tiles, src);
			runs = __shfl_sync(0xffffffffu, runs, src);
			const int i0 = __shfl_sync(0xffffffffu, iend - items, src);
			const int t0 = __shfl_sync(0xffffffffu, tend - tiles * a.KVH, src);
			const unsigned at = index - (ITEM ? i0 : t0);
			// KV heads side by side; the last tiles, which see the most, first
			f.b = b0 + src;
			f.s0 = s0;
			f.n = n;
			f.kv = kv;
			const unsigned rest = a.by_kvh.div(at);
			f.kvh = at - rest * a.KVH;
			const unsigned rank = ITEM ? rest / (unsigned)runs : rest;
			if (rank >= (unsigned)tiles)   // sums that do not fit (see above)
				return false;
			f.run = ITEM ? rest - rank * (unsigned)runs : 0;
			f.first = i0 + rank * runs * a.KVH + f.kvh;
			f.tile = tiles - 1 - (int)rank;
			f.r0 = f.tile * RPT;
			f.rows = min(RPT, n * a.G - f.r0);
			const int p0 = kv - n + a.by_g.div(f.r0), p1 = kv - n + a.by_g.div(f.r0 + f.rows - 1);
			f.lo = a.window ? max(0, p0 - a.window + 1) : 0;
			f.hi = a.causal ? min(kv, p1 + 1) : kv;
			const int ta = f.lo / kAttnTile, tb = max(ta, (f.hi + kAttnTile - 1) / kAttnTile);
			f.runs = max(1, (int)((unsigned)(tb - ta + run - 1) / (unsigned)run));
			f.t0 = min(tb, ta + f.run * run);
			f.t1 = min(tb, f.t0 + run);
			// q_start that does not rise can name more items than it has
			// tokens for: those behind the plan's bound are left out
			return f.first >= 0 && f.first + (int64_t)(runs - 1) * a.KVH < a.items &&
			       (!ITEM || f.run < f.runs);
		}
		item0 = __shfl_sync(0xffffffffu, iend, 31);
		tile0 = __shfl_sync(0xffffffffu, tend, 31);
	}
	return false;
}

// found by the CTA's first warp for all of them
template <int RPT, bool ITEM>
__device__ __forceinline__ bool cta_item(const AttnArgs &a, int index, Item &f)
{
	__shared__ Item found;
	__shared__ int ok;
	if (threadIdx.x < 32) {
		Item x;
		const bool in = find_item<RPT, ITEM>(a, index, x);
		if (threadIdx.x == 0) {
			found = x;
			ok = in;
		}
	}
	__syncthreads();
	f = found;
	return ok;
}

__device__ __forceinline__ float ex2(float x)
{
	float y;
	asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
	return y;
}

__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi)
{
	return h2_bits(__floats2half2_rn(lo, hi));
}

// half `at` of a word
__device__ __forceinline__ float half_of(uint32_t w, int at)
{
	const __half2 h = bits_h2(w);
	return at ? __high2float(h) : __low2float(h);
}

__device__ __forceinline__ uint32_t set_half(uint32_t w, int at, float v)
{
	const uint32_t h = __half_as_ushort(__float2half_rn(v));
	return at ? (w & 0xffffu) | h << 16 : (w & 0xffff0000u) | h;
}

// Row r of a tile as it leaves: sums over the weights' sum, zeros where nothing was
// seen, and its log-sum-exp
template <typename T>
struct RowOut {
	T *p;
	float *lse_at;
	float il, l, bias;
	bool vec;
	__device__ __forceinline__ RowOut(const AttnArgs &a, const Item &it, int r, float bias_, float l_)
		: il(l_ == 0.0f ? 0.0f : 1.0f / l_), l(l_), bias(bias_), vec(a.o_vec)
	{
		const int qr = it.r0 + r, i = a.by_g.div(qr);
		const int token = it.s0 + i, head = it.kvh * a.G + qr - i * a.G;
		p = static_cast<T *>(a.out) + token * a.o_ts + head * a.o_hs;
		lse_at = a.lse ? a.lse + (int64_t)token * a.H + head : nullptr;
	}
	__device__ __forceinline__ void two(int e, float x, float y) const
	{
		x *= il;
		y *= il;
		if (!vec) {
			p[e] = from_f32<T>(x);
			p[e + 1] = from_f32<T>(y);
		} else if constexpr (sizeof(T) == 4) {
			*reinterpret_cast<float2 *>(p + e) = make_float2(x, y);
		} else {
			T v[2] = {from_f32<T>(x), from_f32<T>(y)};
			*reinterpret_cast<uint32_t *>(p + e) = *reinterpret_cast<uint32_t *>(v);
		}
	}
	// 8 values side by side (of rows in 16 bits)
	__device__ __forceinline__ void eight(int e, const float (&v)[8]) const
	{
		T t[8];
#pragma unroll
		for (int k = 0; k < 8; k++)
			t[k] = from_f32<T>(v[k] * il);
		if (vec) {
			*reinterpret_cast<uint4 *>(p + e) = *reinterpret_cast<uint4 *>(t);
		} else {
#pragma unroll
			for (int k = 0; k < 8; k++)
				p[e + k] = t[k];
		}
	}
	__device__ __forceinline__ void lse() const
	{
		if (lse_at)
			*lse_at = l == 0.0f ? -__int_as_float(0x7f800000)
					    : 0.693147180559945f * (log2f(l) - bias);
	}
};

// 16 bytes to shared memory, in flight until its group is waited for
__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t *src)
{
	asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// all but the newest N groups have landed
template <int N>
__device__ __forceinline__ void copies_wait()
{
	asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// The runs of a tile's query rows joined, a CTA a tile or some rows of it: each row by
// as many of its warps as the rows leave it, which take the runs in turn.  A few
// dependent loads long, so the sums of a warp's first runs leave before the factors
// are known (latency: 2 to 5 us behind the kernel above).
constexpr int kMergeWarps = 4;
template <typename T, int HL, int RPT>
__global__ void __launch_bounds__(32 * kMergeWarps) kv_merge_kernel(AttnArgs a)
{
	constexpr int OS = HL + 4, E4 = HL / 4;                  // float4s of a row
	constexpr int W = E4 < 32 ? E4 : 32, SIDE = 32 / W, NV = E4 / W;
	constexpr int BATCH = 4;
	__shared__ float4 red[kMergeWarps][E4];
	Item it;
	const bool mine = cta_item<RPT, false>(a, blockIdx.x, it) && it.runs > 1;
	griddep_wait();   // the runs are written
	if (!mine)
		return;
	const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
	// the CTA's rows of the tile; warps of a row
	const int each = (a.part_rows + gridDim.y - 1) / gridDim.y;
	const int from = blockIdx.y * each, to = min(from + each, it.rows);
	int share = kMergeWarps;
	while (share > 1 && share * (to - from) > kMergeWarps)
		share /= 2;
	const int part = warp % share, ds = share * SIDE;
	const int64_t step = (int64_t)a.KVH * a.part_rows * OS;   // between the runs of a tile
	for (int r0 = from; r0 < to; r0 += kMergeWarps / share) {
		const int r = r0 + warp / share;
		const bool row = r < to;   // the whole warp
		const float *pp = a.part + ((int64_t)it.first * a.part_rows + (row ? r : 0)) * OS;
		const int s0 = part * SIDE + lane / W, e = lane % W * 4;
		const int runs = row ? it.runs : 0;
		float4 x[BATCH][NV], o[NV];
		float xb[BATCH];
		auto load = [&](int s) {
#pragma unroll
			for (int k = 0; k < BATCH; k++) {
				const float *p = pp + (s + k * ds) * step;
				const bool in = s + k * ds < runs;
				xb[k] = in ? p[HL] : kNoMax;
#pragma unroll
				for (int v = 0; v < NV; v++)
					x[k][v] = in ? *reinterpret_cast<const float4 *>(p + e + 4 * W * v)
						     : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
			}
		};
		load(s0);
		float b = kNoMax, l = 0.0f;
		for (int s = lane; s < runs; s += 32)
			b = fminf(b, pp[s * step + HL]);
		b = -warp_max(-b);
		for (int s = lane; s < runs; s += 32)
			l += pp[s * step + HL + 1] * ex2(b - pp[s * step + HL]);
		l = warp_sum(l);
#pragma unroll
		for (int v = 0; v < NV; v++)
			o[v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
		for (int s = s0;;) {
#pragma unroll
			for (int k = 0; k < BATCH; k++) {
				const float f = ex2(b - xb[k]);
#pragma unroll
				for (int v = 0; v < NV; v++) {
					o[v].x = fmaf(x[k][v].x, f, o[v].x);
					o[v].y = fmaf(x[k][v].y, f, o[v].y);
					o[v].z = fmaf(x[k][v].z, f, o[v].z);
					o[v].w = fmaf(x[k][v].w, f, o[v].w);
				}
			}
			s += BATCH * ds;
			if (s - lane / W >= runs)
				break;
			load(s);
		}
#pragma unroll
		for (int v = 0; v < NV; v++) {
			if (SIDE == 2) {
				o[v].x += __shfl_xor_sync(0xffffffffu, o[v].x, 16);
				o[v].y += __shfl_xor_sync(0xffffffffu, o[v].y, 16);
				o[v].z += __shfl_xor_sync(0xffffffffu, o[v].z, 16);
				o[v].w += __shfl_xor_sync(0xffffffffu, o[v].w, 16);
			}
			if (share > 1 && lane < W)
				red[warp][lane + W * v] = o[v];
		}
		if (share > 1) {   // one round of rows then: share * rows <= the warps
			__syncthreads();
			if (part == 0 && lane < W) {
#pragma unroll
				for (int v = 0; v < NV; v++)
					for (int w = 1; w < share; w++) {
						const float4 y = red[warp + w][lane + W * v];
						o[v].x += y.x;
						o[v].y += y.y;
						o[v].z += y.z;
						o[v].w += y.w;
					}
			}
		}
		if (row && part == 0 && lane < W) {
			const RowOut<T> out(a, it, r, b, l);
#pragma unroll
			for (int v = 0; v < NV; v++) {
				out.two(e + 4 * W * v, o[v].x, o[v].y);
				out.two(e + 4 * W * v + 2, o[v].z, o[v].w);
			}
			if (lane == 0)
				out.lse();
		}
	}
}

// the sizes that a launch is planned with, from the call's bounds alone
struct Plan {
	int nt = 1, rpt = 8;     // column tiles, query rows of an item
	int rows = 8;            // rows of them that can be in use
	int64_t tiles = 0;       // at most so many query tiles x KV heads
	int64_t items = 0;       // and items
	int target = 0;
	bool split = false;      // runs at all
	bool folds = false;      // items that may have more than kFold tiles
	size_t part_bytes = 0;
};

// the launch behind a kernel whose tiles have runs
template <typename T, int HL, int RPT>
cudaError_t launch_merge(const AttnArgs &a, const Plan &p, cudaStream_t st)
{
	if (!p.split)
		return cudaSuccess;
	cudaLaunchConfig_t cfg{};
	// few tiles: their rows over several CTAs, up to one a row (one CTA a tile: 8
	// drafted tokens 39 us, 23; 4 x 131072 rows 137, 126)
	const int64_t y = 8 * (int64_t)sm_count() / p.tiles;
	cfg.gridDim = dim3((unsigned)p.tiles, (unsigned)(y < 1 ? 1 : y < p.rows ? y : p.rows));
	cfg.blockDim = dim3(32 * kMergeWarps);
	cfg.stream = st;
	cudaLaunchAttribute at[1];
	at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
	at[0].val.programmaticStreamSerializationAllowed = 1;
	cfg.attrs = at;
	cfg.numAttrs = pdl_enabled() ? 1 : 0;
	return cudaLaunchKernelEx(&cfg, kv_merge_kernel<T, HL, RPT>, a);
}

// kvwide.cu: fp16 or bf16 rows (type), head_len 64 or 128, items of kWideRows query rows
constexpr int kWideRows = 256;
cudaError_t launch_wide(const AttnArgs &a, const Plan &p, int type, int HL, cudaStream_t st);

}  // namespace kva
}  // namespace moe
