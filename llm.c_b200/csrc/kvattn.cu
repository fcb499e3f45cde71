// kvattn.cu — attention over the paged 4-bit cache (moe_kv_attention).
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q.k_j - max)
//
// What has to be read is the cache: 0.5625 bytes a value.  A GPU reads such
// values faster than its CUDA cores can multiply them (46 values a clock and
// SM at 6.5 TB/s), so both products run on mma.sync, with the codes as exact
// fp16 numbers and the block scales applied in fp32 outside of the products:
//
//   S^T = K q^T    A = 16 rows of codes, B = q^T (8 columns).  A row's scale of
//                  block b multiplies the block's partial sums.
//   O^T += V^T P^T A = 16 values of the head x 16 rows, B = the weights, times
//                  the rows' scale of the block that the 16 values belong to.
//
// With the cache as the 16-row operand a decode step's few queries (the heads
// of a KV head's group) fill 8 columns instead of 16 rows, and the codes go
// from shared memory to operand registers without a transposition: the page
// layout places a thread's nibbles of all blocks side by side.  S^T comes out
// with a row per lane group and P^T wants a column per lane group: one
// movmatrix per 8 x 8 tile turns it.
//
// fp16 weights: p <= 16 (the running maximum may lag by 4, in exponents of 2;
// then nothing needs rescaling), times 2^10, times the row's V scale brought to
// [1, 2) by a power of two per block, so weights down to 2^-24 of the largest
// keep fp16's full precision.  q is brought to 2^13 by a power of two per row.
// fp32 rows take two columns, the fp16 value and the fp16 remainder.
//
// Work: an item is a KV head of a sequence, a tile of its query rows (query
// token x head of the group) and a run of 32-row key tiles; the CTA's 4 warps
// take the run's tiles in turn, each with a ring of bulk copies of its own, and
// join their sums at the end.  The run's length is chosen on the device from
// the batch's lengths so that the items fill the GPU however ragged they are;
// a tile of queries with several runs is joined by a second kernel.
#include "kv.cuh"
#include "expert_core.cuh"

namespace moe {
namespace {

constexpr int kAttnWarps = 4, kAttnThreads = 32 * kAttnWarps;
constexpr int kAttnTile = 32;      // key rows of a warp's copy
constexpr int kAttnStages = 3;     // copies in a warp's ring
constexpr int kRunMin = kAttnWarps;          // tiles of a run: one for each warp
constexpr int kRunMax = 256 * kAttnWarps;    // 512 products a warp in one fp32 chain
constexpr float kLag = 4.0f;       // exponents of 2 that the running maximum may lag
constexpr float kLift = 10.0f;     // weights are held times 2^10

struct AttnArgs {
	BatchArgs b;
	const void *q;
	void *out;
	int64_t q_ts, q_hs, o_ts, o_hs;
	float *lse;
	const uint8_t *pages;
	int64_t page_bytes;
	int H, KVH, G;
	int causal, window;
	float scale2;        // scale * log2 e
	int q_vec, o_vec;    // 16-byte aligned rows
	int target;          // items wanted (0: one run a tile)
	int64_t items;       // items that the workspace holds
	float *part;         // [item][row][HL + 2]
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
		if (blockIdx.x == 0)
			atomicOr(a.b.err, kKvErrBatch);
	}
	return ok;
}

// key tiles of a sequence, over all of its queries
__device__ __forceinline__ int seq_tiles(const AttnArgs &a, int n, int kv)
{
	const int lo = a.window ? max(0, kv - n - a.window + 1) : 0;
	return (kv + kAttnTile - 1) / kAttnTile - lo / kAttnTile;
}

// sums of v over the CTA's threads before this one, and of all of them
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t &all, int64_t *red)
{
	const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
	int64_t s = v;
#pragma unroll
	for (int o = 1; o < 32; o *= 2) {
		const int64_t w = __shfl_up_sync(0xffffffffu, s, o);
		if (lane >= o)
			s += w;
	}
	__syncthreads();
	if (lane == 31)
		red[warp] = s;
	__syncthreads();
	int64_t before = 0;
	all = 0;
#pragma unroll
	for (int w = 0; w < kAttnWarps; w++) {
		if (w < warp)
			before += red[w];
		all += red[w];
	}
	return before + s - v;
}

// Item `index` of the batch (ITEM), or tile `index` of its query tiles with
// the tile's number of runs.  Every CTA of both kernels derives the same plan
// from the lengths: all work in key tiles over the items wanted gives the
// run's length; sums over the sequences before give a sequence's first item.
template <int RPT, bool ITEM>
__device__ __forceinline__ bool find_item(const AttnArgs &a, int64_t index, Item &it)
{
	__shared__ int64_t red[kAttnWarps];
	__shared__ Item found;
	__shared__ int hit;
	const int B = a.b.B;
	int s0 = 0, n = 0, kv = 0;
	int64_t all = 0;
	for (int b0 = 0; b0 < B; b0 += kAttnThreads) {
		const int b = b0 + threadIdx.x;
		int64_t w = 0, sum;
		if (b < B && seq_of(a, b, s0, n, kv))
			w = (int64_t)((n * (int64_t)a.G + RPT - 1) / RPT) * seq_tiles(a, n, kv);
		block_scan(w, sum, red);
		all += sum;
	}
	all *= a.KVH;
	int64_t run = (int64_t)1 << 40;   // target 0: query tiles enough, one run each
	if (a.target) {
		run = (all + a.target - 1) / a.target;
		run = run < kRunMin ? kRunMin : run > kRunMax ? kRunMax : run;
	}
	if (threadIdx.x == 0)
		hit = 0;
	int64_t item0 = 0, tile0 = 0;
	for (int b0 = 0; b0 < B; b0 += kAttnThreads) {
		const int b = b0 + threadIdx.x;
		int64_t tiles = 0, runs = 0, items, sum, tsum;
		if (B > kAttnThreads) {
			n = 0;
			if (b < B)
				seq_of(a, b, s0, n, kv);
		}
		if (b < B && n > 0) {
			tiles = (n * (int64_t)a.G + RPT - 1) / RPT;
			runs = (seq_tiles(a, n, kv) + run - 1) / run;
			runs = runs < 1 ? 1 : runs;
		}
		items = tiles * runs * a.KVH;
		const int64_t i0 = item0 + block_scan(items, sum, red);
		const int64_t q0 = tile0 + block_scan(tiles * a.KVH, tsum, red);
		const int64_t at = index - (ITEM ? i0 : q0);
		if (at >= 0 && at < (ITEM ? items : tiles * a.KVH)) {
			// KV heads side by side; the last tiles, which see the most, first
			Item f;
			f.b = b;
			f.s0 = s0;
			f.n = n;
			f.kv = kv;
			f.kvh = (int)(at % a.KVH);
			const int64_t rest = at / a.KVH;
			f.run = ITEM ? (int)(rest % runs) : 0;
			const int64_t rank = ITEM ? rest / runs : rest;
			f.tile = (int)(tiles - 1 - rank);
			const int64_t first = i0 + rank * runs * a.KVH + f.kvh;
			f.first = (int)first;
			f.r0 = f.tile * RPT;
			f.rows = (int)min((int64_t)RPT, n * (int64_t)a.G - f.r0);
			const int p0 = kv - n + f.r0 / a.G, p1 = kv - n + (f.r0 + f.rows - 1) / a.G;
			f.lo = a.window ? max(0, p0 - a.window + 1) : 0;
			f.hi = a.causal ? min(kv, p1 + 1) : kv;
			const int ta = f.lo / kAttnTile, tb = max(ta, (f.hi + kAttnTile - 1) / kAttnTile);
			f.runs = max(1, (int)((tb - ta + run - 1) / run));
			f.t0 = ta + (int)(f.run * run);
			f.t1 = (int)min((int64_t)tb, f.t0 + run);
			found = f;
			// q_start that does not rise can name more items than it has
			// tokens for: those behind the plan's bound are left out
			hit = first + (runs - 1) * a.KVH < a.items;
		}
		item0 += sum;
		tile0 += tsum;
	}
	__syncthreads();
	it = found;
	return hit && (!ITEM || it.run < it.runs);
}

__device__ __forceinline__ void mma_step(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
					 uint32_t b1)
{
	asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
		     "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
		     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
		     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x)
{
	uint32_t y;
	asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
	return y;
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

// codes in the low nibbles of bytes 0 and 2 as fp16 code - 8: 1024 + code by
// placing the nibble in 1024's mantissa, less 1032
__device__ __forceinline__ uint32_t codes_low(uint32_t w)
{
	return h2_bits(__hsub2(bits_h2((w & 0x000f000fu) | 0x64006400u), bits_h2(0x64086408u)));
}
// the high nibbles: 1024 + 16 code, over 16, less 72 (each step exact)
__device__ __forceinline__ uint32_t codes_high(uint32_t w)
{
	return h2_bits(__hfma2(bits_h2((w & 0x00f000f0u) | 0x64006400u), bits_h2(0x2c002c00u),
			       bits_h2(0xd480d480u)));
}

// tile row of A's row j: rows j and j ^ 2.. stay within 16; chosen so that the
// 8 rows of a shared-memory read touch both halves of the banks
__device__ __forceinline__ int tile_row(int j) { return j ^ ((j >> 1) & 1); }

// NW 32-bit words from shared memory
template <int NW>
__device__ __forceinline__ void lds_words(const uint8_t *p, uint32_t (&w)[NW])
{
	if constexpr (NW % 4 == 0) {
#pragma unroll
		for (int i = 0; i < NW; i += 4) {
			const uint4 v = *reinterpret_cast<const uint4 *>(p + 4 * i);
			w[i] = v.x;
			w[i + 1] = v.y;
			w[i + 2] = v.z;
			w[i + 3] = v.w;
		}
	} else if constexpr (NW == 2) {
		const uint2 v = *reinterpret_cast<const uint2 *>(p);
		w[0] = v.x;
		w[1] = v.y;
	} else {
		w[0] = *reinterpret_cast<const uint32_t *>(p);
	}
}

// values e .. e + 3 of row r of a tile: the sums over the weights' sum, and
// with e 0 the row's log-sum-exp
template <typename T>
__device__ __forceinline__ void write_row(const AttnArgs &a, const Item &it, int r, int e, float4 v,
					  float m, float l, bool first)
{
	const int qr = it.r0 + r, token = it.s0 + qr / a.G, head = it.kvh * a.G + qr % a.G;
	// nothing seen: zeros
	const float il = l == 0.0f ? 0.0f : 1.0f / l;
	T *p = static_cast<T *>(a.out) + token * a.o_ts + head * a.o_hs + e;
	const float x[4] = {v.x * il, v.y * il, v.z * il, v.w * il};
	if (a.o_vec && sizeof(T) == 4) {
		*reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
	} else if (a.o_vec) {
		uint2 u;
		T *h = reinterpret_cast<T *>(&u);
#pragma unroll
		for (int k = 0; k < 4; k++)
			h[k] = from_f32<T>(x[k]);
		*reinterpret_cast<uint2 *>(p) = u;
	} else {
#pragma unroll
		for (int k = 0; k < 4; k++)
			p[k] = from_f32<T>(x[k]);
	}
	if (first && a.lse)
		a.lse[(int64_t)token * a.H + head] =
			l == 0.0f ? -__int_as_float(0x7f800000) : 0.693147180559945f * (m + log2f(l) - kLift);
}

template <int HL>
struct StageLayout {
	static constexpr int NB = HL / 32;
	static constexpr int kCodes = kAttnTile * HL / 2, kScales = kAttnTile * NB * 2;
	static constexpr int kKS = kCodes, kVC = kCodes + kScales, kVS = 2 * kCodes + kScales;
	static constexpr int kBytes = 2 * (kCodes + kScales);
};

template <int HL, int NT>
constexpr int attn_smem()
{
	constexpr int ring = kAttnWarps * kAttnStages * StageLayout<HL>::kBytes;
	constexpr int join = kAttnWarps * 8 * NT * (HL + 4) * 4;
	return ring > join ? ring : join;
}

template <int HL, int NT>
constexpr bool kQInRegs = HL * NT <= 256;

template <typename T, int HL, int NT>
__global__ void __launch_bounds__(kAttnThreads) kv_attn_kernel(AttnArgs a)
{
	constexpr bool SPLIT = sizeof(T) == 4;        // two columns a row
	constexpr int RPN = SPLIT ? 4 : 8;            // rows of an 8-column tile
	constexpr int RPT = RPN * NT, NB = HL / 32, COLS = 8 * NT;
	constexpr bool QR = kQInRegs<HL, NT>;
	using SL = StageLayout<HL>;
	extern __shared__ __align__(128) uint8_t smem[];
	__shared__ __align__(8) uint64_t bars[kAttnWarps][kAttnStages];
	__shared__ float sm_m[kAttnWarps][COLS], sm_l[kAttnWarps][COLS];
	__shared__ uint2 sm_q[QR ? 1 : 2 * NB * NT][32];
	__shared__ float sm_qs[COLS];
	const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, c = lane % 4;

	griddep_launch_dependents();
	if (threadIdx.x < kAttnWarps * kAttnStages)
		mbar_init(&bars[0][0] + threadIdx.x, 1);
	fence_mbar_init();
	Item it;
	if (!find_item<RPT, true>(a, blockIdx.x, it))   // its barriers order the inits too
		return;

	// ---- the warp's key tiles: t0 + warp, + 4, ..: lane l keeps the pages of
	// the next 32 of them (two where a page is half a tile)
	const int ntile = max(0, (it.t1 - it.t0 - warp + kAttnWarps - 1) / kAttnWarps);
	const int32_t *table = a.b.table + it.b * a.b.table_stride;
	const int P = 1 << a.b.page_log2;
	const bool small = P < kAttnTile;
	uint8_t *ring = smem + warp * kAttnStages * SL::kBytes;
	uint64_t *bar = bars[warp];
	auto key0 = [&](int i) { return (it.t0 + warp + i * kAttnWarps) * kAttnTile; };
	// which halves of tile i hold rows that the query tile sees
	auto needs = [&](int i) -> int {
		const int k0 = key0(i);
		return (k0 < it.hi && k0 + 16 > it.lo ? 1 : 0) |
		       (k0 + 16 < it.hi && k0 + 32 > it.lo ? 2 : 0);
	};
	int page_a = -1, page_b = -1;   // of tile (i & ~31) + lane
	auto load_pages = [&](int i) {
		page_a = page_b = -1;
		if (i + lane < ntile) {
			const int need = needs(i + lane), k0 = key0(i + lane);
			if (need & (small ? 1 : 3))
				page_a = table[k0 >> a.b.page_log2];
			if (small && (need & 2))
				page_b = table[(k0 + 16) >> a.b.page_log2];
			const bool bad = ((need & (small ? 1 : 3)) && (unsigned)page_a >= (unsigned)a.b.n_pages) ||
					 (small && (need & 2) && (unsigned)page_b >= (unsigned)a.b.n_pages);
			if (bad)
				atomicOr(a.b.err, kKvErrPage);
			if ((unsigned)page_a >= (unsigned)a.b.n_pages)
				page_a = -1;
			if ((unsigned)page_b >= (unsigned)a.b.n_pages)
				page_b = -1;
		}
	};
	// the halves of tile i that are in the ring (pages outside the cache are
	// not read: their rows count as unseen)
	auto present = [&](int i) -> int {
		const int pa = __shfl_sync(0xffffffffu, page_a, i & 31);
		const int pb = __shfl_sync(0xffffffffu, page_b, i & 31);
		const int need = needs(i);
		if (!small)
			return pa >= 0 ? need : 0;
		return (pa >= 0 ? need & 1 : 0) | (pb >= 0 ? need & 2 : 0);
	};
	const int64_t half_rec = (int64_t)(HL / 2 + HL / 16) << a.b.page_log2;
	auto copy_rows = [&](uint8_t *st, uint64_t *br, int page, int k0, int at, int n) {
		const uint8_t *rec = a.pages + page * a.page_bytes + 2 * it.kvh * half_rec;
		const int r = k0 & (P - 1);
		const uint8_t *sc = rec + ((int64_t)(HL / 2) << a.b.page_log2);
		bulk_g2s(st + at * (HL / 2), rec + r * (HL / 2), n * (HL / 2), br);
		bulk_g2s(st + SL::kKS + at * NB * 2, sc + r * NB * 2, n * NB * 2, br);
		bulk_g2s(st + SL::kVC + at * (HL / 2), rec + half_rec + r * (HL / 2), n * (HL / 2), br);
		bulk_g2s(st + SL::kVS + at * NB * 2, sc + half_rec + r * NB * 2, n * NB * 2, br);
	};
	unsigned ring_have = 0;   // 2 bits a stage: the halves in it
	auto issue = [&](int i) {
		const int have = present(i), at = 2 * (i % kAttnStages);
		ring_have = (ring_have & ~(3u << at)) | (unsigned)have << at;
		const int pa = __shfl_sync(0xffffffffu, page_a, i & 31);
		const int pb = __shfl_sync(0xffffffffu, page_b, i & 31);
		if (lane == 0) {
			uint8_t *st = ring + (i % kAttnStages) * SL::kBytes;
			uint64_t *br = bar + i % kAttnStages;
			const int k0 = key0(i);
			constexpr int row = 2 * (HL / 2 + NB * 2);
			mbar_arrive_expect_tx(br, ((have & 1) + (have >> 1)) * 16 * row);
			if (!small && have == 3) {
				copy_rows(st, br, pa, k0, 0, 32);
			} else {
				if (have & 1)
					copy_rows(st, br, pa, k0, 0, 16);
				if (have & 2)
					copy_rows(st, br, small ? pb : pa, k0 + 16, 16, 16);
			}
		}
	};
	load_pages(0);
	const int pre = min(ntile, kAttnStages);
	for (int i = 0; i < pre; i++)
		issue(i);

	// ---- the queries: column n = g of every 8-column tile, values 4 c .. of
	// each half block, as B fragments
	uint2 qf[QR ? 2 * NB * NT : 1];
	const T *qp = static_cast<const T *>(a.q) + (int64_t)it.kvh * a.G * a.q_hs;
	float qs_own[QR ? NT : 1];
	for (int nt = QR ? 0 : warp; nt < NT; nt += QR ? 1 : kAttnWarps) {
		const int r = nt * RPN + (SPLIT ? g / 2 : g);
		float x[HL / 4];
		if (r < it.rows) {
			const int qr = it.r0 + r;
			const T *p = qp + (it.s0 + qr / a.G) * a.q_ts + (qr % a.G) * a.q_hs;
#pragma unroll
			for (int h = 0; h < HL / 16; h++) {
				if (a.q_vec && sizeof(T) == 4) {
					const float4 v = *reinterpret_cast<const float4 *>(p + 16 * h + 4 * c);
					x[4 * h] = v.x;
					x[4 * h + 1] = v.y;
					x[4 * h + 2] = v.z;
					x[4 * h + 3] = v.w;
				} else if (a.q_vec) {
					uint2 v = *reinterpret_cast<const uint2 *>(p + 16 * h + 4 * c);
					const T *e = reinterpret_cast<const T *>(&v);
#pragma unroll
					for (int k = 0; k < 4; k++)
						x[4 * h + k] = to_f32(e[k]);
				} else {
#pragma unroll
					for (int k = 0; k < 4; k++)
						x[4 * h + k] = to_f32(p[16 * h + 4 * c + k]);
				}
			}
		} else {
#pragma unroll
			for (int k = 0; k < HL / 4; k++)
				x[k] = 0.0f;
		}
		float top = 0.0f;
		bool bad = false;
#pragma unroll
		for (int k = 0; k < HL / 4; k++) {
			top = fmaxf(top, fabsf(x[k]));
			bad |= !(fabsf(x[k]) <= 3.402823466e38f);
		}
		top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
		top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
		const unsigned badm = __ballot_sync(0xffffffffu, bad);
		bad = (badm >> (4 * g)) & 15;
		const int e = top > 0.0f && !bad ? 13 - ilogbf(top) : 0;   // -114 .. 162
		const float up0 = __int_as_float((127 + e / 2) << 23);
		const float up1 = __int_as_float((127 + e - e / 2) << 23);
		// a query with an infinity or a NaN has no finite scores: NaN
		const float qs = bad ? __int_as_float(0x7fffffff) : scalbnf(a.scale2, -e);
#pragma unroll
		for (int k = 0; k < HL / 4; k++) {
			const float v = bad ? 0.0f : x[k] * up0 * up1;
			const float hi = __half2float(__float2half_rn(v));
			x[k] = SPLIT && (g & 1) ? v - hi : hi;
		}
#pragma unroll
		for (int h = 0; h < HL / 16; h++) {
			const uint2 f = make_uint2(pack_h2(x[4 * h], x[4 * h + 2]),
						   pack_h2(x[4 * h + 1], x[4 * h + 3]));
			if constexpr (QR)
				qf[nt * 2 * NB + h] = f;
			else
				sm_q[nt * 2 * NB + h][lane] = f;
		}
		if constexpr (QR)
			qs_own[nt] = qs;
		else if (c == 0)
			sm_qs[nt * 8 + g] = qs;
	}
	if constexpr (!QR)
		__syncthreads();
	// factors of this lane's columns 2 c, 2 c + 1 of each tile
	float qs0[NT], qs1[NT];
#pragma unroll
	for (int nt = 0; nt < NT; nt++) {
		if constexpr (QR) {
			qs0[nt] = __shfl_sync(0xffffffffu, qs_own[nt], 8 * c);
			qs1[nt] = __shfl_sync(0xffffffffu, qs_own[nt], 8 * c + 4);
		} else {
			qs0[nt] = sm_qs[nt * 8 + 2 * c];
			qs1[nt] = sm_qs[nt * 8 + 2 * c + 1];
		}
	}
	// the cache row at which each column's query stands
	int row0[NT], row1[NT];
#pragma unroll
	for (int nt = 0; nt < NT; nt++) {
		const int ra = it.r0 + nt * RPN + (SPLIT ? c : 2 * c);
		row0[nt] = it.kv - it.n + ra / a.G;
		row1[nt] = SPLIT ? row0[nt] : it.kv - it.n + (ra + 1) / a.G;
	}
	const int first_row = it.kv - it.n + it.r0 / a.G;
	const int last_row = it.kv - it.n + (it.r0 + it.rows - 1) / a.G;

	float o[2 * NB][NT][4];
	float m0[NT], m1[NT], l0[NT], l1[NT], rv[NB];
#pragma unroll
	for (int i = 0; i < 2 * NB; i++)
#pragma unroll
		for (int nt = 0; nt < NT; nt++)
#pragma unroll
			for (int k = 0; k < 4; k++)
				o[i][nt][k] = 0.0f;
#pragma unroll
	for (int nt = 0; nt < NT; nt++) {
		m0[nt] = m1[nt] = -3.0e38f;
		l0[nt] = l1[nt] = 0.0f;
	}
#pragma unroll
	for (int b = 0; b < NB; b++)
		rv[b] = 1.7014118e38f;   // 2^127: the first V scale sets it

	const int ja = tile_row(g);                                  // A's rows g and g + 8
	const int va = tile_row(2 * c), vb = tile_row(2 * c + 1);    // A's columns 2 c ..
	int i = 0;
	for (; i < ntile; i++) {
		if (!mbar_wait(bar + i % kAttnStages, (i / kAttnStages) & 1))
			break;
		const uint8_t *st = ring + (i % kAttnStages) * SL::kBytes;
		const int have = ring_have >> (2 * (i % kAttnStages)) & 3;
		const int k0 = key0(i);
		const bool full = have == 3 && k0 >= it.lo && k0 + kAttnTile <= it.kv &&
				  (!a.causal || k0 + kAttnTile - 1 <= first_row) &&
				  (!a.window || k0 > last_row - a.window);
#pragma unroll 1
		for (int u = 0; u < 2; u++) {
			if (!(have >> u & 1))
				continue;
			const int base = 16 * u;
			// ---- scores
			float s[NT][4];
#pragma unroll
			for (int nt = 0; nt < NT; nt++)
#pragma unroll
				for (int k = 0; k < 4; k++)
					s[nt][k] = 0.0f;
			{
				uint32_t ka[NB], kb[NB], da[NB / 2], db[NB / 2];
				const uint8_t *kp = st + (base + ja) * (HL / 2) + c * 4 * NB;
				lds_words<NB>(kp, ka);
				lds_words<NB>(kp + 8 * (HL / 2), kb);
				const uint8_t *ks = st + SL::kKS + (base + ja) * NB * 2;
				lds_words<NB / 2>(ks, da);
				lds_words<NB / 2>(ks + 8 * NB * 2, db);
#pragma unroll
				for (int b = 0; b < NB; b++) {
					const uint32_t lo[4] = {codes_low(ka[b]), codes_low(kb[b]),
								codes_low(ka[b] >> 8), codes_low(kb[b] >> 8)};
					const uint32_t hi[4] = {codes_high(ka[b]), codes_high(kb[b]),
								codes_high(ka[b] >> 8), codes_high(kb[b] >> 8)};
					const float dka = half_bits_to_float((uint16_t)(da[b / 2] >> (16 * (b & 1))));
					const float dkb = half_bits_to_float((uint16_t)(db[b / 2] >> (16 * (b & 1))));
#pragma unroll
					for (int nt = 0; nt < NT; nt++) {
						uint2 q0, q1;
						if constexpr (QR) {
							q0 = qf[nt * 2 * NB + 2 * b];
							q1 = qf[nt * 2 * NB + 2 * b + 1];
						} else {
							q0 = sm_q[nt * 2 * NB + 2 * b][lane];
							q1 = sm_q[nt * 2 * NB + 2 * b + 1][lane];
						}
						float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
						mma_step(d, lo, q0.x, q0.y);
						mma_step(d, hi, q1.x, q1.y);
						s[nt][0] = fmaf(dka, d[0], s[nt][0]);
						s[nt][1] = fmaf(dka, d[1], s[nt][1]);
						s[nt][2] = fmaf(dkb, d[2], s[nt][2]);
						s[nt][3] = fmaf(dkb, d[3], s[nt][3]);
					}
				}
			}
			// ---- V scales of this lane's two rows
			const int kra = k0 + base + ja, krb = kra + 8;
			float dva[NB], dvb[NB];
			{
				uint32_t wa[NB / 2], wb[NB / 2];
				const uint8_t *vs = st + SL::kVS + (base + ja) * NB * 2;
				lds_words<NB / 2>(vs, wa);
				lds_words<NB / 2>(vs + 8 * NB * 2, wb);
				if (!full) {
					// rows that no query of the tile sees hold anything
#pragma unroll
					for (int k = 0; k < NB / 2; k++) {
						wa[k] = kra < it.hi && kra >= it.lo ? wa[k] : 0;
						wb[k] = krb < it.hi && krb >= it.lo ? wb[k] : 0;
					}
				}
#pragma unroll
				for (int b = 0; b < NB; b++) {
					dva[b] = half_bits_to_float((uint16_t)(wa[b / 2] >> (16 * (b & 1))));
					dvb[b] = half_bits_to_float((uint16_t)(wb[b / 2] >> (16 * (b & 1))));
				}
			}
			bool grow = false;
#pragma unroll
			for (int b = 0; b < NB; b++)
				grow |= fmaxf(fabsf(dva[b]), fabsf(dvb[b])) * rv[b] > 2.0f;
			if (__any_sync(0xffffffffu, grow)) {
				// the largest V scale so far to [1, 2): a power of two
#pragma unroll
				for (int b = 0; b < NB; b++) {
					float v = fmaxf(fabsf(dva[b]), fabsf(dvb[b]));
					v = warp_max(v);
					if (v * rv[b] > 2.0f) {
						const float r = scalbnf(1.0f, -ilogbf(v));
						const float f = r / rv[b];
						rv[b] = r;
#pragma unroll
						for (int nt = 0; nt < NT; nt++)
#pragma unroll
							for (int k = 0; k < 4; k++) {
								o[2 * b][nt][k] *= f;
								o[2 * b + 1][nt][k] *= f;
							}
					}
				}
			}
#pragma unroll
			for (int b = 0; b < NB; b++) {
				dva[b] *= rv[b];
				dvb[b] *= rv[b];
			}
			// ---- weights
			float p[NT][4];
			bool seen[NT][4];
			bool lag = false;
#pragma unroll
			for (int nt = 0; nt < NT; nt++) {
				if (SPLIT) {
					s[nt][0] = (s[nt][0] + s[nt][1]) * qs0[nt];
					s[nt][2] = (s[nt][2] + s[nt][3]) * qs0[nt];
					s[nt][1] = s[nt][0];
					s[nt][3] = s[nt][2];
				} else {
					s[nt][0] *= qs0[nt];
					s[nt][1] *= qs1[nt];
					s[nt][2] *= qs0[nt];
					s[nt][3] *= qs1[nt];
				}
#pragma unroll
				for (int k = 0; k < 4; k++)
					seen[nt][k] = true;
				if (!full) {
					auto sees = [&](int j, int row) {
						return j < it.kv && (!a.causal || j <= row) &&
						       (!a.window || j > row - a.window);
					};
					seen[nt][0] = sees(kra, row0[nt]);
					seen[nt][2] = sees(krb, row0[nt]);
					seen[nt][1] = SPLIT ? seen[nt][0] : sees(kra, row1[nt]);
					seen[nt][3] = SPLIT ? seen[nt][2] : sees(krb, row1[nt]);
				}
				lag |= (seen[nt][0] && s[nt][0] > m0[nt] + kLag) ||
				       (seen[nt][2] && s[nt][2] > m0[nt] + kLag);
				if (!SPLIT)
					lag |= (seen[nt][1] && s[nt][1] > m1[nt] + kLag) ||
					       (seen[nt][3] && s[nt][3] > m1[nt] + kLag);
			}
			if (__any_sync(0xffffffffu, lag)) {
#pragma unroll
				for (int nt = 0; nt < NT; nt++) {
					float a0 = fmaxf(seen[nt][0] ? s[nt][0] : -3.0e38f,
							 seen[nt][2] ? s[nt][2] : -3.0e38f);
					float a1 = fmaxf(seen[nt][1] ? s[nt][1] : -3.0e38f,
							 seen[nt][3] ? s[nt][3] : -3.0e38f);
#pragma unroll
					for (int x = 4; x < 32; x *= 2) {
						a0 = fmaxf(a0, __shfl_xor_sync(0xffffffffu, a0, x));
						a1 = fmaxf(a1, __shfl_xor_sync(0xffffffffu, a1, x));
					}
					a0 = fmaxf(a0, m0[nt]);
					a1 = fmaxf(a1, m1[nt]);
					const float f0 = ex2(m0[nt] - a0), f1 = ex2(m1[nt] - a1);
					m0[nt] = a0;
					m1[nt] = a1;
					l0[nt] *= f0;
					l1[nt] *= f1;
#pragma unroll
					for (int k = 0; k < 2 * NB; k++) {
						o[k][nt][0] *= f0;
						o[k][nt][1] *= f1;
						o[k][nt][2] *= f0;
						o[k][nt][3] *= f1;
					}
				}
			}
#pragma unroll
			for (int nt = 0; nt < NT; nt++) {
				const float b0 = kLift - m0[nt], b1 = kLift - m1[nt];
				p[nt][0] = ex2(s[nt][0] + b0);
				p[nt][2] = ex2(s[nt][2] + b0);
				p[nt][1] = SPLIT ? p[nt][0] : ex2(s[nt][1] + b1);
				p[nt][3] = SPLIT ? p[nt][2] : ex2(s[nt][3] + b1);
				if (!full) {
#pragma unroll
					for (int k = 0; k < 4; k++)
						p[nt][k] = seen[nt][k] ? p[nt][k] : 0.0f;
				}
				l0[nt] += p[nt][0] + p[nt][2];
				l1[nt] += p[nt][1] + p[nt][3];
			}
			// ---- O += V^T P^T
			uint32_t v0[NB / 2], v1[NB / 2], v2[NB / 2], v3[NB / 2];
			const uint8_t *vp = st + SL::kVC + base * (HL / 2) + g * 2 * NB;
			lds_words<NB / 2>(vp + va * (HL / 2), v0);
			lds_words<NB / 2>(vp + vb * (HL / 2), v1);
			lds_words<NB / 2>(vp + (va + 8) * (HL / 2), v2);
			lds_words<NB / 2>(vp + (vb + 8) * (HL / 2), v3);
#pragma unroll
			for (int b = 0; b < NB; b++) {
				// bytes 2 g, 2 g + 1 of the block, of two rows each
				const uint32_t sel0 = b & 1 ? 0x0602 : 0x0400;
				const uint32_t sel1 = b & 1 ? 0x0703 : 0x0501;
				const uint32_t t0 = __byte_perm(v0[b / 2], v1[b / 2], sel0);
				const uint32_t t1 = __byte_perm(v0[b / 2], v1[b / 2], sel1);
				const uint32_t t2 = __byte_perm(v2[b / 2], v3[b / 2], sel0);
				const uint32_t t3 = __byte_perm(v2[b / 2], v3[b / 2], sel1);
				const uint32_t lo[4] = {codes_low(t0), codes_low(t1), codes_low(t2), codes_low(t3)};
				const uint32_t hi[4] = {codes_high(t0), codes_high(t1), codes_high(t2),
							codes_high(t3)};
#pragma unroll
				for (int nt = 0; nt < NT; nt++) {
					float w[4];
#pragma unroll
					for (int k = 0; k < 4; k++) {
						w[k] = p[nt][k] * (k < 2 ? dva[b] : dvb[b]);
						if (!full)   // a row unseen may hold a NaN scale
							w[k] = seen[nt][k] ? w[k] : 0.0f;
					}
					uint32_t b0, b1;
					if (SPLIT) {
						const float h0 = __half2float(__float2half_rn(w[0]));
						const float h1 = __half2float(__float2half_rn(w[2]));
						b0 = pack_h2(h0, w[0] - h0);
						b1 = pack_h2(h1, w[2] - h1);
					} else {
						b0 = pack_h2(w[0], w[1]);
						b1 = pack_h2(w[2], w[3]);
					}
					b0 = transpose8x8(b0);
					b1 = transpose8x8(b1);
					mma_step(o[2 * b][nt], lo, b0, b1);
					mma_step(o[2 * b + 1][nt], hi, b0, b1);
				}
			}
		}
		__syncwarp();   // every lane has read the stage
		const int next = i + kAttnStages;
		if ((next & 31) == 0 && next < ntile)
			load_pages(next);
		if (next < ntile)
			issue(next);
	}
	if (i < ntile) {
		// a wait ran out: the copies still in flight (each waited for once
		// more) must not land in memory that is used below
		if (lane == 0)
			atomicOr(a.b.err, kKvErrWait);
		for (int s = i; s < min(ntile, i + kAttnStages); s++)
			mbar_wait(bar + s % kAttnStages, (s / kAttnStages) & 1);
	}

	// ---- the warps' sums joined, over the ring's memory
#pragma unroll
	for (int nt = 0; nt < NT; nt++) {
#pragma unroll
		for (int x = 4; x < 32; x *= 2) {
			l0[nt] += __shfl_xor_sync(0xffffffffu, l0[nt], x);
			l1[nt] += __shfl_xor_sync(0xffffffffu, l1[nt], x);
		}
		if (g == 0) {
			sm_m[warp][nt * 8 + 2 * c] = m0[nt];
			sm_m[warp][nt * 8 + 2 * c + 1] = m1[nt];
			sm_l[warp][nt * 8 + 2 * c] = l0[nt];
			sm_l[warp][nt * 8 + 2 * c + 1] = l1[nt];
		}
	}
	__syncthreads();
	auto top_of = [&](int col) {
		float m = sm_m[0][col];
#pragma unroll
		for (int w = 1; w < kAttnWarps; w++)
			m = fmaxf(m, sm_m[w][col]);
		return m;
	};
	constexpr int OS = HL + 4;
	float *ob = reinterpret_cast<float *>(smem);
#pragma unroll
	for (int nt = 0; nt < NT; nt++) {
		const int col = nt * 8 + 2 * c;
		const float f0 = ex2(m0[nt] - top_of(col)), f1 = ex2(m1[nt] - top_of(col + 1));
		float *o0 = ob + (warp * COLS + col) * OS, *o1 = o0 + OS;
#pragma unroll
		for (int k = 0; k < 2 * NB; k++) {
			const float iv = 1.0f / rv[k / 2];
			const int e = 32 * (k / 2) + 16 * (k & 1) + 2 * g;
			*reinterpret_cast<float2 *>(o0 + e) =
				make_float2(o[k][nt][0] * f0 * iv, o[k][nt][2] * f0 * iv);
			*reinterpret_cast<float2 *>(o1 + e) =
				make_float2(o[k][nt][1] * f1 * iv, o[k][nt][3] * f1 * iv);
		}
	}
	__syncthreads();
	for (int i = threadIdx.x; i < it.rows * (HL / 4); i += kAttnThreads) {
		const int r = i / (HL / 4), e = i % (HL / 4) * 4;
		const int col = SPLIT ? r / RPN * 8 + 2 * (r % RPN) : r;
		const float m = top_of(col);
		float l = 0.0f;
		float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
		for (int w = 0; w < kAttnWarps; w++) {
			l += sm_l[w][col] * ex2(sm_m[w][col] - m);
#pragma unroll
			for (int h = 0; h < (SPLIT ? 2 : 1); h++) {
				const float4 x =
					*reinterpret_cast<const float4 *>(ob + (w * COLS + col + h) * OS + e);
				v.x += x.x;
				v.y += x.y;
				v.z += x.z;
				v.w += x.w;
			}
		}
		if (it.runs > 1) {
			float *pp = a.part + ((int64_t)blockIdx.x * RPT + r) * OS;
			*reinterpret_cast<float4 *>(pp + e) = v;
			if (e == 0)
				*reinterpret_cast<float2 *>(pp + HL) = make_float2(m, l);
		} else {
			write_row<T>(a, it, r, e, v, m, l, e == 0);
		}
	}
}

// one tile of query rows with several runs: their sums joined, a warp a row
template <typename T, int HL, int RPT>
__global__ void __launch_bounds__(kAttnThreads) kv_merge_kernel(AttnArgs a)
{
	constexpr int OS = HL + 4, E4 = HL / 4;   // float4s of a row
	Item it;
	const bool mine = find_item<RPT, false>(a, blockIdx.x, it) && it.runs > 1;
	griddep_wait();   // the runs are written
	if (!mine)
		return;
	const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
	const int64_t step = (int64_t)a.KVH * RPT * OS;   // between the runs of a tile
	for (int r = warp; r < it.rows; r += kAttnWarps) {
		const float *pp = a.part + ((int64_t)it.first * RPT + r) * OS;
		float m = -3.0e38f;
		for (int s = lane; s < it.runs; s += 32)
			m = fmaxf(m, pp[s * step + HL]);
		m = warp_max(m);
		float l = 0.0f;
		for (int s = lane; s < it.runs; s += 32)
			l += pp[s * step + HL + 1] * ex2(pp[s * step + HL] - m);
		l = warp_sum(l);
		for (int e = lane; e < E4; e += 32) {
			float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
			for (int s = 0; s < it.runs; s++) {
				const float f = ex2(pp[s * step + HL] - m);
				const float4 x = *reinterpret_cast<const float4 *>(pp + s * step + 4 * e);
				v.x = fmaf(x.x, f, v.x);
				v.y = fmaf(x.y, f, v.y);
				v.z = fmaf(x.z, f, v.z);
				v.w = fmaf(x.w, f, v.w);
			}
			write_row<T>(a, it, r, 4 * e, v, m, l, e == 0);
		}
	}
}

// ---------------------------------------------------------------- launches
// the sizes that a launch is planned with, from the call's bounds alone
struct Plan {
	int nt = 1, rpt = 8;     // column tiles, query rows of an item
	int64_t tiles = 0;       // at most so many query tiles x KV heads
	int64_t items = 0;       // and items
	int target = 0;
	bool split = false;      // runs at all
	size_t part_bytes = 0;
};

Plan plan_of(const moe_kv_cache *c, const moe_kv_batch *b, int64_t H, bool fp32)
{
	Plan p;
	const int64_t HL = c->d.head_len, KVH = c->d.n_kv_heads, G = H / KVH;
	const int64_t rows = b->max_q * G;   // query rows of a sequence's KV head
	const int per = fp32 ? 4 : 8;
	// as few columns as hold the rows; many rows: as many as registers hold
	p.nt = rows <= per ? 1 : rows <= 2 * per || HL == 256 ? 2 : 4;
	p.rpt = per * p.nt;
	const int64_t by_seq = b->n_seqs * ((rows + p.rpt - 1) / p.rpt);
	const int64_t by_token = b->n_tokens * G / p.rpt + b->n_seqs;
	p.tiles = KVH * (by_seq < by_token ? by_seq : by_token);
	p.target = 6 * sm_count();
	p.split = p.tiles < 4 * (int64_t)p.target;
	p.items = p.tiles;
	if (p.split) {
		const int64_t longest = (b->max_kv + kAttnTile - 1) / kAttnTile;
		const int64_t capped = p.tiles * longest / kRunMax + 1;
		p.items += capped > p.target ? capped : p.target;
		p.part_bytes = (size_t)(p.items * p.rpt * (HL + 4) * 4);
	}
	return p;
}

template <typename T, int HL, int NT>
cudaError_t launch_attn_as(const AttnArgs &a, const Plan &p, cudaStream_t st)
{
	constexpr int RPT = (sizeof(T) == 4 ? 4 : 8) * NT;
	constexpr int smem = attn_smem<HL, NT>();
	if (cudaError_t e = ensure_smem(kv_attn_kernel<T, HL, NT>, smem))
		return e;
	kv_attn_kernel<T, HL, NT><<<(unsigned)p.items, kAttnThreads, smem, st>>>(a);
	if (cudaError_t e = cudaGetLastError())
		return e;
	if (!p.split)
		return cudaSuccess;
	cudaLaunchConfig_t cfg{};
	cfg.gridDim = dim3((unsigned)p.tiles);
	cfg.blockDim = dim3(kAttnThreads);
	cfg.stream = st;
	cudaLaunchAttribute at[1];
	at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
	at[0].val.programmaticStreamSerializationAllowed = 1;
	cfg.attrs = at;
	cfg.numAttrs = pdl_enabled() ? 1 : 0;
	return cudaLaunchKernelEx(&cfg, kv_merge_kernel<T, HL, RPT>, a);
}

template <typename T>
cudaError_t launch_attn(const AttnArgs &a, const Plan &p, int HL, cudaStream_t st)
{
	if (HL == 64)
		return p.nt == 1 ? launch_attn_as<T, 64, 1>(a, p, st)
		       : p.nt == 2 ? launch_attn_as<T, 64, 2>(a, p, st)
				   : launch_attn_as<T, 64, 4>(a, p, st);
	if (HL == 128)
		return p.nt == 1 ? launch_attn_as<T, 128, 1>(a, p, st)
		       : p.nt == 2 ? launch_attn_as<T, 128, 2>(a, p, st)
				   : launch_attn_as<T, 128, 4>(a, p, st);
	return p.nt == 1 ? launch_attn_as<T, 256, 1>(a, p, st) : launch_attn_as<T, 256, 2>(a, p, st);
}

// what a call may ask of its workspace: the same for every row type
size_t workspace_of(const moe_kv_cache *c, const moe_kv_batch *b, int64_t H)
{
	const size_t x = plan_of(c, b, H, true).part_bytes, y = plan_of(c, b, H, false).part_bytes;
	return x > y ? x : y;
}

int check_heads(const char *what, const moe_kv_cache *c, int64_t n_heads)
{
	if (n_heads <= 0 || n_heads > 65535 || n_heads % c->d.n_kv_heads)
		return kv_fail(MOE_ERR_INVALID, "%s: %lld heads over %lld KV heads", what,
			       (long long)n_heads, (long long)c->d.n_kv_heads);
	return MOE_OK;
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

int64_t moe_kv_attention_workspace(const moe_kv_cache *cache, const moe_kv_batch *batch,
				   int64_t n_heads)
{
	const char *what = "moe_kv_attention_workspace";
	if (!cache)
		return kv_fail(MOE_ERR_INVALID, "%s: null cache", what);
	if (int rc = check_batch(what, cache, batch, false))
		return rc;
	if (int rc = check_heads(what, cache, n_heads))
		return rc;
	DeviceGuard g(cache->device);
	KV_CK(what, g.e);
	return (int64_t)workspace_of(cache, batch, n_heads);
}

int moe_kv_attention(moe_kv_cache *cache, const moe_kv_batch *batch, const moe_rows *q,
		     const moe_rows *out, float *lse, float scale, int causal, int64_t window,
		     void *workspace, size_t workspace_bytes, void *stream)
{
	const char *what = "moe_kv_attention";
	if (!cache)
		return kv_fail(MOE_ERR_INVALID, "%s: null cache", what);
	int rc = check_batch(what, cache, batch);
	if (rc != MOE_OK)
		return rc;
	if (!q || !out)
		return kv_fail(MOE_ERR_INVALID, "%s: q or out missing", what);
	const int64_t T = batch->n_tokens, D = cache->d.head_len, KVH = cache->d.n_kv_heads;
	rc = check_rows(what, "q", q, T, D, q->type, 0, false);
	if (rc == MOE_OK)
		rc = check_rows(what, "out", out, T, D, q->type, q->n_heads, true);
	if (rc == MOE_OK)
		rc = check_heads(what, cache, q->n_heads);
	if (rc != MOE_OK)
		return rc;
	if (!std::isfinite(scale))
		return kv_fail(MOE_ERR_INVALID, "%s: scale %g", what, (double)scale);
	if (window < 0 || window > (1 << 30) || (window && !causal))
		return kv_fail(MOE_ERR_INVALID, "%s: window %lld (causal %d)", what, (long long)window,
			       causal);
	if ((uintptr_t)lse % 4)
		return kv_fail(MOE_ERR_INVALID, "%s: lse is not aligned", what);
	if (T == 0 || batch->n_seqs == 0 || batch->max_q == 0)
		return MOE_OK;
	cudaStream_t st;
	if ((rc = resolve_stream(what, cache->device, stream, &st)) != MOE_OK)
		return rc;
	DeviceGuard g(cache->device);
	KV_CK(what, g.e);
	const Plan p = plan_of(cache, batch, q->n_heads, q->type == MOE_F32);
	if (p.items > 0x7fffffff || batch->max_q * (q->n_heads / KVH) > (1 << 30))
		return kv_fail(MOE_ERR_INVALID, "%s: batch too large", what);
	const size_t need = workspace_of(cache, batch, q->n_heads);
	if (need && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < need))
		return kv_fail(MOE_ERR_INVALID, "%s: workspace of %zu bytes, needs %zu (16-byte aligned)",
			       what, workspace ? workspace_bytes : 0, need);
	AttnArgs a;
	a.b = batch_args(cache, batch);
	a.q = q->data;
	a.out = out->data;
	a.q_ts = q->token_stride;
	a.q_hs = q->head_stride;
	a.o_ts = out->token_stride;
	a.o_hs = out->head_stride;
	a.lse = lse;
	a.pages = cache->pages;
	a.page_bytes = (int64_t)cache->page_bytes;
	a.H = (int)q->n_heads;
	a.KVH = (int)KVH;
	a.G = (int)(q->n_heads / KVH);
	a.causal = causal != 0;
	a.window = (int)window;
	a.scale2 = scale * 1.44269504088896f;
	a.q_vec = rows_vec16(q);
	a.o_vec = rows_vec16(out);
	a.target = p.split ? p.target : 0;
	a.items = p.items;
	a.part = static_cast<float *>(workspace);
	KV_CK(what, q->type == MOE_F32   ? launch_attn<float>(a, p, (int)D, st)
		    : q->type == MOE_F16 ? launch_attn<__half>(a, p, (int)D, st)
					 : launch_attn<__nv_bfloat16>(a, p, (int)D, st));
	return MOE_OK;
}

}  // extern "C"
