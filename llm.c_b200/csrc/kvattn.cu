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
// layout places a thread's nibbles of all blocks side by side, and a nibble is an
// fp16 number after one or two operations on a pair.  S^T comes out with a row per lane
// group and P^T wants a column per lane group: one movmatrix per 8 x 8 tile
// turns it.
//
// fp16 weights: p <= 16 (the running maximum may lag by 4, in exponents of 2;
// then nothing needs rescaling), times 2^10, times the row's V scale brought below
// 2 by a power of two per block (the block's largest so far to [1, 2), which leaves
// fp16's range to the others), so weights down to 2^-24 of the largest keep fp16's
// full precision where their block's V scale is near its largest.  A weight of 16-bit
// rows is rounded to fp16 and its product with the scale once more: 2^-10 in all,
// below what rounding the output to bf16 costs and twice fp16's; fp32 rows take two
// columns, the fp16 value of the fp32 product and the fp16 remainder.  q is brought
// to 2^13 by a power of two per row, so that fp16 holds 16-bit rows' values exactly
// unless they are below 2^-27 (those that meet high nibbles, which count 16-fold, 2^-23) of
// the row's largest, and is off by 2^-38 (2^-34) of it where not.
//
// Work: an item is a KV head of a sequence, a tile of its query rows (query
// token x head of the group) and a run of 32-row key tiles, and an item is a warp's:
// the 4 warps of a CTA share nothing, so nothing waits.  (4 warps that took an item's
// tiles in turn and joined their sums in shared memory: 47 us instead of 39 for 64
// sequences, 243 instead of 195 for a prompt.)  Sequences of
// many queries in 16 bits go to kvwide.cu.  The run's length is chosen on the
// device from the batch's lengths so that the items fill the GPU however ragged they
// are; a tile of queries with several runs is joined by a second kernel.
#include "kvattn.cuh"

#include <type_traits>

namespace moe {
using namespace kva;
namespace {

constexpr int kAttnWarps = 4, kAttnThreads = 32 * kAttnWarps;
constexpr int kWideMin = kWideRows;   // query rows of a sequence's KV head for kvwide.cu's kernel
constexpr int kAttnStages = 2;     // copies in a warp's ring (3: 39.4 us for 64 sequences, 36.7 with 2)
__device__ __forceinline__ void mma_step(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
					 uint32_t b1)
{
	asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
		     "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
		     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
		     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// the same from a sum of zero
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
					  uint32_t b1)
{
	asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
		     "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
		     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
		     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

// and from sums of the columns' own
__device__ __forceinline__ void mma_from(float (&d)[4], float2 c, const uint32_t (&a)[4], uint32_t b0,
					 uint32_t b1)
{
	asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
		     "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
		     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
		     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c.x), "f"(c.y));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x)
{
	uint32_t y;
	asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
	return y;
}

// half `at` of a word, twice
__device__ __forceinline__ __half2 both(__half2 h, int at)
{
	return at ? __high2half2(h) : __low2half2(h);
}

__device__ __forceinline__ uint32_t smem_addr(const void *p)
{
	return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// Codes as fp16 numbers (the method of adding a code to the bits of a power of two is published:
// Kim et al. 2022, arXiv 2211.10017), a pair from a word's low nibbles (bytes 0 and 2) or high ones.
// 16-bit rows: masked out in place, subnormals code * 2^-24 and code * 2^-20, for one
// logic operation; the -8 of a code is the caller's (RAW) or one exact subtraction more.
// The tensor cores line sums up by a subnormal's nominal exponent, so these sums carry
// about 17 bits, 2^-6 of what rounding the weights costs.  fp32 rows (with subnormals
// 8.4e-6 off, 4.7e-7 so): code - 8 itself (EXACT), from 1024 + code or 1024 + 16 code; for
// all rows that takes 134 us instead of 124 for 4 sequences of 131072 rows, without RAW
// 144.
template <bool RAW, bool EXACT>
__device__ __forceinline__ uint32_t codes_low(uint32_t w)
{
	static_assert(!(RAW && EXACT), "one or the other");
	const uint32_t x = w & 0x000f000fu;
	if (EXACT)
		return h2_bits(__hsub2(bits_h2(x | 0x64006400u), bits_h2(0x64086408u)));
	return RAW ? x : h2_bits(__hsub2(bits_h2(x), bits_h2(0x00080008u)));
}
template <bool RAW, bool EXACT>
__device__ __forceinline__ uint32_t codes_high(uint32_t w)
{
	const uint32_t x = w & 0x00f000f0u;
	if (EXACT)
		return h2_bits(__hfma2(bits_h2(x | 0x64006400u), bits_h2(0x2c002c00u),   // / 16
				       bits_h2(0xd480d480u)));                           // - 72
	return RAW ? x : h2_bits(__hsub2(bits_h2(x), bits_h2(0x00800080u)));
}
constexpr float kCodeUnit = 16777216.0f;   // 2^24: low nibbles as subnormals

// The tile row that stands as row j of A (of 8): any order will do that K and V, and
// so S^T and P^T, share.  This one lets the 8 rows that a shared-memory read takes
// together begin in banks of their own.
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

template <int HL>
struct StageLayout {
	static constexpr int NB = HL / 32;
	static constexpr int kCodes = kAttnTile * HL / 2, kScales = kAttnTile * NB * 2;
	static constexpr int kKS = kCodes, kVC = kCodes + kScales, kVS = 2 * kCodes + kScales;
	static constexpr int kBytes = 2 * (kCodes + kScales);
};

template <int HL>
constexpr int kAttnSmem = kAttnWarps * kAttnStages * StageLayout<HL>::kBytes;

// queries as operands in registers, or in shared memory where there are more of them
// than registers (128 a lane at HL * NT = 512)
template <int HL, int NT>
constexpr bool kQInRegs = HL * NT <= 256;

// CTAs of an SM that the registers are cut for: 4 where 128 a lane do (HL 128, one
// column tile: 4 sequences of 131072 rows 126 us, left to itself 141; 3: 143).
template <int HL, int NT>
constexpr int kAttnCtas = HL == 128 && NT == 1 ? 4 : 1;

// grid: the plan's items, kAttnWarps to a CTA.  Few queries (4 sequences of 131072 rows,
// 32 heads on 8: 526 MB in 124 us, 4.25 TB/s of 6.5) are bound by chains
// of dependent instructions that take codes apart (issue 63 %, ALU 55 %, 14 warps an SM), a batch
// of 64 such sequences of up to 8192 rows (72 MB in 37 us) by latency: a few tiles a warp
// between its plan and its last store.  (Times from CUDA graphs of calls; one call at a time
// takes 2 to 3 us more.)
template <typename T, int HL, int NT, bool FOLD>
__global__ void __launch_bounds__(kAttnThreads, kAttnCtas<HL, NT>) kv_attn_kernel(AttnArgs a)
{
	constexpr bool SPLIT = sizeof(T) == 4;        // two columns a row
	constexpr int RPN = SPLIT ? 4 : 8;            // rows of an 8-column tile
	constexpr int RPT = RPN * NT, NB = HL / 32;
	constexpr bool QR = kQInRegs<HL, NT>;
	// 16-bit rows, one column tile: the keys' -8 sum to -8 sum q, where the scores' sums
	// start
	constexpr bool KRAW = NT == 1 && !SPLIT;
	constexpr float unit = SPLIT ? 1.0f : kCodeUnit, high_unit = SPLIT ? 1.0f : 0.0625f;   // of low nibbles; high ones count 16-fold
	using SL = StageLayout<HL>;
	extern __shared__ __align__(128) uint8_t smem[];
	__shared__ uint2 sm_q[kAttnWarps][QR ? 1 : 2 * NB * NT][32];
	const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, c = lane % 4;

	griddep_launch_dependents();
	Item it;
	const int item = blockIdx.x * kAttnWarps + warp;
	if (!find_item<RPT, true>(a, item, it))
		return;

	// ---- the key tiles t0, t0 + 1, ..: lane l keeps the pages of the next 32 of
	// them (two where a page is half a tile)
	const int ntile = it.t1 - it.t0;
	const int32_t *table = a.b.table + it.b * a.b.table_stride;
	const int P = 1 << a.b.page_log2;
	const bool small = P < kAttnTile;
	uint8_t *ring = smem + warp * kAttnStages * SL::kBytes;
	auto key0 = [&](int i) { return (it.t0 + i) * kAttnTile; };
	// which halves of tile i hold rows that the query tile sees
	auto needs = [&](int k0) -> int {
		return (k0 < it.hi && k0 + 16 > it.lo ? 1 : 0) |
		       (k0 + 16 < it.hi && k0 + 32 > it.lo ? 2 : 0);
	};
	int page_a = -1, page_b = -1;   // of tile (i & ~31) + lane
	auto load_pages = [&](int i) {
		page_a = page_b = -1;
		if (i + lane < ntile) {
			const int k0 = key0(i + lane), need = needs(k0);
			const bool wa = need & (small ? 1 : 3), wb = small && (need & 2);
			if (wa)
				page_a = table[k0 >> a.b.page_log2];
			if (wb)
				page_b = table[(k0 + 16) >> a.b.page_log2];
			const bool ba = (unsigned)page_a >= (unsigned)a.b.n_pages;
			const bool bb = (unsigned)page_b >= (unsigned)a.b.n_pages;
			if ((wa && ba) || (wb && bb))
				atomicOr(a.b.err, kKvErrPage);
			page_a = ba ? -1 : page_a;
			page_b = bb ? -1 : page_b;
		}
	};
	const int half_rec = (HL / 2 + HL / 16) << a.b.page_log2;
	const uint8_t *head_pages = a.pages + 2 * (int64_t)it.kvh * half_rec;
	// this lane's 16 bytes of every 512 of a tile's codes; of its scales, K's
	// and V's side by side over the lanes
	constexpr int CH = SL::kCodes / 512, SLN = SL::kScales / 16, SCH = (2 * SLN + 31) / 32;
	const uint32_t ring_at = smem_addr(ring) + lane * 16;
	const uint8_t *codes_at = head_pages + lane * 16;
	const uint8_t *scales_at = head_pages + ((HL / 2) << a.b.page_log2) +
				   (lane < SLN ? lane * 16 : half_rec + (lane - SLN) * 16);
	const uint32_t to_scales = smem_addr(ring) + (lane < SLN ? SL::kKS + lane * 16
								 : SL::kVS + (lane - SLN) * 16);
	unsigned ring_have = 0;   // 2 bits a stage: the halves in it
	auto issue = [&](int i, int stage) {
		const int k0 = key0(i);
		const int pa = __shfl_sync(0xffffffffu, page_a, i & 31);
		if (!small && SCH == 1 && k0 >= it.lo && k0 + 16 < it.hi && pa >= 0) {
			// both halves, of one page
			const int r = k0 & (P - 1);
			const int64_t at = pa * a.page_bytes;
			const uint8_t *p = codes_at + at + r * (HL / 2), *v = p + half_rec;
			const uint32_t st = ring_at + stage * SL::kBytes;
#pragma unroll
			for (int q = 0; q < CH; q++) {
				copy16(st + 512 * q, p + 512 * q);
				copy16(st + SL::kVC + 512 * q, v + 512 * q);
			}
			if (lane < 2 * SLN)
				copy16(to_scales + stage * SL::kBytes, scales_at + at + r * NB * 2);
			ring_have |= 3u << 2 * stage;
			return;
		}
		int pb = pa;
		if (small)
			pb = __shfl_sync(0xffffffffu, page_b, i & 31);
		// pages outside the cache are not read: their rows count as unseen
		const int have = needs(k0) & ((pa >= 0 ? 1 : 0) | (pb >= 0 ? 2 : 0));
		ring_have = (ring_have & ~(3u << 2 * stage)) | (unsigned)have << 2 * stage;
		const uint32_t st = ring_at + stage * SL::kBytes;
		const int r = k0 & (P - 1);
		const uint8_t *src = head_pages + pa * a.page_bytes + r * (HL / 2) + lane * 16;
		// the second half's rows: 16 further on, or another page's first
		const uint8_t *src2 = small ? head_pages + pb * a.page_bytes + lane * 16 - 16 * (HL / 2) : src;
#pragma unroll
		for (int q = 0; q < CH; q++) {
			const uint8_t *p = (q < CH / 2 ? src : src2) + 512 * q;
			if (have >> (q < CH / 2 ? 0 : 1) & 1) {
				copy16(st + 512 * q, p);
				copy16(st + SL::kVC + 512 * q, p + half_rec);
			}
		}
#pragma unroll
		for (int q = 0; q < SCH; q++) {
			const int j = lane + 32 * q, isv = j >= SLN, jj = isv ? j - SLN : j;
			const int h = jj * 2 >= SLN;
			if (j < 2 * SLN && (have >> h & 1)) {
				const int row = small && h ? -16 : r;
				const uint8_t *p = head_pages + (small && h ? pb : pa) * a.page_bytes +
						   (((HL / 2) << a.b.page_log2) + (isv ? half_rec : 0) +
						    row * NB * 2 + jj * 16);
				copy16(st - lane * 16 + (isv ? SL::kVS : SL::kKS) + jj * 16, p);
			}
		}
	};
	load_pages(0);
#pragma unroll
	for (int i = 0; i < kAttnStages - 1; i++) {
		if (i < ntile)
			issue(i, i);
		copies_commit();
	}

	// ---- the queries: column n = g of every 8-column tile, values 4 c .. of
	// each half block, as B fragments
	uint2 qf[QR ? 2 * NB * NT : 1];
	float2 q_off[KRAW ? NB : 1];
	const T *qp = static_cast<const T *>(a.q) + (int64_t)it.kvh * a.G * a.q_hs;
	// factors of the lane's columns 2 c, 2 c + 1 of each tile
	float qs0[NT], qs1[NT];
#pragma unroll
	for (int nt = 0; nt < NT; nt++) {
		const int r = nt * RPN + (SPLIT ? g / 2 : g);
		float x[HL / 4];
		if (r < it.rows) {
			const int qr = it.r0 + r;
			const int i = a.by_g.div(qr);
			const T *p = qp + (it.s0 + i) * a.q_ts + (qr - i * a.G) * a.q_hs;
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
		// the largest magnitude, by its bits: an infinity or a NaN is above all
		uint32_t bits = 0;
#pragma unroll
		for (int k = 0; k < HL / 4; k++)
			bits = max(bits, __float_as_uint(x[k]) & 0x7fffffffu);
		bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 1));
		bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 2));
		const float top = __uint_as_float(bits);
		const bool bad = bits >= 0x7f800000u;
		const int e = top == 0.0f || bad ? 0 : 13 - ilogbf(top);   // -114 .. 162
		const float up = __int_as_float((127 + min(e, 127)) << 23);
		if (e > 127) {
#pragma unroll
			for (int k = 0; k < HL / 4; k++)
				x[k] *= __int_as_float((e - 127 + 127) << 23);
		}
		// a query with an infinity or a NaN has no finite scores: NaN
		const float qs = bad ? __int_as_float(0x7fffffff) : scalbnf(a.scale2 * unit, -e);
#pragma unroll
		for (int k = 0; k < HL / 4; k++) {
			const float v = bad ? 0.0f : x[k] * up;
			const float hi = __half2float(__float2half_rn(v));
			x[k] = SPLIT && (g & 1) ? v - hi : hi;
		}
		if constexpr (KRAW) {
			// -8 sum of the column's values of each block, as rounded
#pragma unroll
			for (int b = 0; b < NB; b++) {
				float t = 0.0f;
#pragma unroll
				for (int k = 0; k < 8; k++)
					t += SPLIT ? __half2float(__float2half_rn(x[8 * b + k])) : x[8 * b + k];
				t += __shfl_xor_sync(0xffffffffu, t, 1);
				t += __shfl_xor_sync(0xffffffffu, t, 2);
				t *= -8.0f / kCodeUnit;
				q_off[b] = make_float2(__shfl_sync(0xffffffffu, t, 8 * c),
						       __shfl_sync(0xffffffffu, t, 8 * c + 4));
			}
		}
#pragma unroll
		for (int h = 0; h < HL / 16; h++) {
			const float u = h & 1 ? high_unit : 1.0f;
			const uint2 f = make_uint2(pack_h2(x[4 * h] * u, x[4 * h + 2] * u),
						   pack_h2(x[4 * h + 1] * u, x[4 * h + 3] * u));
			if constexpr (QR)
				qf[nt * 2 * NB + h] = f;
			else
				sm_q[warp][nt * 2 * NB + h][lane] = f;   // the lane's own
		}
		qs0[nt] = __shfl_sync(0xffffffffu, qs, 8 * c);
		qs1[nt] = __shfl_sync(0xffffffffu, qs, 8 * c + 4);
	}
	// the cache row at which each column's query stands
	auto row_of = [&](int r) { return it.kv - it.n + a.by_g.div(it.r0 + r); };
	auto row0 = [&](int nt) { return row_of(nt * RPN + (SPLIT ? c : 2 * c)); };
	auto row1 = [&](int nt) { return row_of(nt * RPN + (SPLIT ? c : 2 * c + 1)); };
	const int first_row = row_of(0), last_row = row_of(it.rows - 1);

	// running sums of columns 2 c (0) and 2 c + 1 (1): o and l relative to the
	// largest score m so far, kept as b = kLift - m
	float o[2 * NB][NT][4];
	float b0[NT], b1[NT], l0[NT], l1[NT];
#pragma unroll
	for (int i = 0; i < 2 * NB; i++)
#pragma unroll
		for (int nt = 0; nt < NT; nt++)
#pragma unroll
			for (int k = 0; k < 4; k++)
				o[i][nt][k] = 0.0f;
#pragma unroll
	for (int nt = 0; nt < NT; nt++) {
		b0[nt] = b1[nt] = kNoMax;
		l0[nt] = l1[nt] = 0.0f;
	}
	// the V scales' factors, a power of two for each block, two to a word, and
	// the largest scales that they hold in range (2 over the factor)
	uint32_t v_fac[NB / 2], v_top[NB / 2];
#pragma unroll
	for (int k = 0; k < NB / 2; k++) {
		v_fac[k] = 0x78007800u;   // 2^15
		v_top[k] = 0x04000400u;   // 2^-14
	}
	// scores up to a0, a1 (in exponents of 2) seen
	auto raise = [&](int nt, float a0, float a1) {
		const float n0 = fminf(b0[nt], kLift - a0), n1 = fminf(b1[nt], kLift - a1);
		const float f0 = ex2(n0 - b0[nt]), f1 = ex2(n1 - b1[nt]);
		b0[nt] = n0;
		b1[nt] = n1;
		l0[nt] *= f0;
		l1[nt] *= f1;
#pragma unroll
		for (int k = 0; k < 2 * NB; k++) {
			o[k][nt][0] *= f0;
			o[k][nt][1] *= f1;
			o[k][nt][2] *= f0;
			o[k][nt][3] *= f1;
		}
	};

	const int ja = tile_row(g);                                  // A's rows g and g + 8
	const int va = tile_row(2 * c), vb = tile_row(2 * c + 1);    // A's columns 2 c ..
	// 16 rows of a tile (FULL: every query of the item sees them all)
	auto rows16 = [&](auto full_c, const uint8_t *st, int base, int k0) {
		constexpr bool FULL = decltype(full_c)::value;
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
				const uint32_t lo[4] = {codes_low<KRAW, SPLIT>(ka[b]), codes_low<KRAW, SPLIT>(kb[b]),
							codes_low<KRAW, SPLIT>(ka[b] >> 8), codes_low<KRAW, SPLIT>(kb[b] >> 8)};
				const uint32_t hi[4] = {codes_high<KRAW, SPLIT>(ka[b]), codes_high<KRAW, SPLIT>(kb[b]),
							codes_high<KRAW, SPLIT>(ka[b] >> 8),
							codes_high<KRAW, SPLIT>(kb[b] >> 8)};
				const float dka = half_of(da[b / 2], b & 1), dkb = half_of(db[b / 2], b & 1);
#pragma unroll
				for (int nt = 0; nt < NT; nt++) {
					uint2 q0, q1;
					if constexpr (QR) {
						q0 = qf[nt * 2 * NB + 2 * b];
						q1 = qf[nt * 2 * NB + 2 * b + 1];
					} else {
						q0 = sm_q[warp][nt * 2 * NB + 2 * b][lane];
						q1 = sm_q[warp][nt * 2 * NB + 2 * b + 1][lane];
					}
					float d[4];
					if constexpr (KRAW)
						mma_from(d, q_off[b], lo, q0.x, q0.y);
					else
						mma_first(d, lo, q0.x, q0.y);
					mma_step(d, hi, q1.x, q1.y);
					s[nt][0] = fmaf(dka, d[0], s[nt][0]);
					s[nt][1] = fmaf(dka, d[1], s[nt][1]);
					s[nt][2] = fmaf(dkb, d[2], s[nt][2]);
					s[nt][3] = fmaf(dkb, d[3], s[nt][3]);
				}
			}
		}
		// ---- weights, times 2^kLift over the largest so far
		const int kra = k0 + base + ja, krb = kra + 8;
		float p[NT][4];
		bool seen[NT][4], lag = false;
#pragma unroll
		for (int nt = 0; nt < NT; nt++) {
			if (SPLIT) {
				s[nt][0] += s[nt][1];
				s[nt][2] += s[nt][3];
			}
			p[nt][0] = fmaf(s[nt][0], qs0[nt], b0[nt]);
			p[nt][2] = fmaf(s[nt][2], qs0[nt], b0[nt]);
			p[nt][1] = SPLIT ? p[nt][0] : fmaf(s[nt][1], qs1[nt], b1[nt]);
			p[nt][3] = SPLIT ? p[nt][2] : fmaf(s[nt][3], qs1[nt], b1[nt]);
			if (!FULL) {
				auto sees = [&](int j, int row) {
					return j < it.kv && (!a.causal || j <= row) &&
					       (!a.window || j > row - a.window);
				};
				seen[nt][0] = sees(kra, row0(nt));
				seen[nt][2] = sees(krb, row0(nt));
				seen[nt][1] = SPLIT ? seen[nt][0] : sees(kra, row1(nt));
				seen[nt][3] = SPLIT ? seen[nt][2] : sees(krb, row1(nt));
			}
#pragma unroll
			for (int k = 0; k < 4; k += SPLIT ? 2 : 1)
				lag |= (FULL || seen[nt][k]) && p[nt][k] > kLift + kLag;
		}
		if (__any_sync(0xffffffffu, lag)) {
#pragma unroll
			for (int nt = 0; nt < NT; nt++) {
				float t[4];
#pragma unroll
				for (int k = 0; k < 4; k++) {
					const bool first = SPLIT || k % 2 == 0;
					t[k] = s[nt][SPLIT ? k & 2 : k] * (first ? qs0[nt] : qs1[nt]);
					if (!FULL)
						t[k] = seen[nt][k] ? t[k] : -kNoMax;
				}
				float a0 = fmaxf(t[0], t[2]), a1 = fmaxf(t[1], t[3]);
#pragma unroll
				for (int x = 4; x < 32; x *= 2) {
					a0 = fmaxf(a0, __shfl_xor_sync(0xffffffffu, a0, x));
					a1 = fmaxf(a1, __shfl_xor_sync(0xffffffffu, a1, x));
				}
				raise(nt, a0, a1);
				p[nt][0] = fmaf(s[nt][0], qs0[nt], b0[nt]);
				p[nt][2] = fmaf(s[nt][2], qs0[nt], b0[nt]);
				p[nt][1] = SPLIT ? p[nt][0] : fmaf(s[nt][1], qs1[nt], b1[nt]);
				p[nt][3] = SPLIT ? p[nt][2] : fmaf(s[nt][3], qs1[nt], b1[nt]);
			}
		}
#pragma unroll
		for (int nt = 0; nt < NT; nt++) {
			p[nt][0] = ex2(p[nt][0]);
			p[nt][2] = ex2(p[nt][2]);
			p[nt][1] = SPLIT ? p[nt][0] : ex2(p[nt][1]);
			p[nt][3] = SPLIT ? p[nt][2] : ex2(p[nt][3]);
			if (!FULL) {
#pragma unroll
				for (int k = 0; k < 4; k++)
					p[nt][k] = seen[nt][k] ? p[nt][k] : 0.0f;
			}
			l0[nt] += p[nt][0] + p[nt][2];
			if (!SPLIT)
				l1[nt] += p[nt][1] + p[nt][3];
		}
		// ---- O += V^T P^T
		uint32_t wa[NB / 2], wb[NB / 2];
		const uint8_t *vs = st + SL::kVS + (base + ja) * NB * 2;
		lds_words<NB / 2>(vs, wa);
		lds_words<NB / 2>(vs + 8 * NB * 2, wb);
#pragma unroll
		for (int k = 0; k < NB / 2; k++) {
			wa[k] = h2_bits(__hmul2(bits_h2(wa[k]), bits_h2(v_fac[k])));
			wb[k] = h2_bits(__hmul2(bits_h2(wb[k]), bits_h2(v_fac[k])));
		}
		uint32_t p2[NT][2], keep[NT][2];   // 16-bit rows: two columns' weights, and what of them is seen
#pragma unroll
		for (int nt = 0; nt < NT; nt++) {
			if (SPLIT)
				continue;
			p2[nt][0] = pack_h2(p[nt][0], p[nt][1]);
			p2[nt][1] = pack_h2(p[nt][2], p[nt][3]);
			if (!FULL) {
				keep[nt][0] = (seen[nt][0] ? 0xffffu : 0) | (seen[nt][1] ? 0xffff0000u : 0);
				keep[nt][1] = (seen[nt][2] ? 0xffffu : 0) | (seen[nt][3] ? 0xffff0000u : 0);
			}
		}
		uint32_t v0[NB / 2], v1[NB / 2], v2[NB / 2], v3[NB / 2];
		const uint8_t *vp = st + SL::kVC + base * (HL / 2) + g * 2 * NB;
		lds_words<NB / 2>(vp + va * (HL / 2), v0);
		lds_words<NB / 2>(vp + vb * (HL / 2), v1);
		lds_words<NB / 2>(vp + (va + 8) * (HL / 2), v2);
		lds_words<NB / 2>(vp + (vb + 8) * (HL / 2), v3);
#pragma unroll
		for (int b = 0; b < NB; b++) {
			// bytes 2 g, 2 g + 1 of the block, of two rows each
			const uint32_t sel0 = b & 1 ? 0x0602 : 0x0400, sel1 = b & 1 ? 0x0703 : 0x0501;
			const uint32_t t0 = __byte_perm(v0[b / 2], v1[b / 2], sel0);
			const uint32_t t1 = __byte_perm(v0[b / 2], v1[b / 2], sel1);
			const uint32_t t2 = __byte_perm(v2[b / 2], v3[b / 2], sel0);
			const uint32_t t3 = __byte_perm(v2[b / 2], v3[b / 2], sel1);
			const uint32_t lo[4] = {codes_low<false, SPLIT>(t0), codes_low<false, SPLIT>(t1), codes_low<false, SPLIT>(t2),
						codes_low<false, SPLIT>(t3)};
			const uint32_t hi[4] = {codes_high<false, SPLIT>(t0), codes_high<false, SPLIT>(t1),
						codes_high<false, SPLIT>(t2), codes_high<false, SPLIT>(t3)};
			// the rows' weights of this block
			const __half2 da = both(bits_h2(wa[b / 2]), b & 1), db = both(bits_h2(wb[b / 2]), b & 1);
#pragma unroll
			for (int nt = 0; nt < NT; nt++) {
				uint32_t x0, x1;
				if (SPLIT) {
					float w0 = p[nt][0] * __low2float(da), w1 = p[nt][2] * __low2float(db);
					if (!FULL) {   // a row unseen may hold a NaN scale
						w0 = seen[nt][0] ? w0 : 0.0f;
						w1 = seen[nt][2] ? w1 : 0.0f;
					}
					const float h0 = __half2float(__float2half_rn(w0));
					const float h1 = __half2float(__float2half_rn(w1));
					x0 = pack_h2(h0, w0 - h0);
					x1 = pack_h2(h1, w1 - h1);
				} else {
					x0 = h2_bits(__hmul2(bits_h2(p2[nt][0]), da));
					x1 = h2_bits(__hmul2(bits_h2(p2[nt][1]), db));
					if (!FULL) {
						x0 &= keep[nt][0];
						x1 &= keep[nt][1];
					}
				}
				x0 = transpose8x8(x0);
				x1 = transpose8x8(x1);
				mma_step(o[2 * b][nt], lo, x0, x1);
				mma_step(o[2 * b + 1][nt], hi, x0, x1);
			}
		}
	};

	// rows that every query of the item sees
	const int all_lo = a.window ? max(it.lo, last_row - a.window + 1) : it.lo;
	const int all_hi = a.causal ? min(it.kv, first_row + 1) : it.kv;
	int stage = 0;
	auto tile_at = [&](int i) {
		copies_wait<kAttnStages - 2>();
		__syncwarp();   // every lane's copies are in, and the stage before is read
		{
			const int next = i + kAttnStages - 1;
			if ((next & 31) == 0)
				load_pages(next);
			if (next < ntile)
				issue(next, stage == 0 ? kAttnStages - 1 : stage - 1);
			copies_commit();
		}
		const uint8_t *st = ring + stage * SL::kBytes;
		const int have = ring_have >> (2 * stage) & 3;
		const int k0 = key0(i);
		const bool full = have == 3 && k0 >= all_lo && k0 + kAttnTile <= all_hi;
		// ---- the V scales' range: lane = row (rows not in the ring, or that
		// no query sees, may hold anything)
		{
			uint32_t w[NB / 2];
			lds_words<NB / 2>(st + SL::kVS + lane * NB * 2, w);
			const bool use = full || ((have >> (lane / 16) & 1) && k0 + lane >= it.lo &&
						  k0 + lane < it.hi);
			bool grow = false;
#pragma unroll
			for (int k = 0; k < NB / 2; k++)
				grow |= !__hble2(__habs2(bits_h2(w[k])), bits_h2(v_top[k]));
			if (__any_sync(0xffffffffu, grow && use)) {
				// the largest so far to [1, 2): a power of two from 2^15 down
#pragma unroll
				for (int b = 0; b < NB; b++) {
					const float v = warp_max(use ? fabsf(half_of(w[b / 2], b & 1)) : 0.0f);
					const float had = half_of(v_fac[b / 2], b & 1);
					if (v * had > 2.0f) {
						const float r = scalbnf(1.0f, -min(ilogbf(v), 15));
						const float f = r / had;
						v_fac[b / 2] = set_half(v_fac[b / 2], b & 1, r);
						v_top[b / 2] = set_half(v_top[b / 2], b & 1, 2.0f / r);
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
		}
		if (full) {
#pragma unroll 1
			for (int u = 0; u < 2; u++)
				rows16(std::true_type{}, st, 16 * u, k0);
		} else {
#pragma unroll 1
			for (int u = 0; u < 2; u++)
				if (have >> u & 1)
					rows16(std::false_type{}, st, 16 * u, k0);
		}
		stage = stage + 1 == kAttnStages ? 0 : stage + 1;
	};

	// ---- out of the registers: a lane has values 2 g, 2 g + 1 of every half block
	// of its columns' rows, 8 lanes 16 values side by side.  To the item's record, on top of
	// what is there (!first), or (last, no other runs) to the results
	constexpr int OS = HL + 4;
	auto leave = [&](bool first, bool last) {
		float iv[NB];   // sums in true size: the codes' unit, the V scales' factors
#pragma unroll
		for (int b = 0; b < NB; b++)
			iv[b] = unit / half_of(v_fac[b / 2], b & 1);
#pragma unroll
		for (int nt = 0; nt < NT; nt++) {
#pragma unroll
			for (int x = 4; x < 32; x *= 2) {
				l0[nt] += __shfl_xor_sync(0xffffffffu, l0[nt], x);
				if (!SPLIT)
					l1[nt] += __shfl_xor_sync(0xffffffffu, l1[nt], x);
			}
#pragma unroll
			for (int h = 0; h < (SPLIT ? 1 : 2); h++) {   // the columns' rows: one, or two
				const int r = nt * RPN + (SPLIT ? c : 2 * c + h);
				const float bias = h ? b1[nt] : b0[nt];
				float l = h ? l1[nt] : l0[nt], f = 0.0f;
				float *pp = a.part + ((int64_t)item * a.part_rows + r) * OS;
				if (!first) {
					if (r < it.rows) {
						f = ex2(bias - pp[HL]);   // (the maximum only rises)
						l = fmaf(pp[HL + 1], f, l);
					}
					__syncwarp();   // read by all before one writes it
				}
				if (r >= it.rows)
					continue;
				auto value = [&](int k, int i) {   // i: the first or second of the two
					const float v = SPLIT ? o[k][nt][2 * i] + o[k][nt][2 * i + 1] : o[k][nt][2 * i + h];
					return v * (k & 1 ? iv[k / 2] * high_unit : iv[k / 2]);
				};
				auto two = [&](int k) {
					float2 v = make_float2(value(k, 0), value(k, 1));
					if (!first) {
						const float2 w = *reinterpret_cast<const float2 *>(pp + 16 * k + 2 * g);
						v = make_float2(fmaf(w.x, f, v.x), fmaf(w.y, f, v.y));
					}
					return v;
				};
				if (!last || it.runs > 1) {
#pragma unroll
					for (int k = 0; k < 2 * NB; k++)
						*reinterpret_cast<float2 *>(pp + 16 * k + 2 * g) = two(k);
					if (g == 0)
						*reinterpret_cast<float2 *>(pp + HL) = make_float2(bias, l);
				} else {
					const RowOut<T> out(a, it, r, bias, l);
#pragma unroll
					for (int k = 0; k < 2 * NB; k++) {
						const float2 v = two(k);
						out.two(16 * k + 2 * g, v.x, v.y);
					}
					if (g == 0)
						out.lse();
				}
			}
		}
	};
	for (int i0 = 0;;) {
		const int i1 = FOLD ? min(i0 + kFold, ntile) : ntile;
		for (int i = i0; i < i1; i++)
			tile_at(i);
		leave(!FOLD || i0 == 0, !FOLD || i1 == ntile);
		if (!FOLD || i1 == ntile)
			break;
		i0 = i1;
#pragma unroll
		for (int nt = 0; nt < NT; nt++) {
			l0[nt] = l1[nt] = 0.0f;
#pragma unroll
			for (int k = 0; k < 2 * NB; k++)
#pragma unroll
				for (int x = 0; x < 4; x++)
					o[k][nt][x] = 0.0f;
		}
		__syncwarp();   // the record, before it is read
	}
	copies_wait<0>();
}

// ---------------------------------------------------------------- launches
// `rows` is the most query rows of a sequence's KV head, p.rpt an item's and `wave` the
// items that a GPU has at a time
void plan_items(Plan &p, const moe_kv_cache *c, const moe_kv_batch *b, int64_t G, int64_t rows,
		int64_t wave)
{
	const int64_t KVH = c->d.n_kv_heads;
	const int64_t by_seq = b->n_seqs * ((rows + p.rpt - 1) / p.rpt);
	const int64_t by_token = b->n_tokens * G / p.rpt + b->n_seqs;
	p.tiles = KVH * (by_seq < by_token ? by_seq : by_token);
	p.rows = (int)(rows < p.rpt ? rows : p.rpt);
	// items for whole waves, the runs' remainders among them (a remainder a query tile
	// at most; left out of the count: 41.4 us for 64 sequences, 39.3).  Two waves: 46,
	// and 142 instead of 126 for 4 x 131072 rows
	int64_t want = wave - p.tiles;
	while (want < wave / 2)
		want += wave;
	p.target = (int)want;
	// split unless there are tiles enough, or every sequence is a single run
	const int64_t longest = (b->max_kv + kAttnTile - 1) / kAttnTile;
	p.split = p.tiles < 4 * wave && longest > kRunMin;
	p.folds = (p.split ? p.tiles * longest / p.target + 1 : longest) > kFold;
	p.items = p.tiles;
	if (p.split) {
		const int64_t capped = p.tiles * longest / kRunMax + 1;
		const int64_t most = p.tiles * ((longest + kRunMin - 1) / kRunMin);
		p.items += 1 + (capped > p.target ? capped : p.target);
		p.items = p.items < most ? p.items : most;
	}
	if (p.split || p.folds)
		p.part_bytes = (size_t)(p.items * p.rows * (c->d.head_len + 4) * 4);
}

// The kernels of a call: an item a warp (`narrow`), an item a CTA (`wide`), or both, each
// for its sequences.  A wide item pays for kWideRows query rows whether they are there or
// not.  Measured with 4096 cache rows, bf16 (narrow, wide): 8 sequences of 64 rows 71, 141
// us; of 128 124, 148; of 256 288, 178; one of 256 46, 47; one of 2048 283, 175.
struct Plans {
	bool narrow = false, wide = false;
	Plan n, w;
	size_t bytes() const { return n.part_bytes + w.part_bytes; }
};

Plans plan_of(const moe_kv_cache *c, const moe_kv_batch *b, int64_t H, bool fp32)
{
	Plans ps;
	const int64_t HL = c->d.head_len, G = H / c->d.n_kv_heads;
	const int64_t rows = b->max_q * G;   // query rows of a sequence's KV head
	ps.wide = !fp32 && HL <= 128 && rows >= kWideMin;
	// sequences of as many queries as the longest, or one
	ps.narrow = !ps.wide || (b->n_seqs > 1 && b->n_tokens < b->n_seqs * b->max_q);
	if (ps.narrow) {
		const int64_t r = ps.wide ? kWideMin - 1 : rows;
		const int per = fp32 ? 4 : 8;
		// as few columns as hold the rows (4 tiles for a decode batch's 4 rows: 82 us
		// instead of 39); many rows: as many as registers hold (a prompt with 2: 216,
		// with 4: 196)
		ps.n.nt = r <= per ? 1 : r <= 2 * per || HL == 256 ? 2 : 4;
		ps.n.rpt = per * ps.n.nt;
		// 16 resident warps an SM, fewer for wide tiles (at head length 64 the registers
		// leave 8 to 12 of the 16)
		plan_items(ps.n, c, b, G, r, (int64_t)sm_count() * kAttnWarps * (HL * ps.n.nt <= 128 ? 4 : 2));
	}
	if (ps.wide) {
		ps.w.rpt = kWideRows;
		plan_items(ps.w, c, b, G, rows, sm_count());
	}
	return ps;
}

template <typename T, int HL, int NT>
cudaError_t launch_attn_as(const AttnArgs &a, const Plan &p, cudaStream_t st)
{
	constexpr int RPT = (sizeof(T) == 4 ? 4 : 8) * NT;
	constexpr int smem = kAttnSmem<HL>;
	auto kernel = p.folds ? kv_attn_kernel<T, HL, NT, true> : kv_attn_kernel<T, HL, NT, false>;
	if (cudaError_t e = ensure_smem(kernel, smem))
		return e;
	kernel<<<(unsigned)((p.items + kAttnWarps - 1) / kAttnWarps), kAttnThreads, smem, st>>>(a);
	if (cudaError_t e = cudaGetLastError())
		return e;
	return launch_merge<T, HL, RPT>(a, p, st);
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
	const size_t x = plan_of(c, b, H, true).bytes(), y = plan_of(c, b, H, false).bytes();
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
	const Plans p = plan_of(cache, batch, q->n_heads, q->type == MOE_F32);
	if (p.n.items > 0x7fffffff || p.w.items > 0x7fffffff || batch->max_q * (q->n_heads / KVH) > (1 << 30))
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
	a.by_g = QuickDiv((unsigned)a.G);
	a.by_kvh = QuickDiv((unsigned)KVH);
	a.causal = causal != 0;
	a.window = (int)window;
	a.scale2 = scale * 1.44269504088896f;
	a.q_vec = rows_vec16(q);
	a.o_vec = rows_vec16(out);
	uint8_t *part = static_cast<uint8_t *>(workspace);
	auto plan_args = [&](const Plan &x, int64_t least, int64_t most) {
		a.target = x.split ? x.target : 0;
		a.items = x.items;
		a.part = x.part_bytes ? reinterpret_cast<float *>(part) : nullptr;
		a.part_rows = x.rows;
		a.min_rows = (int)least;
		a.max_rows = (int)most;
		part += x.part_bytes;
	};
	if (p.wide) {   // first: its items take longest
		plan_args(p.w, p.narrow ? kWideMin : 0, 1 << 30);
		KV_CK(what, launch_wide(a, p.w, q->type, (int)D, st));
	}
	if (p.narrow) {
		plan_args(p.n, 0, p.wide ? kWideMin - 1 : 1 << 30);
		KV_CK(what, q->type == MOE_F32   ? launch_attn<float>(a, p.n, (int)D, st)
			    : q->type == MOE_F16 ? launch_attn<__half>(a, p.n, (int)D, st)
						 : launch_attn<__nv_bfloat16>(a, p.n, (int)D, st));
	}
	return MOE_OK;
}

}  // extern "C"
