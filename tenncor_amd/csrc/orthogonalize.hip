// The orthogonalised update of a weight matrix (the step of a momentum matrix G
// along its singular directions): with an odd polynomial p(s) = a s + b s^3 + c s^5
// and X = G / (|G| + eps), transposed when it has more rows than columns,
//
//   A = X X^T      B = b A + c A A      X <- a X + B X       `steps` times
//
// which applies p to every singular value of X and leaves its singular vectors.
// With m rows and n >= m columns a step is m^2 n + m^3 + 2 m^2 n multiplications
// and additions (one triangle of the symmetric A and A A): bound by the matrix
// instructions.
//
// fp32: an operand of a product is two halves of 16 bits, x s = hi + lo with
// hi = half(x s), lo = half(x s - hi) and a power of two s that puts the largest
// value the matrix can hold (the host follows the polynomial from |x| <= 1) at
// 2^15.  Each conversion is off by 2^-11 of what it converts at most, so 2^-22 of
// the value is lost in the worst case, or, where lo is too small for that, half a
// step of the smallest halves, 2^-25: 2^-39 of the largest value.  A product is
// hi hi + hi lo + lo hi with the sums in fp32; lo lo would be 2^-22 of the product.
// Three half-precision matrix instructions (2.5 PFLOP/s / 3) stand for one fp32
// instruction (0.157 PFLOP/s), and one load of hi and lo feeds three of them.
//
// What an error of X does is multiplied by up to a in each later step along the
// weak directions of G, while one of A is read through B, which is small against
// a there.  So a X is taken from X in fp32, and the sums of B X are cut into parts
// that are added up apart, so that neither a part nor their sum is a long chain of
// roundings (sum_cut below).
//
// double: the same steps on fp64 matrix instructions (78.6 TFLOP/s); they also take the
// floats of a polynomial whose terms lie too far apart for halves (halves_hold below).
#include "tcg_internal.hpp"

#include <cmath>
#include <new>
#include <type_traits>

namespace
{

typedef _Float16 f16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

// A row of a split matrix: for every 32 elements 32 hi and then 32 lo, 128 bytes
constexpr uint32_t BLOCK = 64; // halves

struct Split
{
	f16 hi, lo;
};

__device__ __forceinline__ Split split (float v)
{
	Split s;
	s.hi = (f16) v;
	s.lo = (f16) (v - (float) s.hi);
	return s;
}

/// hi | lo << 16
__device__ __forceinline__ uint32_t packed (Split s)
{
	return (uint32_t) __builtin_bit_cast(uint16_t, s.hi) | (uint32_t) __builtin_bit_cast(uint16_t, s.lo) << 16;
}

// ---- the norm, and the first split -------------------------------------------------

constexpr uint32_t NORM_PARTS = 512; // workgroups that sum one matrix at most
constexpr uint64_t NORM_RUN = 1024;  // elements of a row a wave takes at a time

template <typename T>
struct PrepArgs
{
	const T* g;
	uint64_t ldg, stride_g;
	uint64_t rows, cols;
	uint32_t parts;
	double* sums; // [batch][parts][RANGES]
	double eps;
	float scale;
	uint32_t* arrived; // [batch][arrivals], cleared here for the products that count in them
	uint32_t arrivals;
	// products of halves: X and X^T as split matrices, padded; in double: dense, padded
	f16* x;
	f16* xt;
	uint64_t ldx, stride_x, ldxt, stride_xt;
	float* x32; // X in fp32, place32
	double* dense[2]; // X, X^T
	uint64_t stride_dense;
	bool tall; // X = G^T
};

/// N values summed over the workgroup at once, in every lane
template <int N>
__device__ __forceinline__ void group_sums (double (&v)[N], double* red)
{
#pragma unroll
	for (int d = TCG_WAVE / 2; d > 0; d >>= 1)
	{
#pragma unroll
		for (int k = 0; k < N; ++k) { v[k] += __shfl_xor(v[k], d); }
	}
	if ((threadIdx.x & (TCG_WAVE - 1)) == 0)
	{
#pragma unroll
		for (int k = 0; k < N; ++k) { red[threadIdx.x / TCG_WAVE * N + k] = v[k]; }
	}
	__syncthreads();
#pragma unroll
	for (int k = 0; k < N; ++k)
	{
		v[k] = 0;
		for (uint32_t w = 0; w < blockDim.x / TCG_WAVE; ++w) { v[k] += red[w * N + k]; }
	}
	__syncthreads();
}

// Sums of squares in double: an error of the norm is one of every singular value.  The
// square of a float is a normal double.  Those of doubles beyond 2^500 are taken of
// v 2^-600 and those below 2^-500 of v 2^600, each into a sum of their own.
template <typename T>
constexpr int RANGES = std::is_same<T,double>::value ? 3 : 1; // as they are, large, small

template <typename T>
__global__ __launch_bounds__(256) void ortho_norm_k (PrepArgs<T> a)
{
	__shared__ double red[4 * RANGES<T>];
	const T* g = a.g + blockIdx.y * a.stride_g;
	double sum[RANGES<T>] = {};
	// runs of the rows dealt to the workgroups' waves, lanes along a run
	const uint32_t wave = threadIdx.x / TCG_WAVE, lane = threadIdx.x & (TCG_WAVE - 1);
	const uint64_t runs = (a.cols + NORM_RUN - 1) / NORM_RUN;
	for (uint64_t at = (uint64_t) blockIdx.x * 4 + wave; at < a.rows * runs; at += (uint64_t) a.parts * 4)
	{
		const T* p = g + at / runs * a.ldg;
		const uint64_t from = at % runs * NORM_RUN, to = from + NORM_RUN < a.cols ? from + NORM_RUN : a.cols;
#pragma unroll 8
		for (uint64_t col = from + lane; col < to; col += TCG_WAVE)
		{
			const double v = p[col];
			if constexpr (RANGES<T> == 1) { sum[0] += v * v; }
			else
			{
				// (a NaN is neither large nor small)
				const bool large = fabs(v) >= 0x1p500, small = fabs(v) < 0x1p-500;
				const double w = v * (large ? 0x1p-600 : small ? 0x1p600 : 1.), square = w * w;
				sum[0] += large || small ? 0. : square;
				sum[1] += large ? square : 0.;
				sum[2] += small ? square : 0.;
			}
		}
	}
	if (blockIdx.x == 0)
	{
		for (uint32_t i = threadIdx.x; i < a.arrivals; i += blockDim.x) { a.arrived[(uint64_t) blockIdx.y * a.arrivals + i] = 0; }
	}
	group_sums(sum, red);
	if (threadIdx.x == 0)
	{
#pragma unroll
		for (int k = 0; k < RANGES<T>; ++k) { a.sums[((uint64_t) blockIdx.y * a.parts + blockIdx.x) * RANGES<T> + k] = sum[k]; }
	}
}

/// X = (G shift) inverse, `shift` a power of two
struct Normed
{
	double shift, inverse;

	template <typename T>
	__device__ __forceinline__ double operator () (T v) const { return (double) v * shift * inverse; }
};

/// The norm's part in every lane; `scale`: what X is multiplied by besides
template <typename T>
__device__ __forceinline__ Normed normed (const PrepArgs<T>& a, uint32_t batch, double* red, double scale)
{
	double sum[RANGES<T>] = {};
	for (uint32_t p = threadIdx.x; p < a.parts; p += blockDim.x)
	{
#pragma unroll
		for (int k = 0; k < RANGES<T>; ++k) { sum[k] += a.sums[((uint64_t) batch * a.parts + p) * RANGES<T> + k]; }
	}
	group_sums(sum, red);
	double square = sum[0];
	Normed out = {1., 0.};
	if constexpr (RANGES<T> > 1)
	{
		square += sum[2] * 0x1p-600 * 0x1p-600;
		if (sum[1] > 0)
		{
			square = sum[1] + sum[0] * 0x1p-600 * 0x1p-600;
			out.shift = 0x1p-600;
		}
		else if (sum[0] == 0 && a.eps < 0x1p-400)
		{
			// nothing but small values, or zeros, whose quotient is zero for the smallest epsilon too
			square = sum[2];
			out.shift = 0x1p600;
		}
	}
	out.inverse = 1. / (::sqrt(square) + a.eps * out.shift) * scale;
	return out;
}

/// Where the 32 x 32 block (bi, bj) of a matrix of `rows` rows keeps its values in fp32:
/// lane l's four values (8 r + 4 (l / 32) + 0..3, l % 32) at 256 r + 4 l
__device__ __forceinline__ uint64_t place32 (uint32_t rows, uint32_t bi, uint32_t bj)
{
	return ((uint64_t) bj * (rows / 32) + bi) * 1024;
}

/// A thread's 16 values of the 64 x 64 tile of G at (r0, c0): rows threadIdx.x / 64 + 4 i of
/// column threadIdx.x % 64, zero outside of G.  No branch around a load, so that all are on
/// their way together (a branch each, waited for in turn: 13 us instead of 10 at 768 x 2048)
template <typename T>
__device__ __forceinline__ void tile_values (T (&v)[16], const PrepArgs<T>& a, const T* g, uint64_t r0, uint64_t c0)
{
	const uint64_t col = c0 + threadIdx.x % 64, at = col < a.cols ? col : a.cols - 1;
#pragma unroll
	for (int i = 0; i < 16; ++i)
	{
		const uint64_t row = r0 + threadIdx.x / 64 + 4 * i;
		v[i] = g[(row < a.rows ? row : a.rows - 1) * a.ldg + at];
	}
#pragma unroll
	for (int i = 0; i < 16; ++i)
	{
		if (col >= a.cols || r0 + threadIdx.x / 64 + 4 * i >= a.rows) { v[i] = 0; }
	}
}

// X = G / (|G| + eps) and X^T as split matrices, a 64 x 64 tile a workgroup; what
// lies outside G is zero
__global__ __launch_bounds__(256) void ortho_split_k (PrepArgs<float> a, uint32_t tiles_x)
{
	__shared__ double red[4 * RANGES<float>];
	__shared__ float tile[64][65];
	const uint32_t batch = blockIdx.y;
	const uint64_t r0 = (uint64_t) (blockIdx.x / tiles_x) * 64, c0 = (uint64_t) (blockIdx.x % tiles_x) * 64;
	float v[16];
	tile_values(v, a, a.g + batch * a.stride_g, r0, c0);
	const Normed x = normed(a, batch, red, a.scale);
#pragma unroll
	for (int i = 0; i < 16; ++i) { tile[threadIdx.x / 64 + 4 * i][threadIdx.x % 64] = (float) x(v[i]); }
	__syncthreads();
	// G's rows are X's rows, or X^T's
	f16* along = (a.tall ? a.xt + batch * a.stride_xt : a.x + batch * a.stride_x);
	f16* across = (a.tall ? a.x + batch * a.stride_x : a.xt + batch * a.stride_xt);
	const uint64_t ld_along = a.tall ? a.ldxt : a.ldx, ld_across = a.tall ? a.ldx : a.ldxt;
#pragma unroll
	for (int k = 0; k < 4; ++k)
	{
		const uint32_t r = threadIdx.x / 16 + 16 * k, c = threadIdx.x % 16 * 4;
		f16x4 hi, lo, thi, tlo;
#pragma unroll
		for (int i = 0; i < 4; ++i)
		{
			const Split s = split(tile[r][c + i]), t = split(tile[c + i][r]);
			hi[i] = s.hi; lo[i] = s.lo;
			thi[i] = t.hi; tlo[i] = t.lo;
		}
		f16* p = along + (r0 + r) * ld_along + (c0 + c) / 32 * BLOCK + c % 32;
		*reinterpret_cast<f16x4*>(p) = hi;
		*reinterpret_cast<f16x4*>(p + 32) = lo;
		f16* q = across + (c0 + r) * ld_across + (r0 + c) / 32 * BLOCK + c % 32;
		*reinterpret_cast<f16x4*>(q) = thi;
		*reinterpret_cast<f16x4*>(q + 32) = tlo;
		// X(i, j) in fp32: four neighbouring i, which are G's columns if it is tall
		const float4 wide = a.tall ? make_float4(tile[r][c], tile[r][c + 1], tile[r][c + 2], tile[r][c + 3]) :
			make_float4(tile[c][r], tile[c + 1][r], tile[c + 2][r], tile[c + 3][r]);
		const uint32_t row = (uint32_t) (a.tall ? c0 : r0) + c, col = (uint32_t) (a.tall ? r0 : c0) + r;
		float* to = a.x32 + batch * (a.stride_x / 2) + place32((uint32_t) (a.ldxt / 2), row / 32, col / 32);
		*reinterpret_cast<float4*>(to + row % 32 / 8 * 256 + (row % 8 / 4 * 32 + col % 32) * 4) = wide;
	}
}

// ---- the products over split matrices ------------------------------------------------

enum Product
{
	GRAM = 0, // A = X X^T
	FACTOR,   // B = b A + c A A
	APPLY,    // X <- a X + B X, X^T along with it
	LAST      // the same into the caller's matrix
};

struct PairArgs
{
	// C(i, j) = sum_k P(i, k) Q(j, k): rows of two split matrices
	const f16* p;
	const f16* q;
	uint64_t ldp, ldq, stride_p, stride_q;
	uint32_t rows_p, rows_q; // padded to whole blocks of 32
	uint32_t slabs; // of 32 summed indices
	uint32_t cut;   // slabs between two cuts of the sums of B X
	// GRAM: `parts` workgroups share a tile, `share` slabs each; their sums meet in `partial`
	// [batch][tiles][parts][tile], and the last to arrive adds them up, in order
	uint32_t parts, share;
	float* partial;
	uint32_t* arrived; // [batch][tiles], zero between two launches
	uint32_t tiles_m, tiles_n, tiles; // tiles: of one matrix (one triangle of them for GRAM and FACTOR)
	// C alpha + add beta, and that in fp32 as it is in the registers of the matrix
	// instructions (`place32`): nothing but the next product of the same tiles reads it
	const float* add32;  // NULL for GRAM
	float* out32;        // NULL for FACTOR and LAST
	uint64_t stride32;
	float alpha, beta;
	// the result: row i, and row j of its transposed
	f16* out;
	f16* out_t;
	uint64_t ldo, ldot, stride_o, stride_ot;
	// LAST
	float* last;
	uint64_t ldl, stride_l;
	uint32_t m, n;
	bool tall;
};

/// Tile number `at` of a lower triangle, row after row
__device__ __forceinline__ void triangle_place (uint32_t at, uint32_t& bi, uint32_t& bj)
{
	bi = (uint32_t) ((sqrtf(8.f * (float) at + 1.f) - 1.f) * 0.5f);
	while (bi * (bi + 1) / 2 > at) { --bi; }
	while ((bi + 1) * (bi + 2) / 2 <= at) { ++bi; }
	bj = at - bi * (bi + 1) / 2;
}

/// Which 16 bytes of a row's 128 lie in which place in LDS: rows whose chunks a
/// load of a matrix operand reads together never share banks
__device__ __forceinline__ uint32_t swizzle (uint32_t row) { return ((row >> 1) & 7) ^ ((row & 1) << 2); }

// WT: 32 x 32 blocks along each side of a wave's tile; four waves 2 x 2 make a tile of
// the result.  SLABS slabs of 32 summed indices have room in LDS.
template <int WT, int SLABS>
constexpr int pair_lds = SLABS * 2 * 64 * WT * 128 > 16 * 32 * WT * (32 * WT + 1) ? SLABS * 2 * 64 * WT * 128 : 16 * 32 * WT * (32 * WT + 1);

template <int WT, int SLABS, int MODE>
__global__ __launch_bounds__(256) void ortho_pair_k (PairArgs g)
{
	constexpr int TILE = 64 * WT;
	constexpr int OPERAND = TILE * 128; // bytes of an operand's slab in LDS
	constexpr int LOADS = 2 * WT;       // a wave's loads per operand and slab
	constexpr bool SYMMETRIC = MODE == GRAM || MODE == FACTOR;
	constexpr bool CUT = MODE == APPLY || MODE == LAST;
	constexpr bool SHARED = MODE == GRAM && WT == 1; // a larger tile has no need of it
	extern __shared__ __attribute__((aligned(1024))) char lds[];

	// consecutive workgroups go to the XCDs in turn: each XCD gets a run of
	// neighbouring tiles, which share rows of P
	const uint32_t total = gridDim.x, xcd = blockIdx.x % 8, each = total / 8, more = total % 8;
	uint32_t at = xcd * each + (xcd < more ? xcd : more) + blockIdx.x / 8;
	uint32_t part = 0, slabs = g.slabs;
	if constexpr (SHARED)
	{
		part = at % g.parts;
		at /= g.parts;
		slabs = slabs - part * g.share < g.share ? slabs - part * g.share : g.share;
	}
	const uint32_t batch = at / g.tiles;
	const uint32_t tile = at % g.tiles;
	uint32_t bi, bj;
	if constexpr (SYMMETRIC)
	{
		triangle_place(tile, bi, bj);
	}
	else
	{
		bi = tile % g.tiles_m;
		bj = tile / g.tiles_m;
	}
	const uint32_t wave = threadIdx.x / TCG_WAVE, lane = threadIdx.x & (TCG_WAVE - 1);
	const uint32_t wi = wave / 2, wj = wave % 2, l32 = lane & 31, half = lane >> 5;

	// where a lane's loads start: 8 rows a load, 8 lanes a row
	const f16* from[2][LOADS];
	uint32_t to[2][LOADS];
#pragma unroll
	for (int i = 0; i < LOADS; ++i)
	{
		const uint32_t r = wave * (16 * WT) + i * 8 + lane / 8;
		const uint32_t chunk = (lane & 7) ^ swizzle(r);
		// rows past the end: the last one again, never stored
		const uint32_t rp = bi * TILE + r, rq = bj * TILE + r;
		const uint64_t first = SHARED ? (uint64_t) part * g.share * BLOCK : 0;
		from[0][i] = g.p + batch * g.stride_p + (uint64_t) (rp < g.rows_p ? rp : g.rows_p - 1) * g.ldp + first + chunk * 8;
		from[1][i] = g.q + batch * g.stride_q + (uint64_t) (rq < g.rows_q ? rq : g.rows_q - 1) * g.ldq + first + chunk * 8;
		const uint32_t base = (uint32_t) (uintptr_t) (const __attribute__((address_space(3))) char*) lds + (wave * (16 * WT) + i * 8) * 128;
		to[0][i] = __builtin_amdgcn_readfirstlane(base);
		to[1][i] = __builtin_amdgcn_readfirstlane(base + OPERAND);
	}
	uint32_t ahead = BLOCK;
	// load number `l` of a wave's 2 LOADS of a slab into LDS buffer `b`, 16 bytes a lane
	// straight from memory.  The instruction itself: for its builtin the compiler waits for
	// every such load before any later read of LDS.  The s_nop is the wait state between
	// the write of M0 and its use.
	auto issue = [&] (uint32_t b, int l)
	{
		const int o = l / LOADS, i = l % LOADS;
		asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
			: : "v"(from[o][i]), "s"(to[o][i] + b * 2 * OPERAND) : "memory", "m0");
		from[o][i] += ahead;
	};
	f32x16 acc[WT][WT] = {}, sum[WT][WT] = {};
	// what a lane supplies to the matrix instructions of half a slab (16 summed indices):
	// hi and lo of its WT rows of P, then of Q
	struct Half
	{
		f16x8 v[4][WT];
	};
	constexpr int READS = 4 * WT, PRODUCTS = 3 * WT * WT;
	auto read = [&] (Half& h, uint32_t b, uint32_t s, int n)
	{
		const int t = n / 4, what = n % 4, o = what / 2;
		const uint32_t row = (o ? wj : wi) * (32 * WT) + t * 32 + l32;
		const uint32_t chunk = (2 * s + half + 4 * (what % 2)) ^ swizzle(row);
		h.v[what][t] = *reinterpret_cast<const f16x8*>(lds + (b * 2 + o) * OPERAND + row * 128 + chunk * 16);
	};
	// The matrix instructions of half a slab (lo and hi, hi and lo, hi and hi: neighbours
	// never wait for each other's sums) and, after number m of them, what goes out
	// meanwhile: `also(m)`.  A wave's instructions are issued in order, and an LDS read
	// or a load holds the ones behind it up for as long as the waves share that unit:
	// all of them together in front of the products left the matrix unit idle half of
	// the time (1530 instead of 770 cycles a slab at WT = 2).
	auto multiply = [&] (const Half& h, auto also)
	{
#pragma unroll
		for (int kind = 0; kind < 3; ++kind)
		{
#pragma unroll
			for (int i = 0; i < WT; ++i)
			{
#pragma unroll
				for (int j = 0; j < WT; ++j)
				{
					acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(h.v[kind == 0 ? 1 : 0][i], h.v[kind == 1 ? 3 : 2][j], acc[i][j], 0, 0, 0);
					also((kind * WT + i) * WT + j);
					__builtin_amdgcn_sched_barrier(0);
				}
			}
		}
	};
	// Half a slab is multiplied while the next half is on its way out of LDS.  Between the
	// halves of slab s: slab s + 1 has landed (loads complete in order, and those of
	// SLABS - 3 later slabs may still be out), and behind the barrier every wave is done
	// with slab s - 1, whose buffer the loads of slab s + SLABS - 1 overwrite (past the
	// end none is left: the last one again, never used).
	auto landed = [] ()
	{
		constexpr int OUT = (SLABS - 3) * 2 * LOADS;
		static_assert(OUT >= 0 && OUT < 64, "vmcnt holds six bits");
		__builtin_amdgcn_sched_barrier(0);
		__builtin_amdgcn_s_waitcnt(0x0f70 | (OUT & 15) | (OUT >> 4) << 14); // vmcnt(OUT)
		__builtin_amdgcn_s_barrier();
		__builtin_amdgcn_sched_barrier(0);
	};
	uint32_t issued = 0, fill = 0, use = 0;
	auto begin = [&] () { if (++issued >= slabs) { ahead = 0; } }; // stays at the last slab
	auto done = [&] () { fill = fill + 1 == SLABS ? 0 : fill + 1; };
	auto whole = [&] ()
	{
		begin();
#pragma unroll
		for (int l = 0; l < 2 * LOADS; ++l) { issue(fill, l); }
		done();
	};
	for (int k = 0; k < SLABS - 2; ++k) { whole(); }
	landed(); // the first slab
	whole();
	Half even, odd;
#pragma unroll
	for (int n = 0; n < READS; ++n) { read(even, 0, 0, n); }
	// reads go out with the first two thirds of the products, loads with all of them
	constexpr int FIRST = PRODUCTS * 2 / 3;
	for (uint32_t s = 0; s < slabs;)
	{
		const uint32_t stop = CUT && s + g.cut < slabs ? s + g.cut : slabs;
		for (; s < stop; ++s)
		{
			multiply(even, [&] (int m)
			{
#pragma unroll
				for (int n = 0; n < READS; ++n) { if (n * FIRST / READS == m) { read(odd, use, 1, n); } }
			});
			landed();
			begin();
			use = use + 1 == SLABS ? 0 : use + 1;
			multiply(odd, [&] (int m)
			{
#pragma unroll
				for (int n = 0; n < READS; ++n) { if (n * FIRST / READS == m) { read(even, use, 0, n); } }
#pragma unroll
				for (int l = 0; l < 2 * LOADS; ++l) { if (l * PRODUCTS / (2 * LOADS) == m) { issue(fill, l); } }
			});
			done();
		}
		if constexpr (CUT)
		{
#pragma unroll
			for (int i = 0; i < WT; ++i)
			{
#pragma unroll
				for (int j = 0; j < WT; ++j)
				{
					sum[i][j] += acc[i][j];
					acc[i][j] = f32x16{};
				}
			}
		}
	}
	// nothing is on its way any more, LDS is free for the result
	__builtin_amdgcn_s_waitcnt(0x0070);
	__syncthreads();
	if constexpr (SHARED)
	{
		if (g.parts > 1)
		{
			// Stores and loads that pass the L2 of the XCD by, which is not coherent with the
			// others': a fence, which writes all of that L2 back, took 25 us a product
			uint64_t* mine = reinterpret_cast<uint64_t*>(g.partial + (uint64_t) at * g.parts * (TILE * TILE)) + threadIdx.x;
#pragma unroll
			for (int r = 0; r < 8; ++r)
			{
				__hip_atomic_store(mine + part * (TILE * TILE / 2) + r * 256, __builtin_bit_cast(uint64_t, make_float2(acc[0][0][2 * r], acc[0][0][2 * r + 1])),
					__ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
			}
			// they have arrived, those of every wave, before the workgroup counts
			__builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
			__builtin_amdgcn_s_waitcnt(0x0070);
			__syncthreads();
			uint32_t* count = reinterpret_cast<uint32_t*>(lds);
			if (threadIdx.x == 0) { *count = __hip_atomic_fetch_add(g.arrived + at, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
			__syncthreads();
			if (*count + 1 != g.parts) { return; }
			if (threadIdx.x == 0) { __hip_atomic_store(g.arrived + at, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
			f32x16 all = {};
#pragma unroll 4
			for (uint32_t q = 0; q < g.parts; ++q)
			{
#pragma unroll
				for (int r = 0; r < 8; ++r)
				{
					const float2 v = __builtin_bit_cast(float2, __hip_atomic_load(mine + q * (TILE * TILE / 2) + r * 256, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
					all[2 * r] += v.x; all[2 * r + 1] += v.y;
				}
			}
			acc[0][0] = all;
			__syncthreads(); // `count` lies where the result goes
		}
	}
	const uint32_t i0 = bi * TILE + wi * (32 * WT), j0 = bj * TILE + wj * (32 * WT);
	// a block of 32 x 32 lies inside the padded result or outside
	auto inside = [&] (int ti, int tj) { return i0 + ti * 32 < g.rows_p && j0 + tj * 32 < g.rows_q; };
	const uint64_t first32 = batch * g.stride32 + lane * 4;
	float4 add[WT][WT][4];
	if constexpr (MODE != GRAM)
	{
#pragma unroll
		for (int ti = 0; ti < WT; ++ti)
		{
#pragma unroll
			for (int tj = 0; tj < WT; ++tj)
			{
				const float* from = g.add32 + first32 + place32(g.rows_p, i0 / 32 + ti, j0 / 32 + tj);
#pragma unroll
				for (int r = 0; r < 4; ++r) { if (inside(ti, tj)) { add[ti][tj][r] = *reinterpret_cast<const float4*>(from + r * 256); } }
			}
		}
	}
	// The wave's tile by way of LDS, [i][j], as hi | lo << 16 (LAST: as it is): a store out of
	// the registers would be 8 bytes in each of 32 rows, 20 us a tile of 192 x 192
	constexpr uint32_t PITCH = 32 * WT + 1;
	uint32_t* meet = reinterpret_cast<uint32_t*>(lds) + wave * (32 * WT) * PITCH;
#pragma unroll
	for (int ti = 0; ti < WT; ++ti)
	{
#pragma unroll
		for (int tj = 0; tj < WT; ++tj)
		{
			if (!inside(ti, tj)) { continue; }
			const f32x16 c = CUT ? sum[ti][tj] : acc[ti][tj];
			float* out32 = nullptr;
			if constexpr (MODE == GRAM || MODE == APPLY) { out32 = g.out32 + first32 + place32(g.rows_p, i0 / 32 + ti, j0 / 32 + tj); }
#pragma unroll
			for (int r = 0; r < 4; ++r)
			{
				float4 v = make_float4(c[4 * r] * g.alpha, c[4 * r + 1] * g.alpha, c[4 * r + 2] * g.alpha, c[4 * r + 3] * g.alpha);
				if constexpr (MODE != GRAM)
				{
					const float4 x = add[ti][tj][r];
					v.x += x.x * g.beta; v.y += x.y * g.beta; v.z += x.z * g.beta; v.w += x.w * g.beta;
				}
				if constexpr (MODE == GRAM || MODE == APPLY) { *reinterpret_cast<float4*>(out32 + r * 256) = v; }
				const float w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
				for (int e = 0; e < 4; ++e)
				{
					meet[(ti * 32 + 8 * r + 4 * half + e) * PITCH + tj * 32 + l32] = MODE == LAST ? __builtin_bit_cast(uint32_t, w[e]) : packed(split(w[e]));
				}
			}
		}
	}
	// the wave reads what it wrote itself
	__builtin_amdgcn_s_waitcnt(0xc07f); // lgkmcnt(0)
	__builtin_amdgcn_wave_barrier();
	constexpr uint32_t QUADS = 8 * WT; // groups of four along a row
	// row `major` of the wave's tile (of its transposed: across), four elements from `minor` on
	auto four = [&] (uint32_t major, uint32_t minor, bool across)
	{
		const uint32_t* p = across ? meet + minor * PITCH + major : meet + major * PITCH + minor;
		const uint32_t step = across ? PITCH : 1;
		return make_uint4(p[0], p[step], p[2 * step], p[3 * step]);
	};
	auto store = [&] (f16* to, uint64_t ld, uint32_t major0, uint32_t minor0, uint32_t majors, uint32_t minors, bool across)
	{
#pragma unroll 4
		for (uint32_t t = 0; t < 32 * WT * QUADS / TCG_WAVE; ++t)
		{
			const uint32_t e = t * TCG_WAVE + lane, major = e / QUADS, minor = e % QUADS * 4;
			if (major0 + major >= majors || minor0 + minor >= minors) { continue; }
			const uint4 v = four(major, minor, across);
			uint2 hi, lo;
			hi.x = (v.x & 0xffff) | v.y << 16; hi.y = (v.z & 0xffff) | v.w << 16;
			lo.x = v.x >> 16 | (v.y & 0xffff0000u); lo.y = v.z >> 16 | (v.w & 0xffff0000u);
			f16* p = to + (uint64_t) (major0 + major) * ld + (uint64_t) ((minor0 + minor) / 32) * BLOCK + (minor0 + minor) % 32;
			*reinterpret_cast<uint2*>(p) = hi;
			*reinterpret_cast<uint2*>(p + 32) = lo;
		}
	};
	if constexpr (MODE != LAST)
	{
		store(g.out_t + batch * g.stride_ot, g.ldot, j0, i0, g.rows_q, g.rows_p, true);
		// a tile on the diagonal of a symmetric result is complete
		if (SYMMETRIC && bi == bj) { return; }
		store(g.out + batch * g.stride_o, g.ldo, i0, j0, g.rows_p, g.rows_q, false);
	}
	else
	{
		const uint32_t major0 = g.tall ? j0 : i0, minor0 = g.tall ? i0 : j0, majors = g.tall ? g.n : g.m, minors = g.tall ? g.m : g.n;
#pragma unroll 4
		for (uint32_t t = 0; t < 32 * WT * QUADS / TCG_WAVE; ++t)
		{
			const uint32_t e = t * TCG_WAVE + lane, major = e / QUADS, minor = e % QUADS * 4;
			if (major0 + major >= majors || minor0 + minor >= minors) { continue; }
			const uint4 v = four(major, minor, g.tall);
			float* p = g.last + batch * g.stride_l + (uint64_t) (major0 + major) * g.ldl + minor0 + minor;
			const float w[4] = {__builtin_bit_cast(float, v.x), __builtin_bit_cast(float, v.y), __builtin_bit_cast(float, v.z), __builtin_bit_cast(float, v.w)};
			if (minor0 + minor + 4 <= minors) { *reinterpret_cast<f32x4_any*>(p) = f32x4_any{w[0], w[1], w[2], w[3]}; }
			else
			{
#pragma unroll
				for (int k = 0; k < 4; ++k) { if (minor0 + minor + k < minors) { p[k] = w[k]; } }
			}
		}
	}
}

// ---- a small matrix in one workgroup ---------------------------------------------------
// X in registers (fp32, 32 x 32 tiles dealt to the waves, up to two each), its halves
// and those of A and B in LDS: all steps in one launch, bound by the barriers between
// their parts instead of by fifteen launches (four matrices of 64 x 96: 76 us by
// launches).  MT: tiles along m, at most 4; nt tiles along n.  The region of X holds
// the halves of X (for A), where waves share a tile of A their fp32 parts of it, and
// the halves of X^T (for B X), one after the other.
constexpr int SMALL_STEPS = 64;

struct SmallArgs
{
	const float* g;
	uint64_t ldg, stride_g;
	float* out;
	uint64_t ldo, stride_o;
	uint32_t m, n, nt;
	uint32_t parts; // waves that share a tile of A, each a part of the summed index
	int steps;
	bool tall;
	double eps;
	float scale; // of X before the first step
	// step k: A = gram C, B = factor C + keep A, X <- apply C + stay X
	float gram[SMALL_STEPS], factor[SMALL_STEPS], keep[SMALL_STEPS], apply[SMALL_STEPS], stay[SMALL_STEPS];
};

/// LDS address of 16 bytes (8 indices of hi: chunk 0..3, of lo: 4..7) of row `row` in
/// block `kb` of 32 summed indices of a matrix of `rows` rows
__device__ __forceinline__ uint32_t small_place (uint32_t rows, uint32_t kb, uint32_t row, uint32_t chunk)
{
	return (kb * rows + row) * 128 + (chunk ^ swizzle(row)) * 16;
}

/// acc += P(rows of tile pi) Q(rows of tile qi)^T over blocks [from, to) of 32 indices
__device__ __forceinline__ void small_product (f32x16& acc, const char* P, uint32_t p_rows, uint32_t pi, const char* Q, uint32_t q_rows, uint32_t qi,
	uint32_t from, uint32_t to, uint32_t l32, uint32_t half)
{
	const uint32_t rp = pi * 32 + l32, rq = qi * 32 + l32;
#pragma unroll 1
	for (uint32_t kb = from; kb < to; ++kb)
	{
#pragma unroll
		for (uint32_t s = 0; s < 2; ++s)
		{
			const uint32_t c = 2 * s + half;
			const f16x8 ph = *reinterpret_cast<const f16x8*>(P + small_place(p_rows, kb, rp, c));
			const f16x8 pl = *reinterpret_cast<const f16x8*>(P + small_place(p_rows, kb, rp, c + 4));
			const f16x8 qh = *reinterpret_cast<const f16x8*>(Q + small_place(q_rows, kb, rq, c));
			const f16x8 ql = *reinterpret_cast<const f16x8*>(Q + small_place(q_rows, kb, rq, c + 4));
			acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph, ql, acc, 0, 0, 0);
			acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(pl, qh, acc, 0, 0, 0);
			acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph, qh, acc, 0, 0, 0);
		}
	}
}

template <int MT, int TILES>
__global__ __launch_bounds__(1024) void ortho_small_k (SmallArgs g)
{
	extern __shared__ __attribute__((aligned(1024))) char lds[];
	constexpr uint32_t ROWS = MT * 32;
	const uint32_t cols = g.nt * 32;
	char* X = lds;                                  // MT * nt tiles of 4 KiB
	char* A = lds + MT * g.nt * 4096;               // MT * MT tiles
	float* scratch = reinterpret_cast<float*>(lds); // tiles of fp32 in the region of X
	const uint32_t waves = blockDim.x / TCG_WAVE, wave = threadIdx.x / TCG_WAVE, lane = threadIdx.x & (TCG_WAVE - 1);
	const uint32_t l32 = lane & 31, half = lane >> 5;
	const float* in = g.g + blockIdx.x * g.stride_g;
	float* out = g.out + blockIdx.x * g.stride_o;

	// the wave's tiles: element r of a lane is X(i, j), i = 32 ti + r % 4 + 8 (r / 4) + 4 half, j = 32 tj + l32
	// (single values, not the vectors of the matrix instructions: those are moved whole when
	// registers run short)
	float x[TILES][16];
	uint32_t ti[TILES], tj[TILES];
	double sum = 0;
#pragma unroll
	for (int t = 0; t < TILES; ++t)
	{
		const uint32_t tile = wave + t * waves;
		ti[t] = tile % MT;
		tj[t] = tile / MT; // nt and more: no such tile
		const uint32_t j = tj[t] * 32 + l32;
#pragma unroll
		for (int r = 0; r < 16; ++r)
		{
			const uint32_t i = ti[t] * 32 + r % 4 + 8 * (r / 4) + 4 * half;
			float v = 0;
			if (i < g.m && j < g.n) { v = g.tall ? in[(uint64_t) j * g.ldg + i] : in[(uint64_t) i * g.ldg + j]; }
			x[t][r] = v;
			sum += (double) v * v;
		}
	}
	{
		double* red = reinterpret_cast<double*>(lds);
#pragma unroll
		for (int d = TCG_WAVE / 2; d > 0; d >>= 1) { sum += __shfl_xor(sum, d); }
		if (lane == 0) { red[wave] = sum; }
		__syncthreads();
		sum = 0;
		for (uint32_t w = 0; w < waves; ++w) { sum += red[w]; }
		__syncthreads();
	}
	const double inv = (double) g.scale / (::sqrt(sum) + g.eps);
#pragma unroll
	for (int t = 0; t < TILES; ++t)
	{
#pragma unroll
		for (int r = 0; r < 16; ++r) { x[t][r] = (float) ((double) x[t][r] * inv); }
	}

	const uint32_t own_lane = lane;
	for (int k = 0; k < g.steps; ++k)
	{
		// a value the compiler cannot follow from step to step: it would otherwise work out
		// every LDS address before the first step and spill them (2100 registers of them)
		uint32_t lane = own_lane;
		asm volatile("" : "+v"(lane));
		const uint32_t l32 = lane & 31, half = lane >> 5;
		// a tile of a matrix of `rows` rows, where it lies transposed: a lane holds four
		// neighbouring summed indices of row 32 t + l32
		auto put_across = [l32, half] (char* where, uint32_t rows, uint32_t kb, uint32_t t, auto value)
		{
#pragma unroll
			for (int r = 0; r < 4; ++r)
			{
				const uint32_t i = 8 * r + 4 * half;
				f16x4 hi, lo;
#pragma unroll
				for (int e = 0; e < 4; ++e)
				{
					const Split s = split(value(4 * r + e));
					hi[e] = s.hi;
					lo[e] = s.lo;
				}
				*reinterpret_cast<f16x4*>(where + small_place(rows, kb, t * 32 + l32, i / 8) + i % 8 * 2) = hi;
				*reinterpret_cast<f16x4*>(where + small_place(rows, kb, t * 32 + l32, i / 8 + 4) + i % 8 * 2) = lo;
				__builtin_amdgcn_sched_barrier(0); // one group after the other: 128 registers a lane are few
			}
		};
		// the halves of X: rows i, summed index j.  Neighbouring lanes hold neighbouring j:
		// an even lane takes both values of one row, the odd one those of the next
#pragma unroll
		for (int t = 0; t < TILES; ++t)
		{
			if (tj[t] >= g.nt) { continue; }
			const bool odd = lane & 1;
			const uint32_t j = l32 & ~1u;
#pragma unroll
			for (int r = 0; r < 16; r += 2)
			{
				const uint32_t first = packed(split(x[t][r])), second = packed(split(x[t][r + 1]));
				const uint32_t got = __shfl_xor(odd ? first : second, 1);
				const uint32_t left = odd ? got : first, right = odd ? second : got;
				const uint32_t i = ti[t] * 32 + (r + (odd ? 1 : 0)) % 4 + 8 * (r / 4) + 4 * half;
				*reinterpret_cast<uint32_t*>(X + small_place(ROWS, tj[t], i, j / 8) + j % 8 * 2) = (left & 0xffff) | right << 16;
				*reinterpret_cast<uint32_t*>(X + small_place(ROWS, tj[t], i, j / 8 + 4) + j % 8 * 2) = left >> 16 | (right & 0xffff0000u);
				__builtin_amdgcn_sched_barrier(0);
			}
		}
		__syncthreads();
		// A = X X^T: tile (ai, aj) in the wave that keeps it, with `parts` waves a tile.  A and B
		// are symmetric: what a wave holds of one goes where it lies transposed, and rows of A
		// serve as both operands of A A
		f32x16 a = {};
		const uint32_t tile = wave % (MT * MT), part = wave / (MT * MT), ai = tile % MT, aj = tile / MT;
		if (part < g.parts)
		{
			small_product(a, X, ROWS, ai, X, ROWS, aj, g.nt * part / g.parts, g.nt * (part + 1) / g.parts, l32, half);
		}
		if (g.parts > 1)
		{
			// the other waves' parts by way of the region of X, added in their order
			__syncthreads();
			if (part > 0 && part < g.parts)
			{
				float* p = scratch + ((part - 1) * (MT * MT) + tile) * 1024 + l32;
#pragma unroll
				for (int r = 0; r < 16; ++r) { p[(r % 4 + 8 * (r / 4) + 4 * half) * 32] = a[r]; }
			}
			__syncthreads();
			if (part == 0)
			{
#pragma unroll 1
				for (uint32_t w = 1; w < g.parts; ++w)
				{
					const float* p = scratch + ((w - 1) * (MT * MT) + tile) * 1024 + l32;
#pragma unroll
					for (int r = 0; r < 16; ++r) { a[r] += p[(r % 4 + 8 * (r / 4) + 4 * half) * 32]; }
				}
			}
		}
		float kept[16] = {};
		if (part == 0)
		{
			const float gram = g.gram[k];
#pragma unroll
			for (int r = 0; r < 16; ++r) { kept[r] = a[r] * gram; }
			put_across(A, ROWS, ai, aj, [&kept] (int r) { return kept[r]; });
		}
		__syncthreads();
		f32x16 b = {};
		if (part == 0) { small_product(b, A, ROWS, ai, A, ROWS, aj, 0, MT, l32, half); }
		__syncthreads();
		if (part == 0)
		{
			// A itself from the registers
			const float factor = g.factor[k], keep = g.keep[k];
			put_across(A, ROWS, ai, aj, [&kept, &b, factor, keep] (int r) { return kept[r] * keep + b[r] * factor; });
		}
#pragma unroll
		for (int t = 0; t < TILES; ++t)
		{
			if (tj[t] < g.nt) { put_across(X, cols, ti[t], tj[t], [&x, t] (int r) { return x[t][r]; }); }
		}
		__syncthreads();
		// X <- a X + B X
#pragma unroll
		for (int t = 0; t < TILES; ++t)
		{
			if (tj[t] >= g.nt) { continue; }
			f32x16 d = {};
			small_product(d, A, ROWS, ti[t], X, cols, tj[t], 0, MT, l32, half);
			const float stay = g.stay[k], apply = g.apply[k];
#pragma unroll
			for (int r = 0; r < 16; ++r) { x[t][r] = x[t][r] * stay + d[r] * apply; }
		}
		__syncthreads();
	}
#pragma unroll
	for (int t = 0; t < TILES; ++t)
	{
		const uint32_t j = tj[t] * 32 + l32;
#pragma unroll
		for (int r = 0; r < 16; ++r)
		{
			const uint32_t i = ti[t] * 32 + r % 4 + 8 * (r / 4) + 4 * half;
			if (i < g.m && j < g.n)
			{
				if (g.tall) { out[(uint64_t) j * g.ldo + i] = x[t][r]; }
				else { out[(uint64_t) i * g.ldo + j] = x[t][r]; }
			}
		}
	}
}

// ---- double -----------------------------------------------------------------------------
// The same steps over dense doubles, padded with zeros to multiples of 64 rows and
// columns, both operands with the summed index along memory.  A wave holds TI x TI
// blocks of 16 x 16 (v_mfma_f64_16x16x4: lane i + 16 q supplies element (i, q) of an
// operand and holds elements (4 r + q, i) of the result) and reads its operands straight
// from memory, three groups of eight summed indices ahead: a matrix instruction takes
// 64 cycles, so nothing has to be staged.  KSPLIT = 4: the four waves
// of a workgroup share one tile, every fourth group each, and their parts are added in
// wave order; KSPLIT = 1: a wave to each quarter of a 64 x 64 tile (the operands are read
// half as often as with tiles of 32).

typedef double f64x2 __attribute__((ext_vector_type(2)));
typedef double f64x4 __attribute__((ext_vector_type(4)));

struct DoubleArgs
{
	// C(i, j) = sum_k p(i, k) q(j, k)
	const double* p;
	const double* q;
	uint64_t ldp, ldq, stride_p, stride_q;
	uint32_t depth; // summed indices, a multiple of 64
	uint32_t tiles_m, tiles_n, tiles;
	const double* add; // C alpha + add beta
	uint64_t ldadd, stride_add;
	double alpha, beta;
	double* out;   // (i, j)
	double* out_t; // (j, i)
	uint64_t ldo, ldot, stride_o, stride_ot;
	void* last; // OUT
	uint64_t ldl, stride_l;
	uint32_t m, n;
	bool tall;
};

// OUT: the type of the caller's matrix, which LAST writes
template <int KSPLIT, int TI, int MODE, typename OUT>
__global__ __launch_bounds__(256) void ortho_double_k (DoubleArgs g)
{
	constexpr bool SYMMETRIC = MODE == GRAM || MODE == FACTOR;
	static_assert(KSPLIT == 4 || (KSPLIT == 1 && TI == 2), "four waves share a tile, or hold a quarter of one each");
	constexpr uint32_t WAVE_TILE = 16 * TI, TILE = KSPLIT == 1 ? 64 : WAVE_TILE;
	constexpr uint32_t PITCH = TILE + 1;
	__shared__ double meet[KSPLIT * TILE * PITCH];
	const uint32_t total = gridDim.x, xcd = blockIdx.x % 8, each = total / 8, more = total % 8;
	const uint32_t at = xcd * each + (xcd < more ? xcd : more) + blockIdx.x / 8;
	const uint32_t batch = at / g.tiles, tile = at % g.tiles;
	uint32_t bi, bj;
	if constexpr (SYMMETRIC) { triangle_place(tile, bi, bj); }
	else
	{
		bi = tile % g.tiles_m;
		bj = tile / g.tiles_m;
	}
	const uint32_t wave = threadIdx.x / TCG_WAVE, lane = threadIdx.x & (TCG_WAVE - 1);
	const uint32_t l16 = lane & 15, quarter = lane >> 4;
	const uint32_t wi = KSPLIT == 1 ? wave / 2 : 0, wj = KSPLIT == 1 ? wave % 2 : 0;
	const double* p = g.p + batch * g.stride_p + (uint64_t) (bi * TILE + wi * WAVE_TILE + l16) * g.ldp + 2 * quarter;
	const double* q = g.q + batch * g.stride_q + (uint64_t) (bj * TILE + wj * WAVE_TILE + l16) * g.ldq + 2 * quarter;
	const uint32_t i0 = bi * TILE, j0 = bj * TILE;
	// what C is added to, ahead of everything: its loads would wait for each other's stores
	constexpr uint32_t EACH = TILE * TILE / 256;
	double add[EACH];
#pragma unroll
	for (uint32_t t = 0; t < EACH; ++t)
	{
		const uint32_t e = t * 256 + threadIdx.x;
		add[t] = MODE == GRAM ? 0 : g.add[batch * g.stride_add + (uint64_t) (i0 + e / TILE) * g.ldadd + j0 + e % TILE];
	}
	f64x4 acc[TI][TI] = {};
	constexpr uint32_t STEP = 8 * KSPLIT; // between a wave's groups of eight indices
	const uint32_t groups = g.depth / STEP, first = KSPLIT == 1 ? 0 : wave * 8;
	struct Group
	{
		f64x2 a[TI], b[TI];
	};
	Group ring[4];
	auto load = [&] (Group& to, uint32_t n)
	{
		const uint32_t k = first + (n < groups ? n : groups - 1) * STEP;
#pragma unroll
		for (int t = 0; t < TI; ++t)
		{
			to.a[t] = *reinterpret_cast<const f64x2*>(p + (uint64_t) t * 16 * g.ldp + k);
			to.b[t] = *reinterpret_cast<const f64x2*>(q + (uint64_t) t * 16 * g.ldq + k);
		}
	};
	auto multiply = [&] (const Group& x)
	{
#pragma unroll
		for (int e = 0; e < 2; ++e)
		{
#pragma unroll
			for (int i = 0; i < TI; ++i)
			{
#pragma unroll
				for (int j = 0; j < TI; ++j)
				{
					acc[i][j] = __builtin_amdgcn_mfma_f64_16x16x4f64(x.a[i][e], x.b[j][e], acc[i][j], 0, 0, 0);
				}
			}
		}
	};
#pragma unroll
	for (uint32_t u = 0; u < 3; ++u) { load(ring[u], u); }
	uint32_t n = 0;
	// four groups at a time without a branch between them: with one the compiler waits for
	// every load that is out
	for (; n + 4 <= groups; n += 4)
	{
#pragma unroll
		for (uint32_t u = 0; u < 4; ++u)
		{
			load(ring[(u + 3) % 4], n + u + 3);
			__builtin_amdgcn_sched_barrier(0);
			multiply(ring[u]);
			__builtin_amdgcn_sched_barrier(0);
		}
	}
#pragma unroll
	for (uint32_t u = 0; u < 3; ++u)
	{
		if (n + u < groups) { multiply(ring[u]); }
	}
	OUT* last = static_cast<OUT*>(g.last) + batch * g.stride_l; // NULL and not used but by LAST
	double* mine = meet + (KSPLIT == 1 ? 0 : wave * TILE * PITCH);
#pragma unroll
	for (int i = 0; i < TI; ++i)
	{
#pragma unroll
		for (int j = 0; j < TI; ++j)
		{
#pragma unroll
			for (int r = 0; r < 4; ++r)
			{
				mine[(wi * WAVE_TILE + i * 16 + 4 * r + quarter) * PITCH + wj * WAVE_TILE + j * 16 + l16] = acc[i][j][r];
			}
		}
	}
	__syncthreads();
	// the result where its rows run along memory; what is kept transposed goes by LDS
#pragma unroll
	for (uint32_t t = 0; t < EACH; ++t)
	{
		const uint32_t e = t * 256 + threadIdx.x, i = e / TILE, j = e % TILE;
		double v = 0;
#pragma unroll
		for (int w = 0; w < KSPLIT; ++w) { v += meet[w * TILE * PITCH + i * PITCH + j]; }
		v *= g.alpha;
		if constexpr (MODE != GRAM) { v += g.beta * add[t]; }
		if constexpr (MODE != LAST) { g.out[batch * g.stride_o + (uint64_t) (i0 + i) * g.ldo + j0 + j] = v; }
		else if (!g.tall && i0 + i < g.m && j0 + j < g.n) { last[(uint64_t) (i0 + i) * g.ldl + j0 + j] = (OUT) v; }
		meet[i * PITCH + j] = v; // read by this lane alone until now
	}
	__syncthreads();
	if ((SYMMETRIC && bi == bj) || (MODE == LAST && !g.tall)) { return; }
#pragma unroll
	for (uint32_t t = 0; t < EACH; ++t)
	{
		const uint32_t e = t * 256 + threadIdx.x, j = e / TILE, i = e % TILE;
		const double v = meet[i * PITCH + j];
		if constexpr (MODE != LAST) { g.out_t[batch * g.stride_ot + (uint64_t) (j0 + j) * g.ldot + i0 + i] = v; }
		else if (i0 + i < g.m && j0 + j < g.n) { last[(uint64_t) (j0 + j) * g.ldl + i0 + i] = (OUT) v; }
	}
}

// X = G / (|G| + eps) and X^T, padded: a 64 x 64 tile a workgroup
template <typename T>
__global__ __launch_bounds__(256) void ortho_scale_k (PrepArgs<T> a, uint32_t tiles_x)
{
	__shared__ double red[4 * RANGES<T>];
	__shared__ double tile[64][65];
	const uint32_t batch = blockIdx.y;
	const uint64_t r0 = (uint64_t) (blockIdx.x / tiles_x) * 64, c0 = (uint64_t) (blockIdx.x % tiles_x) * 64;
	T v[16];
	tile_values(v, a, a.g + batch * a.stride_g, r0, c0);
	const Normed x = normed(a, batch, red, 1.);
	double* along = a.dense[a.tall] + batch * a.stride_dense;
	double* across = a.dense[!a.tall] + batch * a.stride_dense;
	const uint64_t ld_along = a.tall ? a.ldxt : a.ldx, ld_across = a.tall ? a.ldx : a.ldxt;
#pragma unroll
	for (int i = 0; i < 16; ++i)
	{
		const uint32_t r = threadIdx.x / 64 + 4 * i, c = threadIdx.x % 64;
		tile[r][c] = x(v[i]);
		along[(r0 + r) * ld_along + c0 + c] = tile[r][c];
	}
	__syncthreads();
#pragma unroll
	for (int i = 0; i < 16; ++i)
	{
		const uint32_t c = threadIdx.x / 64 + 4 * i, r = threadIdx.x % 64;
		across[(c0 + c) * ld_across + r0 + r] = tile[r][c];
	}
}

// ---- the host's side ---------------------------------------------------------------------

struct Plan
{
	int steps;
	double a, b, c;
	// the largest singular value before step k, and the largest value of A and B in it
	std::vector<double> x, gram, factor;
};

/// Follows the largest singular value any matrix can have: false where it grows out of bounds
bool follow (Plan& p)
{
	if (!std::isfinite(p.a) || !std::isfinite(p.b) || !std::isfinite(p.c)) { return false; }
	double top = 1.0001; // |X| <= 1, and the roundings of the norm
	for (int k = 0; k <= p.steps; ++k)
	{
		if (!(top <= 1e6)) { return false; } // a NaN as well
		p.x.push_back(top);
		if (k == p.steps) { break; } // nothing is made of the last X
		// both are largest at an end or where their slope is zero: with q = s^2,
		// p' = a + 3 b q + 5 c q^2 and (b q + c q^2)' = b + 2 c q
		double next = 0, factor = 0;
		auto at = [&] (double q)
		{
			if (!(q > 0 && q <= top * top)) { return; }
			next = std::fmax(next, std::sqrt(q) * std::fabs(p.a + q * (p.b + q * p.c)));
			factor = std::fmax(factor, std::fabs(q * (p.b + q * p.c)));
		};
		at(top * top);
		at(-p.b / (2 * p.c)); // c = 0: infinite or NaN, neither is in range
		const double inner = 9 * p.b * p.b - 20 * p.a * p.c;
		if (inner >= 0)
		{
			// the roots of 5 c q^2 + 3 b q + a without a difference of neighbouring values: with a c
			// that is almost zero, as the sum of a caller's roundings, -3 b + sqrt(inner) would be 0
			// and the polynomial's largest value missed
			const double w = -(3 * p.b + std::copysign(std::sqrt(inner), p.b)) / 2;
			at(w / (5 * p.c));
			at(p.a / w);
		}
		if (!(next <= 1e300 && factor <= 1e12)) { return false; }
		p.gram.push_back(top * top);
		p.factor.push_back(factor * 1.0001);
		top = next * 1.0001;
	}
	return true;
}

/// Whether two halves hold enough of a step's operands.  Their scale follows the largest
/// value that any matrix can have, and what a half loses at the lower end is 2^-39 of
/// that (2^-25 where the largest lies at 2^14 or more), however small this matrix's own
/// values are.  Of A and B it is 2^-39 F with F the largest value of B, and next to a X,
/// which is taken in fp32, no more than 2^-22 of the result if |a| >= 2^-17 F.  A
/// polynomial without a linear term has no such measure to go by (s^3 in float, 300 x
/// 200: off by 6.7e-6 after two steps, zeros after three): its products are in double.
bool halves_hold (const Plan& p)
{
	for (double factor : p.factor)
	{
		if (std::fabs(p.a) < std::ldexp(factor, -17)) { return false; }
	}
	return true;
}

/// The power of two that puts `top` at 2^15, half of what a half can hold
float scale_of (double top)
{
	if (!(top > 1e-9)) { top = 1e-9; }
	int e;
	(void) std::frexp(top, &e); // top < 2^e
	return std::ldexp(1.f, 15 - e);
}

/// A slab is six additions to a sum; cut so that neither a part nor the sum of the parts
/// is a long chain.  Distance from the formulas at 768 rows (24 slabs): cut every 2 or
/// 4 slabs 2.9e-6, every 8 3.6e-6; at 4096 (128 slabs): every 2 4.3e-6, every 9 3.2e-6;
/// fp32 products that are never cut 1.3e-5 and 2.9e-5.  A cut of a tile of 192 x 192 is
/// 3900 cycles, two slabs' worth.
uint32_t sum_cut (uint32_t slabs)
{
	const uint32_t cut = (uint32_t) std::lround(2 * std::sqrt(slabs / 6.));
	return cut < 4 ? 4 : cut;
}

uint64_t padded (uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }

uint32_t norm_parts (uint64_t rows, uint64_t cols)
{
	const uint64_t want = (rows * ((cols + NORM_RUN - 1) / NORM_RUN) + 3) / 4;
	return (uint32_t) (want < NORM_PARTS ? want : NORM_PARTS);
}

template <int WT, int SLABS, int MODE>
hipError_t pair_launch (tcg_ctx* ctx, const PairArgs& g, uint64_t batch)
{
	constexpr int bytes = pair_lds<WT,SLABS>;
	if constexpr (bytes > 65536)
	{
		// what a workgroup may hold beyond the 64 KiB that need no asking for
		hipError_t err = hipFuncSetAttribute((const void*) ortho_pair_k<WT,SLABS,MODE>, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
		if (err != hipSuccess) { return err; }
	}
	ortho_pair_k<WT,SLABS,MODE><<<(unsigned) (g.tiles * batch * (MODE == GRAM ? g.parts : 1)), 256, bytes, ctx->stream>>>(g);
	return hipGetLastError();
}

template <int WT, int SLABS>
hipError_t pair_launch_mode (tcg_ctx* ctx, Product mode, PairArgs& g, uint64_t batch)
{
	g.tiles_m = (g.rows_p + 64 * WT - 1) / (64 * WT);
	g.tiles_n = (g.rows_q + 64 * WT - 1) / (64 * WT);
	g.tiles = mode == GRAM || mode == FACTOR ? g.tiles_m * (g.tiles_m + 1) / 2 : g.tiles_m * g.tiles_n;
	switch (mode)
	{
		case GRAM: return pair_launch<WT,SLABS,GRAM>(ctx, g, batch);
		case FACTOR: return pair_launch<WT,SLABS,FACTOR>(ctx, g, batch);
		case APPLY: return pair_launch<WT,SLABS,APPLY>(ctx, g, batch);
		default: return pair_launch<WT,SLABS,LAST>(ctx, g, batch);
	}
}

// How a product is cut up.  Measured in cycles on this chip (tiles of 64 WT rows and
// columns; a workgroup takes slabs x `slab` + `ends`, with `apply` instead of `slab`
// where sums are cut and X is added):
//   WT 1  five slabs in LDS, two workgroups a CU     slab 500 alone, 800 together, apply 900   ends 7000
//   WT 2  four slabs, one workgroup a CU             slab 950                      apply 1400  ends 9000
//   WT 3  three slabs, one workgroup a CU            slab 2030                     apply 2600  ends 16000
// A larger tile reads less per product (WT 1 is bound by LDS, 48 KiB a slab for 200
// cycles of matrix instructions; WT 3 keeps them busy 85 % of the time) and leaves
// more of the chip idle in its last round.  4096 x 4096, all five steps: 6.6 ms with
// WT 1, 5.6 with WT 2, 4.0 with WT 3; 1024 x 1024: 192, 429 and 740 us.
struct PairCost
{
	uint32_t per_cu;
	double slab, apply, ends;
};
constexpr PairCost pair_costs[4] = {{}, {2, 800, 900, 7000}, {1, 950, 1400, 9000}, {1, 2030, 2600, 16000}};

// Where the tiles of A leave CUs without one, several workgroups share a tile, each a run
// of its slabs: 12 slabs or more, or bringing the parts together costs more than they save
// (all five steps, shared and not: 768 x 2048, 3 workgroups a tile, 199 and 227 us; 256 x
// 4096, 10 a tile, 137 and 220, with runs of 6 slabs 20 more; 640 x 640, where runs would
// be of 6 slabs, 147 and 146).  A part costs the last workgroup about as much as a slab, so
// no more of them than the root of the slabs (4 x 100000: 290 us with 56 parts, 458 with 256)
constexpr uint64_t SHARE_LEAST = 12;
constexpr double SHARE_ENDS = 7000; // cycles to bring the parts together

/// Workgroups that share a tile of A
uint32_t gram_parts (const tcg_ctx* ctx, int wt, uint64_t rows, uint64_t slabs, uint64_t batch)
{
	if (wt != 1) { return 1; }
	const uint64_t tm = rows / 64, tiles = tm * (tm + 1) / 2 * batch;
	uint64_t parts = (uint64_t) ctx->num_cus / tiles;
	if (parts > slabs / SHARE_LEAST) { parts = slabs / SHARE_LEAST; }
	const uint64_t most = (uint64_t) ::sqrt((double) slabs);
	if (parts > most) { parts = most; }
	if (parts < 2) { return 1; }
	const uint64_t share = (slabs + parts - 1) / parts;
	return (uint32_t) ((slabs + share - 1) / share); // none without a slab
}

/// Cycles of one product with tiles of 64 wt
double pair_cycles (const tcg_ctx* ctx, int wt, bool symmetric, uint64_t rows_p, uint64_t rows_q, uint64_t slabs, uint64_t batch, uint32_t parts = 1)
{
	const PairCost& c = pair_costs[wt];
	const uint64_t tm = (rows_p + 64 * wt - 1) / (64 * wt), tn = (rows_q + 64 * wt - 1) / (64 * wt);
	const uint64_t tiles = (symmetric ? tm * (tm + 1) / 2 : tm * tn) * batch;
	const uint64_t room = (uint64_t) ctx->num_cus * c.per_cu;
	double slab = symmetric ? c.slab : c.apply;
	if (wt == 1 && tiles * parts <= (uint64_t) ctx->num_cus) { slab = symmetric ? 500 : 650; }
	if (parts > 1) { return (double) ((slabs + parts - 1) / parts) * slab + c.ends + SHARE_ENDS; }
	return (double) ((tiles + room - 1) / room) * ((double) slabs * slab + c.ends);
}

hipError_t pair_dispatch (tcg_ctx* ctx, Product mode, int wt, PairArgs& g, uint64_t batch)
{
	switch (wt)
	{
		case 1: return pair_launch_mode<1,5>(ctx, mode, g, batch);
		case 2: return pair_launch_mode<2,4>(ctx, mode, g, batch);
		default: return pair_launch_mode<3,3>(ctx, mode, g, batch);
	}
}

/// Tiles of LDS a matrix takes in ortho_small_k, 0: it is not one of its
int small_tiles (uint64_t m, uint64_t n)
{
	const uint64_t mt = (m + 31) / 32, nt = (n + 31) / 32;
	if (mt > 4 || nt > 32 || mt * nt > 32) { return 0; }
	const int tiles = (int) (mt * nt + mt * mt);
	return tiles <= 39 ? tiles : 0; // 156 of 160 KiB
}

template <int MT>
hipError_t small_launch (tcg_ctx* ctx, const SmallArgs& g, uint64_t batch, int lds_tiles)
{
	const unsigned tiles = MT * g.nt, waves = tiles < 16 ? tiles : 16, bytes = lds_tiles * 4096;
	const void* kernel = tiles > 16 ? (const void*) ortho_small_k<MT,2> : (const void*) ortho_small_k<MT,1>;
	if (bytes > 65536)
	{
		hipError_t err = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int) bytes);
		if (err != hipSuccess) { return err; }
	}
	if (tiles > 16) { ortho_small_k<MT,2><<<(unsigned) batch, waves * TCG_WAVE, bytes, ctx->stream>>>(g); }
	else { ortho_small_k<MT,1><<<(unsigned) batch, waves * TCG_WAVE, bytes, ctx->stream>>>(g); }
	return hipGetLastError();
}

int ortho_small (tcg_ctx* ctx, const Plan& plan, uint64_t rows, uint64_t cols, uint64_t batch, const float* in, uint64_t ldg,
	uint64_t stride_g, double eps, float* out, uint64_t ldo, uint64_t stride_o, int lds_tiles)
{
	SmallArgs g = {};
	g.g = in; g.ldg = ldg; g.stride_g = stride_g;
	g.out = out; g.ldo = ldo; g.stride_o = stride_o;
	g.tall = rows > cols;
	g.m = (uint32_t) (g.tall ? cols : rows);
	g.n = (uint32_t) (g.tall ? rows : cols);
	const uint32_t mt = (g.m + 31) / 32;
	g.nt = (g.n + 31) / 32;
	const uint32_t waves = mt * g.nt < 16 ? mt * g.nt : 16;
	// the parts' tiles have to fit where X lies; more than four cost more to add up than they save
	g.parts = waves / (mt * mt);
	if (g.parts > g.nt / mt) { g.parts = g.nt / mt; }
	if (g.parts > 4) { g.parts = 4; }
	g.steps = plan.steps;
	g.eps = eps;
	g.scale = scale_of(plan.x[0]);
	for (int k = 0; k < plan.steps; ++k)
	{
		const float sx = scale_of(plan.x[k]), sa = scale_of(plan.gram[k]), sb = scale_of(plan.factor[k]);
		const float sn = k + 1 == plan.steps ? 1.f : scale_of(plan.x[k + 1]);
		g.gram[k] = sa / sx / sx;
		g.factor[k] = (float) plan.c * (sb / sa / sa);
		g.keep[k] = (float) plan.b * (sb / sa);
		g.apply[k] = sn / sb / sx;
		g.stay[k] = (float) plan.a * (sn / sx);
	}
	hipError_t err;
	switch (mt)
	{
		case 1: err = small_launch<1>(ctx, g, batch, lds_tiles); break;
		case 2: err = small_launch<2>(ctx, g, batch, lds_tiles); break;
		case 3: err = small_launch<3>(ctx, g, batch, lds_tiles); break;
		default: err = small_launch<4>(ctx, g, batch, lds_tiles); break;
	}
	if (err != hipSuccess) { return tcg_fail(ctx, TCG_ERR_HIP, "launch of orthogonalize failed: %s", hipGetErrorString(err)); }
	return TCG_OK;
}

int ortho_float (tcg_ctx* ctx, const Plan& plan, uint64_t rows, uint64_t cols, uint64_t batch, const float* in, uint64_t ldg,
	uint64_t stride_g, double eps, float* out, uint64_t ldo, uint64_t stride_o)
{
	const bool tall = rows > cols;
	const uint64_t m = tall ? cols : rows, n = tall ? rows : cols;
	if (const int tiles = small_tiles(m, n))
	{
		return ortho_small(ctx, plan, rows, cols, batch, in, ldg, stride_g, eps, out, ldo, stride_o, tiles);
	}
	const uint64_t mp = padded(m, 64), np = padded(n, 64);
	TCG_REQUIRE(ctx, mp / 64 * (np / 64) * batch < (1ull << 31), "tcg_orthogonalize: %llu matrices of %llu x %llu are too many",
		(unsigned long long) batch, (unsigned long long) rows, (unsigned long long) cols);
	// A in fp32 goes from GRAM to FACTOR in the order of their tiles: one size for both
	int wt_gram = 1, wt_apply = 1;
	double least_gram = 1e300, least_apply = 1e300;
	for (int wt = 1; wt <= 3; ++wt)
	{
		const double both = pair_cycles(ctx, wt, true, mp, mp, np / 32, batch, gram_parts(ctx, wt, mp, np / 32, batch)) + pair_cycles(ctx, wt, true, mp, mp, mp / 32, batch);
		const double apply = pair_cycles(ctx, wt, false, mp, np, mp / 32, batch);
		if (both < least_gram) { least_gram = both; wt_gram = wt; }
		if (apply < least_apply) { least_apply = apply; wt_apply = wt; }
	}
	const uint32_t gram_shares = gram_parts(ctx, wt_gram, mp, np / 32, batch);
	const uint64_t gram_tiles = gram_shares > 1 ? mp / 64 * (mp / 64 + 1) / 2 : 0;

	// X, X^T and X in fp32 before and after a step, A, A in fp32, B; 32 bits an element each
	const size_t xs = (size_t) mp * np * 2, as = (size_t) mp * mp * 2; // halves
	const uint32_t parts = norm_parts(rows, cols);
	const size_t sums_bytes = ((size_t) batch * parts * sizeof(double) + 255) / 256 * 256;
	const size_t arrived_bytes = ((size_t) batch * gram_tiles * sizeof(uint32_t) + 255) / 256 * 256;
	const size_t partial_bytes = (size_t) batch * gram_tiles * gram_shares * 64 * 64 * sizeof(float);
	const size_t bytes = sums_bytes + arrived_bytes + partial_bytes + (6 * xs + 3 * as) * batch * sizeof(f16);
	void* mem = nullptr;
	int rc = tcg_alloc(ctx, bytes, &mem);
	if (rc != TCG_OK) { return rc; }
	f16* x[2], *xt[2];
	float* x32[2];
	uint32_t* arrived = reinterpret_cast<uint32_t*>((char*) mem + sums_bytes);
	float* partial = reinterpret_cast<float*>((char*) arrived + arrived_bytes);
	f16* p = reinterpret_cast<f16*>((char*) partial + partial_bytes);
	for (int k = 0; k < 2; ++k)
	{
		x[k] = p; p += xs * batch;
		xt[k] = p; p += xs * batch;
		x32[k] = reinterpret_cast<float*>(p); p += xs * batch;
	}
	f16* gram = p;
	f16* factor = gram + as * batch;
	float* gram32 = reinterpret_cast<float*>(factor + as * batch);

	PrepArgs<float> prep = {};
	prep.g = in; prep.ldg = ldg; prep.stride_g = stride_g;
	prep.rows = rows; prep.cols = cols;
	prep.parts = parts; prep.sums = (double*) mem; prep.eps = eps;
	prep.scale = scale_of(plan.x[0]);
	prep.arrived = arrived; prep.arrivals = (uint32_t) gram_tiles;
	prep.x = x[0]; prep.xt = xt[0]; prep.x32 = x32[0];
	prep.ldx = np * 2; prep.ldxt = mp * 2;
	prep.stride_x = prep.stride_xt = xs;
	prep.tall = tall;
	ortho_norm_k<float><<<dim3(parts, (unsigned) batch), 256, 0, ctx->stream>>>(prep);
	const uint32_t tiles_x = (uint32_t) ((tall ? mp : np) / 64);
	ortho_split_k<<<dim3((unsigned) (mp / 64 * (np / 64)), (unsigned) batch), 256, 0, ctx->stream>>>(prep, tiles_x);

	hipError_t err = hipGetLastError();
	auto launch = [&] (Product mode, PairArgs& g)
	{
		if (err != hipSuccess) { return; }
		err = pair_dispatch(ctx, mode, mode == GRAM || mode == FACTOR ? wt_gram : wt_apply, g, batch);
	};
	for (int k = 0; k < plan.steps; ++k)
	{
		const int now = k & 1, next = now ^ 1;
		const float sx = scale_of(plan.x[k]), sa = scale_of(plan.gram[k]), sb = scale_of(plan.factor[k]);
		PairArgs g = {};
		g.rows_p = g.rows_q = (uint32_t) mp;
		g.p = g.q = x[now];
		g.ldp = g.ldq = np * 2; g.stride_p = g.stride_q = xs;
		g.slabs = (uint32_t) (np / 32);
		g.parts = gram_shares; g.share = (g.slabs + g.parts - 1) / g.parts;
		g.partial = partial; g.arrived = arrived;
		g.alpha = sa / sx / sx;
		g.out32 = gram32; g.stride32 = as / 2;
		g.out = g.out_t = gram;
		g.ldo = g.ldot = mp * 2; g.stride_o = g.stride_ot = as;
		launch(GRAM, g);
		g.p = g.q = gram;
		g.ldp = g.ldq = mp * 2; g.stride_p = g.stride_q = as;
		g.add32 = gram32; g.out32 = nullptr;
		g.slabs = (uint32_t) (mp / 32);
		g.alpha = (float) plan.c * (sb / sa / sa);
		g.beta = (float) plan.b * (sb / sa);
		g.out = g.out_t = factor;
		launch(FACTOR, g);
		const bool last = k + 1 == plan.steps;
		const float sn = last ? 1.f : scale_of(plan.x[k + 1]);
		g.rows_q = (uint32_t) np;
		g.p = factor;
		g.q = xt[now];
		g.ldq = mp * 2; g.stride_q = xs;
		g.add32 = x32[now]; g.out32 = x32[next]; g.stride32 = xs / 2;
		g.cut = sum_cut(g.slabs);
		g.alpha = sn / sb / sx;
		g.beta = (float) plan.a * (sn / sx);
		g.out = x[next]; g.ldo = np * 2; g.stride_o = xs;
		g.out_t = xt[next]; g.ldot = mp * 2; g.stride_ot = xs;
		g.last = out; g.ldl = ldo; g.stride_l = stride_o;
		g.m = (uint32_t) m; g.n = (uint32_t) n;
		g.tall = tall;
		launch(last ? LAST : APPLY, g);
	}
	rc = tcg_free(ctx, mem, bytes);
	if (err != hipSuccess) { return tcg_fail(ctx, TCG_ERR_HIP, "launch of orthogonalize failed: %s", hipGetErrorString(err)); }
	return rc;
}

template <int KSPLIT, int TI, typename T>
void double_launch (tcg_ctx* ctx, Product mode, const DoubleArgs& g, uint64_t batch)
{
	const unsigned grid = (unsigned) (g.tiles * batch);
	switch (mode)
	{
		case GRAM: ortho_double_k<KSPLIT,TI,GRAM,double><<<grid, 256, 0, ctx->stream>>>(g); break;
		case FACTOR: ortho_double_k<KSPLIT,TI,FACTOR,double><<<grid, 256, 0, ctx->stream>>>(g); break;
		case APPLY: ortho_double_k<KSPLIT,TI,APPLY,double><<<grid, 256, 0, ctx->stream>>>(g); break;
		default: ortho_double_k<KSPLIT,TI,LAST,T><<<grid, 256, 0, ctx->stream>>>(g); break;
	}
}

/// The iteration in double, of matrices of type T
template <typename T>
int ortho_double (tcg_ctx* ctx, const Plan& plan, uint64_t rows, uint64_t cols, uint64_t batch, const T* in, uint64_t ldg,
	uint64_t stride_g, double eps, T* out, uint64_t ldo, uint64_t stride_o)
{
	const bool tall = rows > cols;
	const uint64_t m = tall ? cols : rows, n = tall ? rows : cols;
	const uint64_t mp = padded(m, 64), np = padded(n, 64);
	const size_t xs = (size_t) mp * np, as = (size_t) mp * mp;
	const uint32_t parts = norm_parts(rows, cols);
	const size_t sums_bytes = ((size_t) batch * parts * RANGES<T> * sizeof(double) + 255) / 256 * 256;
	const size_t bytes = sums_bytes + (4 * xs + 2 * as) * batch * sizeof(double);
	TCG_REQUIRE(ctx, mp / 16 * (np / 16) * batch < (1ull << 31), "tcg_orthogonalize: %llu matrices of %llu x %llu are too many",
		(unsigned long long) batch, (unsigned long long) rows, (unsigned long long) cols);
	void* mem = nullptr;
	int rc = tcg_alloc(ctx, bytes, &mem);
	if (rc != TCG_OK) { return rc; }
	double* x[2][2]; // [before, after a step][X, X^T]
	double* at = (double*) ((char*) mem + sums_bytes);
	for (int k = 0; k < 4; ++k, at += xs * batch) { x[k / 2][k % 2] = at; }
	double* gram = at;
	double* factor = gram + as * batch;
	PrepArgs<T> prep = {};
	prep.g = in; prep.ldg = ldg; prep.stride_g = stride_g;
	prep.rows = rows; prep.cols = cols;
	prep.parts = parts; prep.sums = (double*) mem; prep.eps = eps;
	prep.dense[0] = x[0][0]; prep.dense[1] = x[0][1];
	prep.stride_dense = xs;
	prep.ldx = np; prep.ldxt = mp;
	prep.tall = tall;
	ortho_norm_k<T><<<dim3(parts, (unsigned) batch), 256, 0, ctx->stream>>>(prep);
	ortho_scale_k<T><<<dim3((unsigned) (mp / 64 * (np / 64)), (unsigned) batch), 256, 0, ctx->stream>>>(prep, (uint32_t) ((tall ? mp : np) / 64));
	// Tiles of 64 where there are two for every CU, of 16 where tiles of 32 would leave half
	// of the CUs without one (256 x 256: 127 us with tiles of 32, 85 with tiles of 16;
	// 1024 x 1024: 840 us with tiles of 32, 1000 with tiles of 64, 1460 with tiles of 16)
	auto launch = [&] (Product mode, DoubleArgs& g, uint64_t height, uint64_t width)
	{
		const bool symmetric = mode == GRAM || mode == FACTOR;
		auto tiles = [&] (uint64_t tile)
		{
			const uint64_t tm = height / tile, tn = width / tile;
			return symmetric ? tm * (tm + 1) / 2 : tm * tn;
		};
		const uint64_t cus = (uint64_t) ctx->num_cus;
		const uint32_t tile = tiles(64) * batch >= 2 * cus ? 64 : 2 * tiles(32) * batch <= cus ? 16 : 32;
		g.tiles_m = (uint32_t) (height / tile);
		g.tiles_n = (uint32_t) (width / tile);
		g.tiles = (uint32_t) tiles(tile);
		switch (tile)
		{
			case 64: double_launch<1,2,T>(ctx, mode, g, batch); break;
			case 32: double_launch<4,2,T>(ctx, mode, g, batch); break;
			default: double_launch<4,1,T>(ctx, mode, g, batch); break;
		}
	};
	for (int k = 0; k < plan.steps; ++k)
	{
		double** now = x[k & 1];
		double** next = x[(k & 1) ^ 1];
		DoubleArgs g = {};
		g.p = g.q = now[0];
		g.ldp = g.ldq = np; g.stride_p = g.stride_q = xs;
		g.depth = (uint32_t) np;
		g.alpha = 1;
		g.out = g.out_t = gram;
		g.ldo = g.ldot = mp; g.stride_o = g.stride_ot = as;
		launch(GRAM, g, mp, mp);
		g.p = g.q = g.add = gram;
		g.ldp = g.ldq = g.ldadd = mp; g.stride_p = g.stride_q = g.stride_add = as;
		g.depth = (uint32_t) mp;
		g.alpha = plan.c;
		g.beta = plan.b;
		g.out = g.out_t = factor;
		launch(FACTOR, g, mp, mp);
		g.p = factor;
		g.q = now[1];
		g.ldq = mp; g.stride_q = xs;
		g.add = now[0];
		g.ldadd = np; g.stride_add = xs;
		g.alpha = 1;
		g.beta = plan.a;
		g.out = next[0]; g.ldo = np; g.stride_o = xs;
		g.out_t = next[1]; g.ldot = mp; g.stride_ot = xs;
		g.last = out; g.ldl = ldo; g.stride_l = stride_o;
		g.m = (uint32_t) m; g.n = (uint32_t) n;
		g.tall = tall;
		launch(k + 1 == plan.steps ? LAST : APPLY, g, mp, np);
	}
	hipError_t err = hipGetLastError();
	rc = tcg_free(ctx, mem, bytes);
	if (err != hipSuccess) { return tcg_fail(ctx, TCG_ERR_HIP, "launch of orthogonalize failed: %s", hipGetErrorString(err)); }
	return rc;
}

constexpr uint64_t MOST_ELEMENTS = 1ull << 33; // of one matrix, padding included; its temporaries take up to 48 bytes an element
constexpr uint64_t MOST_BATCH = 65535;
constexpr uint64_t MOST_APART = 1ull << 40; // elements from the first matrix to the last: more than any memory holds

} // namespace

extern "C" {

int tcg_orthogonalize (tcg_ctx* ctx, int dtype, uint64_t rows, uint64_t cols, uint64_t batch, const void* in, uint64_t ldi,
	uint64_t stride_i, int steps, const double coef[3], double eps, void* out, uint64_t ldo, uint64_t stride_o)
{
	if (!ctx) { return TCG_ERR_ARG; }
	TCG_REQUIRE(ctx, dtype == TCG_FLOAT || dtype == TCG_DOUBLE, "tcg_orthogonalize: dtype %d is neither float nor double", dtype);
	TCG_REQUIRE(ctx, ldi >= cols && ldo >= cols, "tcg_orthogonalize: leading dims %llu and %llu of rows of %llu elements",
		(unsigned long long) ldi, (unsigned long long) ldo, (unsigned long long) cols);
	TCG_REQUIRE(ctx, steps >= 1 && steps <= 64, "tcg_orthogonalize: %d steps: 1 to 64 are possible", steps);
	TCG_REQUIRE(ctx, eps >= 0, "tcg_orthogonalize: eps %g is negative or not a number", eps);
	TCG_REQUIRE(ctx, coef, "tcg_orthogonalize: NULL pointer");
	if (0 == rows || 0 == cols || 0 == batch) { return TCG_OK; }
	TCG_REQUIRE(ctx, in && out, "tcg_orthogonalize: NULL pointer");
	TCG_REQUIRE(ctx, rows <= MOST_ELEMENTS / 128 && cols <= MOST_ELEMENTS / 128 && ldi <= MOST_ELEMENTS && ldo <= MOST_ELEMENTS &&
		padded(rows, 128) <= MOST_ELEMENTS / padded(cols, 128) && batch <= MOST_BATCH,
		"tcg_orthogonalize: %llu matrices of %llu x %llu are too many or too large",
		(unsigned long long) batch, (unsigned long long) rows, (unsigned long long) cols);
	TCG_REQUIRE(ctx, batch == 1 || (stride_i <= MOST_APART / (batch - 1) && stride_o <= MOST_APART / (batch - 1)),
		"tcg_orthogonalize: %llu matrices %llu and %llu elements from one to the next are too far apart",
		(unsigned long long) batch, (unsigned long long) stride_i, (unsigned long long) stride_o);
	// a matrix's rows end before the next matrix begins, or the matrices lie side by side in
	// rows that hold one of each
	const auto apart = [&] (uint64_t ld, uint64_t stride)
	{
		return batch == 1 || stride >= (rows - 1) * ld + cols || (stride >= cols && stride <= ld && (batch - 1) * stride <= ld - cols);
	};
	TCG_REQUIRE(ctx, apart(ldi, stride_i) && apart(ldo, stride_o), "tcg_orthogonalize: matrices %llu and %llu elements apart overlap",
		(unsigned long long) stride_i, (unsigned long long) stride_o);
	TCG_REQUIRE(ctx, in != out || (ldi == ldo && (batch == 1 || stride_i == stride_o)),
		"tcg_orthogonalize: in place with another layout");
	if (tcg_small_mode(ctx)) { TCG_SMALL_RETURN(ctx, tcg_small_unsupported(ctx, "an orthogonalised update")); }
	tcg_device_scope device(ctx);
	try
	{
		Plan plan;
		plan.steps = steps;
		plan.a = coef[0];
		plan.b = coef[1];
		plan.c = coef[2];
		TCG_REQUIRE(ctx, follow(plan), "tcg_orthogonalize: with the polynomial %g s + %g s^3 + %g s^5 singular values grow past 1e6",
			coef[0], coef[1], coef[2]);
		if (batch == 1) { stride_i = stride_o = 0; }
		// beside the norm of a matrix of floats, 1e-45 or more, this is nothing either, and its
		// reciprocal, by which zeros are multiplied, is finite
		if (dtype == TCG_FLOAT && eps > 0 && eps < 0x1p-900) { eps = 0x1p-900; }
		if (dtype == TCG_DOUBLE) { return ortho_double(ctx, plan, rows, cols, batch, (const double*) in, ldi, stride_i, eps, (double*) out, ldo, stride_o); }
		return halves_hold(plan) ?
			ortho_float(ctx, plan, rows, cols, batch, (const float*) in, ldi, stride_i, eps, (float*) out, ldo, stride_o) :
			ortho_double(ctx, plan, rows, cols, batch, (const float*) in, ldi, stride_i, eps, (float*) out, ldo, stride_o);
	}
	catch (const std::bad_alloc&)
	{
		return tcg_fail(ctx, TCG_ERR_OOM, "tcg_orthogonalize: out of host memory");
	}
}

} // extern "C"
