// Layer normalisation over the leading `cols` elements of every row, and its
// three gradients.  For a row x of N elements (w, b: weight and bias)
//
//   m = sum x / N     v = sum (x - m)^2 / N     r = 1 / sqrt(v + eps)
//   h = (x - m) r     y = h w + b
//
// and for the gradient g that arrives at y
//
//   dx = r (g w - mean(g w) - h mean(g w h))
//   dw = sum over rows of g h          db = sum over rows of g
//
// Both directions are bound by memory: 2 (forward) and 3 (backward) passes over
// rows x cols elements at 8 and 14 operations an element.
//
// A row is held in registers between its only load and its only store, so the
// statistics cost no second pass over memory.  They are taken in two passes over
// those registers: the mean first, then the sums of d = x - m and of d^2; the
// first of the two is what the rounding of m left (m's error times N), and it is
// taken out of mean and variance, which makes them as good for rows far from
// zero as for centred ones.  Rows that are too long for registers are cut into
// chunks (the *_chunk_* kernels below).
//
// The sums over rows stay in registers of the waves that walk them, one partial
// row of dw and db per workgroup goes to memory, and a second launch adds these
// up in a fixed order: no atomics, the same bits at every call.  All gradients of a
// few rows with known statistics take one launch, in which workgroups of their own
// sum over the rows.
#include "tcg_internal.hpp"

#include <limits>

namespace
{

// ---- loads and stores of 16 bytes at the alignment of one element ------------
// gfx950 takes 128-bit accesses at any 4-byte boundary: rows of odd length and
// rows that start anywhere need no path of their own, only the last, partial
// vector of a row goes element by element.
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef double f64x2_any __attribute__((ext_vector_type(2), aligned(8)));
template <typename T> struct AnyVec;
template <> struct AnyVec<float> { using type = f32x4_any; };
template <> struct AnyVec<double> { using type = f64x2_any; };

template <typename T>
constexpr int VN = Vec16<T>::N;

// ONCE: with the hint that nothing reads or writes this memory again soon
template <typename T, bool RAGGED, bool ONCE = false>
__device__ __forceinline__ typename Vec16<T>::type load_vec (const T* row, uint32_t col, uint32_t cols)
{
	typename Vec16<T>::type v = {};
	if (col + VN<T> <= cols)
	{
		const auto* from = reinterpret_cast<const typename AnyVec<T>::type*>(row + col);
		v = ONCE ? __builtin_nontemporal_load(from) : *from;
	}
	else if constexpr (RAGGED)
	{
#pragma unroll
		for (int i = 0; i < VN<T>; ++i)
		{
			if (col + i < cols) { v[i] = row[col + i]; }
		}
	}
	return v;
}

template <typename T, bool RAGGED, bool ONCE = false>
__device__ __forceinline__ void store_vec (T* row, uint32_t col, uint32_t cols, typename Vec16<T>::type v)
{
	if (col + VN<T> <= cols)
	{
		auto* to = reinterpret_cast<typename AnyVec<T>::type*>(row + col);
		if constexpr (ONCE) { __builtin_nontemporal_store((typename AnyVec<T>::type) v, to); }
		else { *to = v; }
	}
	else if constexpr (RAGGED)
	{
#pragma unroll
		for (int i = 0; i < VN<T>; ++i)
		{
			if (col + i < cols) { row[col + i] = v[i]; }
		}
	}
}

/// Whether element i of the vector at `col` belongs to the row
template <typename T, bool RAGGED>
__device__ __forceinline__ bool in_row (uint32_t col, int i, uint32_t cols)
{
	return RAGGED ? col + i < cols : col < cols;
}

// ---- sums over the lanes that share a row --------------------------------------
template <typename T, int LANES>
__device__ __forceinline__ T lane_sum (T v)
{
#pragma unroll
	for (int d = LANES / 2; d > 0; d >>= 1) { v += __shfl_xor(v, d); }
	return v;
}

/// The sums of a and b over the SPAN lanes of a row, in every one of them.  `red` holds
/// two sets of two values a wave that calls take in turn: a wave that is a call ahead
/// writes the other set, so that one barrier a call is enough.
template <typename T, int SPAN>
__device__ __forceinline__ void row_sums (T& a, T& b, T* red, uint32_t& turn)
{
	a = lane_sum<T,(SPAN < TCG_WAVE ? SPAN : TCG_WAVE)>(a);
	b = lane_sum<T,(SPAN < TCG_WAVE ? SPAN : TCG_WAVE)>(b);
	if constexpr (SPAN > TCG_WAVE)
	{
		constexpr int W = SPAN / TCG_WAVE;
		T* set = red + (turn & 1) * 2 * W;
		++turn;
		const uint32_t wave = threadIdx.x / TCG_WAVE;
		if ((threadIdx.x & (TCG_WAVE - 1)) == 0)
		{
			set[2 * wave] = a;
			set[2 * wave + 1] = b;
		}
		__syncthreads();
		a = 0;
		b = 0;
#pragma unroll
		for (int w = 0; w < W; ++w)
		{
			a += set[2 * w];
			b += set[2 * w + 1];
		}
	}
}

__device__ __forceinline__ float inv_sqrt (float v) { return 1.f / sqrtf(v); }
__device__ __forceinline__ double inv_sqrt (double v) { return 1. / ::sqrt(v); }

/// a b as a value of its own.  A product that the compiler may fuse into the
/// difference x - a b is another number there (not rounded) than where it is
/// kept, and what the rounding left would be taken out of the wrong one.
template <typename T>
__device__ __forceinline__ T rounded (T a, T b)
{
#pragma clang fp contract(off)
	const T product = a * b;
	return product;
}

__device__ __forceinline__ float fused (float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double fused (double a, double b, double c) { return __builtin_fma(a, b, c); }

/// v / n by way of inv_n = 1 / n rounded: the remainder puts the last bit right, so that
/// a quotient that is a number of the type comes out as that (41 x (1 / 41) does not).
/// Not for infinite v.
template <typename T>
__device__ __forceinline__ T quotient (T v, T n, T inv_n)
{
	const T q = rounded(v, inv_n);
	return fused(fused(-q, n, v), inv_n, q);
}

/// Mean and reciprocal deviation of the row held in v (PER vectors a lane); what
/// is left of a value after the mean is (x - m) - c, see above.  In a row of equal elements
/// all sums but the first are exact, and so are c and c ds: nothing is left, and the variance
/// is zero.  (With c = ds inv_n 83 elements of 16.2 came to -4e-11 in place of 0 and 141 of
/// 1.9e7 to -4e-5.)  Where the sum of squares is infinite r is zero.
template <typename T, int SPAN, int PER, bool RAGGED>
__device__ __forceinline__ void row_stats (const typename Vec16<T>::type (&v)[PER], uint32_t lane, uint32_t cols, T n, T inv_n, T eps,
	T* red, uint32_t& turn, T& m, T& c, T& r)
{
	T sum = 0, none = 0;
#pragma unroll
	for (int j = 0; j < PER; ++j)
	{
#pragma unroll
		for (int i = 0; i < VN<T>; ++i) { sum += v[j][i]; }
	}
	row_sums<T,SPAN>(sum, none, red, turn);
	m = rounded(sum, inv_n);
	T ds = 0, dq = 0;
#pragma unroll
	for (int j = 0; j < PER; ++j)
	{
		const uint32_t col = (j * SPAN + lane) * VN<T>;
#pragma unroll
		for (int i = 0; i < VN<T>; ++i)
		{
			const T d = in_row<T,RAGGED>(col, i, cols) ? v[j][i] - m : (T) 0;
			ds += d;
			dq += d * d;
		}
	}
	row_sums<T,SPAN>(ds, dq, red, turn);
	c = quotient(ds, n, inv_n);
	T var = fused(-c, ds, dq) * inv_n;
	var = var < 0 ? (T) 0 : var;
	r = inv_sqrt(var + eps);
}

/// m + c, or m where that is not finite (c is then a NaN, the mean is not)
template <typename T>
__device__ __forceinline__ T whole_mean (T m, T c)
{
	return fabs(m) <= std::numeric_limits<T>::max() ? m + c : m;
}

template <typename T>
struct NormArgs
{
	const T* x;
	uint64_t ldx;
	const T* weight; // NULL: ones
	const T* bias;   // NULL: zeros
	T* y;
	uint64_t ldy;
	T* mean;         // NULL, or one value a row
	T* rstd;
	uint64_t rows;
	uint32_t cols;
	T eps, n, inv_n; // n: cols, in a scalar register next to its reciprocal
};

/// Workgroups of 256 lanes take several rows at once; a row of more lanes has one to itself
constexpr int group_size (int span) { return span < 256 ? 256 : span; }
constexpr uint32_t rows_at_once (int span) { return group_size(span) / span; }

// SPAN lanes share a row
template <typename T, int SPAN, int PER, bool RAGGED>
__global__ __launch_bounds__(group_size(SPAN)) void layer_norm_k (NormArgs<T> a)
{
	using V = typename Vec16<T>::type;
	__shared__ T red[4 * group_size(SPAN) / TCG_WAVE];
	uint32_t turn = 0;
	constexpr uint32_t ROWS = rows_at_once(SPAN);
	const uint32_t lane = threadIdx.x % SPAN;
	V w[PER], b[PER];
#pragma unroll
	for (int j = 0; j < PER; ++j)
	{
		const uint32_t col = (j * SPAN + lane) * VN<T>;
		w[j] = V{} + (T) 1;
		b[j] = V{};
		if (a.weight) { w[j] = load_vec<T,RAGGED>(a.weight, col, a.cols); }
		if (a.bias) { b[j] = load_vec<T,RAGGED>(a.bias, col, a.cols); }
	}
	uint64_t row = (uint64_t) blockIdx.x * ROWS + threadIdx.x / SPAN;
	for (; row < a.rows; row += (uint64_t) gridDim.x * ROWS)
	{
		const T* x = a.x + row * a.ldx;
		V v[PER];
#pragma unroll
		for (int j = 0; j < PER; ++j) { v[j] = load_vec<T,RAGGED>(x, (j * SPAN + lane) * VN<T>, a.cols); }
		T m, c, r;
		row_stats<T,SPAN,PER,RAGGED>(v, lane, a.cols, a.n, a.inv_n, a.eps, red, turn, m, c, r);
		T* y = a.y + row * a.ldy;
#pragma unroll
		for (int j = 0; j < PER; ++j)
		{
			V out;
#pragma unroll
			for (int i = 0; i < VN<T>; ++i) { out[i] = ((v[j][i] - m) - c) * r * w[j][i] + b[j][i]; }
			store_vec<T,RAGGED>(y, (j * SPAN + lane) * VN<T>, a.cols, out);
		}
		if (a.mean && lane == 0)
		{
			a.mean[row] = whole_mean(m, c);
			a.rstd[row] = r;
		}
	}
}

template <typename T>
struct GradArgs
{
	const T* dy;
	uint64_t lddy;
	const T* x;
	uint64_t ldx;
	const T* weight; // NULL: ones
	const T* mean;   // NULL: taken from x here
	const T* rstd;
	T* dx;           // NULL: not wanted
	uint64_t lddx;
	T* partial;      // [workgroup][dw, db][cols]
	uint64_t rows;
	uint32_t cols;
	T eps, n, inv_n; // n: cols, in a scalar register next to its reciprocal
};

// ONCE: x, dy and dx are more than the caches hold.
// (The next row's loads ahead of the row in hand changed nothing: 32768 x 4096 295 us
// without them, 289 and 301 with them, depending on where the statistics were loaded.)
template <typename T, int SPAN, int PER, bool RAGGED, bool DX, bool PARAMS, bool ONCE>
__device__ __forceinline__ void grad_rows (const GradArgs<T>& a, uint32_t group, uint32_t groups)
{
	using V = typename Vec16<T>::type;
	__shared__ T red[4 * group_size(SPAN) / TCG_WAVE];
	uint32_t turn = 0;
	constexpr uint32_t ROWS = rows_at_once(SPAN);
	const uint32_t lane = threadIdx.x % SPAN;
	V w[PER], dw[PER], db[PER];
#pragma unroll
	for (int j = 0; j < PER; ++j)
	{
		dw[j] = V{};
		db[j] = V{};
		w[j] = V{} + (T) 1;
		if (DX && a.weight) { w[j] = load_vec<T,RAGGED>(a.weight, (j * SPAN + lane) * VN<T>, a.cols); }
	}
	const uint64_t step = (uint64_t) groups * ROWS;
	for (uint64_t row = (uint64_t) group * ROWS + threadIdx.x / SPAN; row < a.rows; row += step)
	{
		const T* x = a.x + row * a.ldx;
		const T* dy = a.dy + row * a.lddy;
		V h[PER], g[PER];
#pragma unroll
		for (int j = 0; j < PER; ++j)
		{
			h[j] = load_vec<T,RAGGED,ONCE>(x, (j * SPAN + lane) * VN<T>, a.cols);
			g[j] = load_vec<T,RAGGED,ONCE>(dy, (j * SPAN + lane) * VN<T>, a.cols);
		}
		T m, c = 0, r;
		if (a.mean)
		{
			m = a.mean[row];
			r = a.rstd[row];
		}
		else { row_stats<T,SPAN,PER,RAGGED>(h, lane, a.cols, a.n, a.inv_n, a.eps, red, turn, m, c, r); }
		T sg = 0, sh = 0;
#pragma unroll
		for (int j = 0; j < PER; ++j)
		{
			const uint32_t col = (j * SPAN + lane) * VN<T>;
#pragma unroll
			for (int i = 0; i < VN<T>; ++i)
			{
				// past the end of the row x reads as zero, which is not the mean
				h[j][i] = in_row<T,RAGGED>(col, i, a.cols) ? ((h[j][i] - m) - c) * r : (T) 0;
				if constexpr (PARAMS)
				{
					dw[j][i] += g[j][i] * h[j][i];
					db[j][i] += g[j][i];
				}
				if constexpr (DX)
				{
					g[j][i] *= w[j][i];
					sg += g[j][i];
					sh += g[j][i] * h[j][i];
				}
			}
		}
		if constexpr (DX)
		{
			row_sums<T,SPAN>(sg, sh, red, turn);
			sg *= a.inv_n;
			sh *= a.inv_n;
			T* dx = a.dx + row * a.lddx;
#pragma unroll
			for (int j = 0; j < PER; ++j)
			{
				V out;
#pragma unroll
				for (int i = 0; i < VN<T>; ++i) { out[i] = r * (g[j][i] - sg - h[j][i] * sh); }
				store_vec<T,RAGGED,ONCE>(dx, (j * SPAN + lane) * VN<T>, a.cols, out);
			}
		}
	}
	if constexpr (PARAMS)
	{
		T* out = a.partial + (uint64_t) group * 2 * a.cols;
		if constexpr (ROWS > 1)
		{
			// the row slots of the workgroup hold sums of the same columns: added in their order
			__shared__ V meet[2][PER][SPAN];
			const uint32_t slot = threadIdx.x / SPAN;
			for (uint32_t turn = 0; turn < ROWS; ++turn)
			{
				if (slot == turn)
				{
#pragma unroll
					for (int j = 0; j < PER; ++j)
					{
						if (turn > 0)
						{
							dw[j] += meet[0][j][lane];
							db[j] += meet[1][j][lane];
						}
						meet[0][j][lane] = dw[j];
						meet[1][j][lane] = db[j];
					}
				}
				__syncthreads();
			}
			if (slot + 1 < ROWS) { return; }
		}
#pragma unroll
		for (int j = 0; j < PER; ++j)
		{
			store_vec<T,RAGGED>(out, (j * SPAN + lane) * VN<T>, a.cols, dw[j]);
			store_vec<T,RAGGED>(out + a.cols, (j * SPAN + lane) * VN<T>, a.cols, db[j]);
		}
	}
}

template <typename T, int SPAN, int PER, bool RAGGED, bool DX, bool PARAMS, bool ONCE>
__global__ __launch_bounds__(group_size(SPAN)) void layer_norm_grad_k (GradArgs<T> a)
{
	grad_rows<T,SPAN,PER,RAGGED,DX,PARAMS,ONCE>(a, blockIdx.x, gridDim.x);
}

// dw and db of the four vectors of columns of a strip, straight from x and dy: 64 lanes take
// every 64th row each and are added up in the order of their lanes' tree and waves
template <typename T>
__device__ __forceinline__ void grad_strip (const GradArgs<T>& a, uint32_t strip, T* dweight, T* dbias)
{
	using V = typename Vec16<T>::type;
	__shared__ V meet[2][4][4];
	const uint32_t place = threadIdx.x % 4, lane = threadIdx.x % TCG_WAVE, wave = threadIdx.x / TCG_WAVE;
	const uint32_t col = (strip * 4 + place) * VN<T>;
	// the row's last whole vector for lanes that would read past it; they keep what is their own
	const uint32_t from = col + VN<T> <= a.cols ? col : a.cols - VN<T>;
	V dw = {}, db = {};
#pragma unroll 4
	for (uint64_t row = threadIdx.x / 4; row < a.rows; row += 64)
	{
		const V x = *reinterpret_cast<const typename AnyVec<T>::type*>(a.x + row * a.ldx + from);
		const V g = *reinterpret_cast<const typename AnyVec<T>::type*>(a.dy + row * a.lddy + from);
		const T m = a.mean[row], r = a.rstd[row];
#pragma unroll
		for (int i = 0; i < VN<T>; ++i)
		{
			dw[i] += g[i] * ((x[i] - m) * r);
			db[i] += g[i];
		}
	}
#pragma unroll
	for (int d = 4; d < TCG_WAVE; d *= 2)
	{
#pragma unroll
		for (int i = 0; i < VN<T>; ++i)
		{
			dw[i] += __shfl_xor(dw[i], d);
			db[i] += __shfl_xor(db[i], d);
		}
	}
	if (lane < 4)
	{
		meet[0][wave][place] = dw;
		meet[1][wave][place] = db;
	}
	__syncthreads();
	if (threadIdx.x >= 4) { return; }
	for (int k = 1; k < 4; ++k)
	{
		dw += meet[0][k][place];
		db += meet[1][k][place];
	}
#pragma unroll
	for (int i = 0; i < VN<T>; ++i)
	{
		if (from + i >= col && from + i < a.cols)
		{
			if (dweight) { dweight[from + i] = dw[i]; }
			if (dbias) { dbias[from + i] = db[i]; }
		}
	}
}

// All three gradients of a few rows with known statistics in one launch: the first
// `strips` workgroups take dw and db, the others dx.  x and dy are read twice, which
// costs less than a second launch as long as they are small.
template <typename T, int SPAN, int PER, bool RAGGED>
__global__ __launch_bounds__(256) void layer_norm_grad_few_k (GradArgs<T> a, uint32_t strips, T* dweight, T* dbias)
{
	if (blockIdx.x < strips) { grad_strip(a, blockIdx.x, dweight, dbias); }
	else { grad_rows<T,SPAN,PER,RAGGED,true,false,false>(a, blockIdx.x - strips, gridDim.x - strips); }
}

// dw[col], db[col] = the sums over `parts` partial rows, 32 columns a workgroup,
// its 32 lane rows each taking every 32nd part; then in lane-row order
template <typename T>
__global__ __launch_bounds__(1024) void layer_norm_params_k (const T* partial, uint32_t parts, uint32_t cols, T* dweight, T* dbias)
{
	__shared__ T meet[32][33];
	const uint32_t tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
	const uint64_t col = (uint64_t) blockIdx.x * 32 + tx; // of the 2 * cols columns of a part
	const uint64_t width = (uint64_t) 2 * cols;
	T sum = 0;
	if (col < width)
	{
#pragma unroll 4
		for (uint32_t p = ty; p < parts; p += 32) { sum += partial[p * width + col]; }
	}
	meet[ty][tx] = sum;
	__syncthreads();
	if (ty == 0 && col < width)
	{
		for (int k = 1; k < 32; ++k) { sum += meet[k][tx]; }
		T* out = col < cols ? dweight : dbias;
		if (out) { out[col < cols ? col : col - cols] = sum; }
	}
}

// ---- rows too long for registers ------------------------------------------------
// A workgroup holds one chunk of a row at a time.  The chunks' statistics meet in
// double: the mean of the means (each weighted with its chunk's length), and the
// chunks' squares plus what their means are off that one.  A chunk's mean is kept
// as the two values m and c of row_stats, the row's as the m of its first chunk
// and the distance from there, so that long rows far from zero are as good as
// short ones.
constexpr uint32_t CHUNK_VECS = 8; // vectors a lane holds

template <typename T>
constexpr uint32_t CHUNK = 256 * CHUNK_VECS * VN<T>;

template <typename T>
struct ChunkArgs
{
	const T* x;
	uint64_t ldx;
	const T* dy;
	uint64_t lddy;
	const T* weight;
	const T* bias;
	T* out; // y, or dx
	uint64_t ldo;
	const T* mean_in; // what the caller has of the statistics, or NULL
	const T* rstd_in;
	T* mean;
	T* rstd;
	double* sums;     // [row][chunk][3]: m, c and squares, or sum of g w and of g w h
	double* stats;    // [row][5]: a mean's two parts, rstd, mean of g w, mean of g w h
	uint64_t rows, cols;
	uint32_t chunks;
	double eps;
};

/// The chunk of workgroup `at`: its row and its place there
template <typename T>
__device__ __forceinline__ void chunk_place (const ChunkArgs<T>& a, uint64_t at, uint64_t& row, uint64_t& from, uint32_t& count)
{
	row = at / a.chunks;
	from = (at % a.chunks) * CHUNK<T>;
	count = (uint32_t) (a.cols - from < CHUNK<T> ? a.cols - from : CHUNK<T>);
}

template <typename T>
__global__ __launch_bounds__(256) void layer_norm_chunk_stats_k (ChunkArgs<T> a)
{
	using V = typename Vec16<T>::type;
	__shared__ T red[16];
	uint32_t turn = 0;
	for (uint64_t at = blockIdx.x; at < a.rows * a.chunks; at += gridDim.x)
	{
		uint64_t row, from;
		uint32_t count;
		chunk_place(a, at, row, from, count);
		const T* x = a.x + row * a.ldx + from;
		V v[CHUNK_VECS];
#pragma unroll
		for (uint32_t j = 0; j < CHUNK_VECS; ++j) { v[j] = load_vec<T,true>(x, (j * 256 + threadIdx.x) * VN<T>, count); }
		T m, c, r;
		row_stats<T,256,CHUNK_VECS,true>(v, threadIdx.x, count, (T) count, (T) 1 / (T) count, (T) 0, red, turn, m, c, r);
		T dq = 0, none = 0;
#pragma unroll
		for (uint32_t j = 0; j < CHUNK_VECS; ++j)
		{
#pragma unroll
			for (int i = 0; i < VN<T>; ++i)
			{
				const T d = in_row<T,true>((j * 256 + threadIdx.x) * VN<T>, i, count) ? (v[j][i] - m) - c : (T) 0;
				dq += d * d;
			}
		}
		row_sums<T,256>(dq, none, red, turn);
		if (threadIdx.x == 0)
		{
			a.sums[3 * at] = m;
			a.sums[3 * at + 1] = fabs(m) <= std::numeric_limits<T>::max() ? c : (T) 0;
			a.sums[3 * at + 2] = dq;
		}
	}
}

template <typename T>
__global__ __launch_bounds__(256) void layer_norm_chunk_merge_k (ChunkArgs<T> a)
{
	const uint64_t row = (uint64_t) blockIdx.x * 256 + threadIdx.x;
	if (row >= a.rows) { return; }
	double* stats = a.stats + 5 * row;
	if (a.mean_in)
	{
		stats[0] = a.mean_in[row];
		stats[1] = 0;
		stats[2] = a.rstd_in[row];
		return;
	}
	const double* sums = a.sums + 3 * row * a.chunks;
	auto count = [&a](uint32_t k)
	{
		const uint64_t left = a.cols - (uint64_t) k * CHUNK<T>;
		return (double) (left < CHUNK<T> ? left : CHUNK<T>);
	};
	const double base = fabs(sums[0]) <= std::numeric_limits<double>::max() ? sums[0] : 0;
	double m = 0, q = 0;
	for (uint32_t k = 0; k < a.chunks; ++k) { m += count(k) * ((sums[3 * k] - base) + sums[3 * k + 1]); }
	m /= (double) a.cols;
	for (uint32_t k = 0; k < a.chunks; ++k)
	{
		const double off = ((sums[3 * k] - base) + sums[3 * k + 1]) - m;
		q += sums[3 * k + 2] + count(k) * off * off;
	}
	const double r = 1. / ::sqrt(q / (double) a.cols + a.eps);
	stats[0] = base;
	stats[1] = m;
	stats[2] = r;
	if (a.mean)
	{
		a.mean[row] = (T) (base + m);
		a.rstd[row] = (T) r;
	}
}

template <typename T>
__global__ __launch_bounds__(256) void layer_norm_chunk_apply_k (ChunkArgs<T> a)
{
	using V = typename Vec16<T>::type;
	for (uint64_t at = blockIdx.x; at < a.rows * a.chunks; at += gridDim.x)
	{
		uint64_t row, from;
		uint32_t count;
		chunk_place(a, at, row, from, count);
		const T* x = a.x + row * a.ldx + from;
		T* y = a.out + row * a.ldo + from;
		const T m = (T) a.stats[5 * row], c = (T) a.stats[5 * row + 1], r = (T) a.stats[5 * row + 2];
#pragma unroll
		for (uint32_t j = 0; j < CHUNK_VECS; ++j)
		{
			const uint32_t col = (j * 256 + threadIdx.x) * VN<T>;
			if (col >= count) { break; }
			const V v = load_vec<T,true>(x, col, count);
			const V w = a.weight ? load_vec<T,true>(a.weight + from, col, count) : V{} + (T) 1;
			const V b = a.bias ? load_vec<T,true>(a.bias + from, col, count) : V{};
			V out;
#pragma unroll
			for (int i = 0; i < VN<T>; ++i) { out[i] = ((v[i] - m) - c) * r * w[i] + b[i]; }
			store_vec<T,true>(y, col, count, out);
		}
	}
}

template <typename T>
__global__ __launch_bounds__(256) void layer_norm_chunk_grad_sums_k (ChunkArgs<T> a)
{
	using V = typename Vec16<T>::type;
	__shared__ T red[16];
	uint32_t turn = 0;
	for (uint64_t at = blockIdx.x; at < a.rows * a.chunks; at += gridDim.x)
	{
		uint64_t row, from;
		uint32_t count;
		chunk_place(a, at, row, from, count);
		const T* x = a.x + row * a.ldx + from;
		const T* dy = a.dy + row * a.lddy + from;
		const T m = (T) a.stats[5 * row], c = (T) a.stats[5 * row + 1], r = (T) a.stats[5 * row + 2];
		T sg = 0, sh = 0;
#pragma unroll
		for (uint32_t j = 0; j < CHUNK_VECS; ++j)
		{
			const uint32_t col = (j * 256 + threadIdx.x) * VN<T>;
			if (col >= count) { break; }
			const V v = load_vec<T,true>(x, col, count);
			const V w = a.weight ? load_vec<T,true>(a.weight + from, col, count) : V{} + (T) 1;
			V g = load_vec<T,true>(dy, col, count); // zero past the end
#pragma unroll
			for (int i = 0; i < VN<T>; ++i)
			{
				if (false == in_row<T,true>(col, i, count)) { continue; }
				g[i] *= w[i];
				sg += g[i];
				sh += g[i] * (((v[i] - m) - c) * r);
			}
		}
		row_sums<T,256>(sg, sh, red, turn);
		if (threadIdx.x == 0)
		{
			a.sums[3 * at] = sg;
			a.sums[3 * at + 1] = sh;
		}
	}
}

template <typename T>
__global__ __launch_bounds__(256) void layer_norm_chunk_grad_merge_k (ChunkArgs<T> a)
{
	const uint64_t row = (uint64_t) blockIdx.x * 256 + threadIdx.x;
	if (row >= a.rows) { return; }
	double sg = 0, sh = 0;
	for (uint32_t k = 0; k < a.chunks; ++k)
	{
		sg += a.sums[3 * (row * a.chunks + k)];
		sh += a.sums[3 * (row * a.chunks + k) + 1];
	}
	a.stats[5 * row + 3] = sg / (double) a.cols;
	a.stats[5 * row + 4] = sh / (double) a.cols;
}

template <typename T>
__global__ __launch_bounds__(256) void layer_norm_chunk_dx_k (ChunkArgs<T> a)
{
	using V = typename Vec16<T>::type;
	for (uint64_t at = blockIdx.x; at < a.rows * a.chunks; at += gridDim.x)
	{
		uint64_t row, from;
		uint32_t count;
		chunk_place(a, at, row, from, count);
		const T* x = a.x + row * a.ldx + from;
		const T* dy = a.dy + row * a.lddy + from;
		T* dx = a.out + row * a.ldo + from;
		const T m = (T) a.stats[5 * row], c = (T) a.stats[5 * row + 1], r = (T) a.stats[5 * row + 2];
		const T sg = (T) a.stats[5 * row + 3], sh = (T) a.stats[5 * row + 4];
#pragma unroll
		for (uint32_t j = 0; j < CHUNK_VECS; ++j)
		{
			const uint32_t col = (j * 256 + threadIdx.x) * VN<T>;
			if (col >= count) { break; }
			const V v = load_vec<T,true>(x, col, count);
			const V g = load_vec<T,true>(dy, col, count);
			const V w = a.weight ? load_vec<T,true>(a.weight + from, col, count) : V{} + (T) 1;
			V out;
#pragma unroll
			for (int i = 0; i < VN<T>; ++i) { out[i] = r * (g[i] * w[i] - sg - ((v[i] - m) - c) * r * sh); }
			store_vec<T,true>(dx, col, count, out);
		}
	}
}

// Partial rows of dw and db: workgroup (x, y) sums 256 columns over every
// gridDim.y-th row
template <typename T>
__global__ __launch_bounds__(256) void layer_norm_chunk_params_k (ChunkArgs<T> a, T* partial)
{
	for (uint64_t col = (uint64_t) blockIdx.x * 256 + threadIdx.x; col < a.cols; col += (uint64_t) gridDim.x * 256)
	{
		T dw = 0, db = 0;
		for (uint64_t row = blockIdx.y; row < a.rows; row += gridDim.y)
		{
			const T g = a.dy[row * a.lddy + col];
			const T m = (T) a.stats[5 * row], c = (T) a.stats[5 * row + 1], r = (T) a.stats[5 * row + 2];
			dw += g * (((a.x[row * a.ldx + col] - m) - c) * r);
			db += g;
		}
		partial[(uint64_t) blockIdx.y * 2 * a.cols + col] = dw;
		partial[(uint64_t) blockIdx.y * 2 * a.cols + a.cols + col] = db;
	}
}

template <typename T>
__global__ __launch_bounds__(256) void layer_norm_chunk_params_sum_k (const T* partial, uint32_t parts, uint64_t cols, T* dweight, T* dbias)
{
	for (uint64_t col = (uint64_t) blockIdx.x * 256 + threadIdx.x; col < 2 * cols; col += (uint64_t) gridDim.x * 256)
	{
		T sum = 0;
		for (uint32_t p = 0; p < parts; ++p) { sum += partial[p * 2 * cols + col]; }
		T* out = col < cols ? dweight : dbias;
		if (out) { out[col < cols ? col : col - cols] = sum; }
	}
}

// ---- launches --------------------------------------------------------------------

/// Lanes a row is spread over and vectors a lane holds: the fewest lanes that hold it
/// in `per_most` vectors.  Fewer than a wave for the shortest rows only (60000 x 64
/// forward with a wave a row: 15 us, three lanes of four idle).
struct RowShape
{
	int span = 0; // 0: too long for registers
	int per = 0;
};

template <typename T>
RowShape row_shape (uint64_t cols, int per_most)
{
	const uint64_t vecs = (cols + VN<T> - 1) / VN<T>;
	if (vecs <= 16) { return {16, 1}; }
	if (vecs <= 32) { return {32, 1}; }
	for (int span : {64, 256, 1024})
	{
		for (int per = 1; per <= per_most; per *= 2)
		{
			if (vecs <= (uint64_t) span * per) { return {span, per}; }
		}
	}
	return {};
}

template <typename T, int SPAN, int PER>
void norm_launch (tcg_ctx* ctx, const NormArgs<T>& a)
{
	const uint64_t groups = (a.rows + rows_at_once(SPAN) - 1) / rows_at_once(SPAN);
	const uint64_t most = (uint64_t) ctx->num_cus * 32;
	const unsigned grid = (unsigned) (groups < most ? groups : most);
	if (a.cols % VN<T>) { layer_norm_k<T,SPAN,PER,true><<<grid, group_size(SPAN), 0, ctx->stream>>>(a); }
	else { layer_norm_k<T,SPAN,PER,false><<<grid, group_size(SPAN), 0, ctx->stream>>>(a); }
}

template <typename T, int SPAN>
void norm_launch_per (tcg_ctx* ctx, const NormArgs<T>& a, int per)
{
	switch (per)
	{
		case 1: norm_launch<T,SPAN,1>(ctx, a); break;
		case 2: norm_launch<T,SPAN,2>(ctx, a); break;
		case 8: // the longest rows only, see norm_run
			if constexpr (SPAN == 1024) { norm_launch<T,SPAN,8>(ctx, a); break; }
		default: norm_launch<T,SPAN,4>(ctx, a); break;
	}
}

template <typename T, int SPAN, int PER, bool RAGGED, bool ONCE>
void grad_launch_once (tcg_ctx* ctx, const GradArgs<T>& a, unsigned grid)
{
	constexpr unsigned threads = group_size(SPAN);
	if (a.dx && a.partial) { layer_norm_grad_k<T,SPAN,PER,RAGGED,true,true,ONCE><<<grid, threads, 0, ctx->stream>>>(a); }
	else if (a.dx) { layer_norm_grad_k<T,SPAN,PER,RAGGED,true,false,ONCE><<<grid, threads, 0, ctx->stream>>>(a); }
	else { layer_norm_grad_k<T,SPAN,PER,RAGGED,false,true,ONCE><<<grid, threads, 0, ctx->stream>>>(a); }
}

// 32768 x 4096 (1.6 GB): 264 us with the hint for memory used once, 293 without; 16384 x 2048
// (400 MB): 69 and 75; 16384 x 1024 (200 MB, in the caches at the next call): 38 and 35.5.
// Forward it costs as much as it gives (4096 x 16384 126 and 117, 32768 x 4096 180 and 187).
constexpr uint64_t CACHES = 256ull << 20;

template <typename T, int SPAN, int PER, bool RAGGED>
void grad_launch (tcg_ctx* ctx, const GradArgs<T>& a, unsigned grid)
{
	if ((a.dx ? 3 : 2) * a.rows * a.cols * sizeof(T) > CACHES) { grad_launch_once<T,SPAN,PER,RAGGED,true>(ctx, a, grid); }
	else { grad_launch_once<T,SPAN,PER,RAGGED,false>(ctx, a, grid); }
}

template <typename T, int SPAN>
void grad_launch_one (tcg_ctx* ctx, const GradArgs<T>& a, unsigned grid)
{
	if (a.cols % VN<T>) { grad_launch<T,SPAN,1,true>(ctx, a, grid); }
	else { grad_launch<T,SPAN,1,false>(ctx, a, grid); }
}

template <typename T, int SPAN>
void grad_launch_per (tcg_ctx* ctx, const GradArgs<T>& a, int per, unsigned grid)
{
	const bool ragged = a.cols % VN<T>;
	switch (per)
	{
		case 1: if (ragged) { grad_launch<T,SPAN,1,true>(ctx, a, grid); } else { grad_launch<T,SPAN,1,false>(ctx, a, grid); } break;
		case 2: if (ragged) { grad_launch<T,SPAN,2,true>(ctx, a, grid); } else { grad_launch<T,SPAN,2,false>(ctx, a, grid); } break;
		default: if (ragged) { grad_launch<T,SPAN,4,true>(ctx, a, grid); } else { grad_launch<T,SPAN,4,false>(ctx, a, grid); } break;
	}
}

template <typename T, int SPAN, int PER>
void grad_few_launch (tcg_ctx* ctx, const GradArgs<T>& a, T* dweight, T* dbias)
{
	const unsigned strips = (unsigned) ((a.cols + 4 * VN<T> - 1) / (4 * VN<T>));
	const unsigned grid = strips + (unsigned) ((a.rows + rows_at_once(SPAN) - 1) / rows_at_once(SPAN));
	if (a.cols % VN<T>) { layer_norm_grad_few_k<T,SPAN,PER,true><<<grid, 256, 0, ctx->stream>>>(a, strips, dweight, dbias); }
	else { layer_norm_grad_few_k<T,SPAN,PER,false><<<grid, 256, 0, ctx->stream>>>(a, strips, dweight, dbias); }
}

template <typename T, int SPAN>
void grad_few_launch_per (tcg_ctx* ctx, const GradArgs<T>& a, int per, T* dweight, T* dbias)
{
	switch (per)
	{
		case 1: grad_few_launch<T,SPAN,1>(ctx, a, dweight, dbias); break;
		case 2: grad_few_launch<T,SPAN,2>(ctx, a, dweight, dbias); break;
		default: grad_few_launch<T,SPAN,4>(ctx, a, dweight, dbias); break;
	}
}

/// Grid of a kernel that walks rows x chunks
unsigned chunk_grid (const tcg_ctx* ctx, uint64_t work)
{
	const uint64_t most = (uint64_t) ctx->num_cus * 32;
	return (unsigned) (work < most ? work : most);
}

template <typename T>
void chunk_setup (ChunkArgs<T>& a, size_t& sums_bytes, size_t& stats_bytes)
{
	a.chunks = (uint32_t) ((a.cols + CHUNK<T> - 1) / CHUNK<T>);
	sums_bytes = a.rows * a.chunks * 3 * sizeof(double);
	stats_bytes = a.rows * 5 * sizeof(double);
}

template <typename T>
int norm_chunked (tcg_ctx* ctx, const NormArgs<T>& n, uint64_t cols, double eps)
{
	ChunkArgs<T> a = {};
	a.x = n.x; a.ldx = n.ldx;
	a.weight = n.weight; a.bias = n.bias;
	a.out = n.y; a.ldo = n.ldy;
	a.mean = n.mean; a.rstd = n.rstd;
	a.rows = n.rows; a.cols = cols; a.eps = eps;
	size_t sums_bytes, stats_bytes;
	chunk_setup(a, sums_bytes, stats_bytes);
	void* mem = nullptr;
	int rc = tcg_alloc(ctx, sums_bytes + stats_bytes, &mem);
	if (rc != TCG_OK) { return rc; }
	a.stats = (double*) mem;
	a.sums = a.stats + 5 * a.rows;
	const unsigned grid = chunk_grid(ctx, a.rows * a.chunks);
	layer_norm_chunk_stats_k<T><<<grid, 256, 0, ctx->stream>>>(a);
	layer_norm_chunk_merge_k<T><<<(unsigned) ((a.rows + 255) / 256), 256, 0, ctx->stream>>>(a);
	layer_norm_chunk_apply_k<T><<<grid, 256, 0, ctx->stream>>>(a);
	hipError_t err = hipGetLastError();
	rc = tcg_free(ctx, mem, sums_bytes + stats_bytes);
	if (err != hipSuccess) { return tcg_fail(ctx, TCG_ERR_HIP, "launch of layer_norm failed: %s", hipGetErrorString(err)); }
	return rc;
}

template <typename T>
int grad_chunked (tcg_ctx* ctx, const GradArgs<T>& g, uint64_t cols, double eps, T* dweight, T* dbias)
{
	ChunkArgs<T> a = {};
	a.x = g.x; a.ldx = g.ldx;
	a.dy = g.dy; a.lddy = g.lddy;
	a.weight = g.weight;
	a.out = g.dx; a.ldo = g.lddx;
	a.mean_in = g.mean; a.rstd_in = g.rstd;
	a.rows = g.rows; a.cols = cols; a.eps = eps;
	size_t sums_bytes, stats_bytes, partial_bytes = 0;
	chunk_setup(a, sums_bytes, stats_bytes);
	uint32_t parts = 0;
	if (dweight || dbias)
	{
		parts = (uint32_t) (a.rows < 16 ? a.rows : a.rows < 16 * 64 ? 16 : a.rows < 128 * 64 ? a.rows / 64 : 128);
		partial_bytes = (size_t) parts * 2 * cols * sizeof(T);
	}
	void* mem = nullptr;
	const size_t bytes = sums_bytes + stats_bytes + partial_bytes;
	int rc = tcg_alloc(ctx, bytes, &mem);
	if (rc != TCG_OK) { return rc; }
	a.stats = (double*) mem;
	a.sums = a.stats + 5 * a.rows;
	T* partial = (T*) (a.sums + 3 * a.rows * a.chunks);
	const unsigned grid = chunk_grid(ctx, a.rows * a.chunks);
	const unsigned row_grid = (unsigned) ((a.rows + 255) / 256);
	if (nullptr == a.mean_in) { layer_norm_chunk_stats_k<T><<<grid, 256, 0, ctx->stream>>>(a); }
	layer_norm_chunk_merge_k<T><<<row_grid, 256, 0, ctx->stream>>>(a);
	// the sums over rows before dx, which may lie where dy or x does, and their results after
	// it: these may lie where the weight does
	if (parts) { layer_norm_chunk_params_k<T><<<dim3(chunk_grid(ctx, (cols + 255) / 256), parts), 256, 0, ctx->stream>>>(a, partial); }
	if (a.out)
	{
		layer_norm_chunk_grad_sums_k<T><<<grid, 256, 0, ctx->stream>>>(a);
		layer_norm_chunk_grad_merge_k<T><<<row_grid, 256, 0, ctx->stream>>>(a);
		layer_norm_chunk_dx_k<T><<<grid, 256, 0, ctx->stream>>>(a);
	}
	if (parts)
	{
		layer_norm_chunk_params_sum_k<T><<<chunk_grid(ctx, (2 * cols + 255) / 256), 256, 0, ctx->stream>>>(partial, parts, cols, dweight, dbias);
	}
	hipError_t err = hipGetLastError();
	rc = tcg_free(ctx, mem, bytes);
	if (err != hipSuccess) { return tcg_fail(ctx, TCG_ERR_HIP, "launch of layer_norm_grad failed: %s", hipGetErrorString(err)); }
	return rc;
}

template <typename T>
int norm_run (tcg_ctx* ctx, uint64_t rows, uint64_t cols, const void* x, uint64_t ldx, const void* weight, const void* bias,
	double eps, void* y, uint64_t ldy, void* mean, void* rstd)
{
	NormArgs<T> a = {};
	a.x = (const T*) x; a.ldx = ldx;
	a.weight = (const T*) weight; a.bias = (const T*) bias;
	a.y = (T*) y; a.ldy = ldy;
	a.mean = (T*) mean; a.rstd = (T*) rstd;
	a.rows = rows;
	// (four vectors a lane: eight, with a wave for 1537 elements, took 13.5 us for 4099 rows
	// instead of 12.3)
	RowShape shape = row_shape<T>(cols, 4);
	if (0 == shape.span) { shape = row_shape<T>(cols, 8); }
	if (0 == shape.span) { return norm_chunked(ctx, a, cols, eps); }
	a.cols = (uint32_t) cols;
	a.eps = (T) eps;
	a.n = (T) cols;
	a.inv_n = (T) (1. / (double) cols);
	switch (shape.span)
	{
		case 16: norm_launch<T,16,1>(ctx, a); break;
		case 32: norm_launch<T,32,1>(ctx, a); break;
		case 64: norm_launch_per<T,64>(ctx, a, shape.per); break;
		case 256: norm_launch_per<T,256>(ctx, a, shape.per); break;
		default: norm_launch_per<T,1024>(ctx, a, shape.per); break;
	}
	TCG_LAUNCH_CHECK(ctx, "layer_norm");
	return TCG_OK;
}

// All gradients in one launch, and in two, calls one behind the other (us): 256 x 64 5.7 and
// 8.0, 768 x 512 5.8 and 8.1, 768 x 777 5.2 and 8.8, 500 x 4096 9.7 and 16.2, 768 x 4096 13.0 and
// 14.5, but 768 x 2048 10.9 and 10.1.  Beyond: 1024 x 64 6.3 and 8.0, 1024 x 512 6.7 and 8.2,
// 1500 x 512 8.7 and 8.6, 1500 x 777 10.1 and 10.5, but 1024 x 2048 14.2 and 11.6, 1024 x 4096
// 16.9 and 15.9, 2048 x 64 9.5 and 8.0: the two cross near 700 rows of 2048 elements and 1500
// of 512, and one number of rows stands for all of them.  Rows of 1024 lanes are left to two
// launches: 200 x 8192 would be 8.7 and 13.1, but 768 x 8192 26 and 20, 500 x 16000 36 and 30.
constexpr uint64_t FEW_ROWS = 768;

template <typename T>
int grad_run (tcg_ctx* ctx, uint64_t rows, uint64_t cols, const void* dy, uint64_t lddy, const void* x, uint64_t ldx,
	const void* weight, const void* mean, const void* rstd, double eps, void* dx, uint64_t lddx, void* dweight, void* dbias)
{
	GradArgs<T> a = {};
	a.dy = (const T*) dy; a.lddy = lddy;
	a.x = (const T*) x; a.ldx = ldx;
	a.weight = (const T*) weight;
	a.mean = (const T*) mean; a.rstd = (const T*) rstd;
	a.dx = (T*) dx; a.lddx = lddx;
	a.rows = rows;
	const RowShape shape = row_shape<T>(cols, 4);
	if (0 == shape.span) { return grad_chunked(ctx, a, cols, eps, (T*) dweight, (T*) dbias); }
	a.cols = (uint32_t) cols;
	a.eps = (T) eps;
	a.n = (T) cols;
	a.inv_n = (T) (1. / (double) cols);
	// one launch for a few rows; dx must not lie where dw's sums still read, nor dw or db where
	// dx still reads the weight
	const auto beside_weight = [&] (const void* p)
	{
		const uintptr_t at = (uintptr_t) p, w = (uintptr_t) weight, bytes = cols * sizeof(T);
		return !p || !weight || (at > w ? at - w : w - at) >= bytes;
	};
	if (dx && (dweight || dbias) && mean && dx != x && dx != dy && beside_weight(dweight) && beside_weight(dbias) &&
		cols >= VN<T> && shape.span <= 256 && rows <= FEW_ROWS)
	{
		switch (shape.span)
		{
			case 16: grad_few_launch<T,16,1>(ctx, a, (T*) dweight, (T*) dbias); break;
			case 32: grad_few_launch<T,32,1>(ctx, a, (T*) dweight, (T*) dbias); break;
			case 64: grad_few_launch_per<T,64>(ctx, a, shape.per, (T*) dweight, (T*) dbias); break;
			default: grad_few_launch_per<T,256>(ctx, a, shape.per, (T*) dweight, (T*) dbias); break;
		}
		hipError_t err = hipGetLastError();
		return err == hipSuccess ? TCG_OK : tcg_fail(ctx, TCG_ERR_HIP, "launch of layer_norm_grad failed: %s", hipGetErrorString(err));
	}
	const uint64_t at_once = rows_at_once(shape.span), groups = (rows + at_once - 1) / at_once;
	const bool params = dweight || dbias;
	// with the sums over rows every workgroup leaves a partial row behind: no more of them
	// than fill the chip.  One, two, three and four a CU (us): 3000 x 512 8.9 9.3 10.1 10.1, 8000 x
	// 512 14.8 14.1 13.9 15.2, 3000 x 777 13.0 12.8 14.2 14.3, 8000 x 777 24.4 22.5 21.1 25.9, 3000
	// x 2048 20.7 19.0 19.5 20.0, 16384 x 1024 37.7 35.6 36.4 37.1, 32768 x 4096 313 264 295 288
	const uint64_t most = (uint64_t) ctx->num_cus * (params ? (shape.span == 1024 ? 1 : 2) : 32);
	// as many workgroups as make equal shares of the rows
	const uint64_t share = (groups + most - 1) / most;
	const unsigned grid = (unsigned) ((groups + share - 1) / share);
	const size_t bytes = params ? (size_t) grid * 2 * cols * sizeof(T) : 0;
	void* mem = nullptr;
	if (params)
	{
		int rc = tcg_alloc(ctx, bytes, &mem);
		if (rc != TCG_OK) { return rc; }
		a.partial = (T*) mem;
	}
	switch (shape.span)
	{
		case 16: grad_launch_one<T,16>(ctx, a, grid); break;
		case 32: grad_launch_one<T,32>(ctx, a, grid); break;
		case 64: grad_launch_per<T,64>(ctx, a, shape.per, grid); break;
		case 256: grad_launch_per<T,256>(ctx, a, shape.per, grid); break;
		default: grad_launch_per<T,1024>(ctx, a, shape.per, grid); break;
	}
	if (params)
	{
		const unsigned strips = (unsigned) ((2 * cols + 31) / 32);
		layer_norm_params_k<T><<<strips, 1024, 0, ctx->stream>>>(a.partial, grid, a.cols, (T*) dweight, (T*) dbias);
	}
	hipError_t err = hipGetLastError();
	int rc = params ? tcg_free(ctx, mem, bytes) : TCG_OK;
	if (err != hipSuccess) { return tcg_fail(ctx, TCG_ERR_HIP, "launch of layer_norm_grad failed: %s", hipGetErrorString(err)); }
	return rc;
}

// rows x ld elements have to be addressable; the chunked path's temporaries follow
constexpr uint64_t MOST_ELEMENTS = 1ull << 40;

bool sizes_fit (uint64_t rows, uint64_t ld)
{
	return ld == 0 || rows <= MOST_ELEMENTS / ld;
}

/// An epsilon above zero stays above zero in the type of the rows
double kept_eps (int dtype, double eps)
{
	const double least = std::numeric_limits<float>::denorm_min();
	return dtype == TCG_FLOAT && eps > 0 && eps < least ? least : eps;
}

} // namespace

extern "C" {

int tcg_layer_norm (tcg_ctx* ctx, int dtype, uint64_t rows, uint64_t cols, const void* x, uint64_t ldx,
	const void* weight, const void* bias, double eps, void* y, uint64_t ldy, void* mean, void* rstd)
{
	if (!ctx) { return TCG_ERR_ARG; }
	TCG_REQUIRE(ctx, dtype == TCG_FLOAT || dtype == TCG_DOUBLE, "tcg_layer_norm: dtype %d is neither float nor double", dtype);
	TCG_REQUIRE(ctx, cols > 0, "tcg_layer_norm: a row of no elements has no mean");
	TCG_REQUIRE(ctx, ldx >= cols && ldy >= cols, "tcg_layer_norm: leading dims %llu and %llu of rows of %llu elements",
		(unsigned long long) ldx, (unsigned long long) ldy, (unsigned long long) cols);
	TCG_REQUIRE(ctx, sizes_fit(rows, ldx) && sizes_fit(rows, ldy), "tcg_layer_norm: %llu rows are too many", (unsigned long long) rows);
	TCG_REQUIRE(ctx, eps >= 0, "tcg_layer_norm: eps %g is negative or not a number", eps);
	TCG_REQUIRE(ctx, (nullptr == mean) == (nullptr == rstd), "tcg_layer_norm: mean and rstd are wanted together or not at all");
	TCG_REQUIRE(ctx, 0 == rows || (x && y), "tcg_layer_norm: NULL pointer");
	TCG_REQUIRE(ctx, x != y || ldx == ldy, "tcg_layer_norm: in place with leading dims %llu and %llu",
		(unsigned long long) ldx, (unsigned long long) ldy);
	if (tcg_small_mode(ctx)) { TCG_SMALL_RETURN(ctx, tcg_small_unsupported(ctx, "a layer normalisation")); }
	if (0 == rows) { return TCG_OK; }
	eps = kept_eps(dtype, eps);
	tcg_device_scope device(ctx);
	return dtype == TCG_FLOAT ? norm_run<float>(ctx, rows, cols, x, ldx, weight, bias, eps, y, ldy, mean, rstd) :
		norm_run<double>(ctx, rows, cols, x, ldx, weight, bias, eps, y, ldy, mean, rstd);
}

int tcg_layer_norm_grad (tcg_ctx* ctx, int dtype, uint64_t rows, uint64_t cols, const void* dy, uint64_t lddy,
	const void* x, uint64_t ldx, const void* weight, const void* mean, const void* rstd, double eps,
	void* dx, uint64_t lddx, void* dweight, void* dbias)
{
	if (!ctx) { return TCG_ERR_ARG; }
	TCG_REQUIRE(ctx, dtype == TCG_FLOAT || dtype == TCG_DOUBLE, "tcg_layer_norm_grad: dtype %d is neither float nor double", dtype);
	TCG_REQUIRE(ctx, cols > 0, "tcg_layer_norm_grad: a row of no elements has no mean");
	TCG_REQUIRE(ctx, lddy >= cols && ldx >= cols && (!dx || lddx >= cols),
		"tcg_layer_norm_grad: leading dims %llu, %llu and %llu of rows of %llu elements",
		(unsigned long long) lddy, (unsigned long long) ldx, (unsigned long long) lddx, (unsigned long long) cols);
	TCG_REQUIRE(ctx, sizes_fit(rows, ldx) && sizes_fit(rows, lddy) && (!dx || sizes_fit(rows, lddx)),
		"tcg_layer_norm_grad: %llu rows are too many", (unsigned long long) rows);
	TCG_REQUIRE(ctx, eps >= 0, "tcg_layer_norm_grad: eps %g is negative or not a number", eps);
	TCG_REQUIRE(ctx, (nullptr == mean) == (nullptr == rstd), "tcg_layer_norm_grad: mean and rstd are given together or not at all");
	TCG_REQUIRE(ctx, dx || dweight || dbias, "tcg_layer_norm_grad: no gradient is wanted");
	TCG_REQUIRE(ctx, 0 == rows || (x && dy), "tcg_layer_norm_grad: NULL pointer");
	TCG_REQUIRE(ctx, !dx || ((dx != dy || lddx == lddy) && (dx != x || lddx == ldx)),
		"tcg_layer_norm_grad: dx in place of an operand with another leading dim");
	if (tcg_small_mode(ctx)) { TCG_SMALL_RETURN(ctx, tcg_small_unsupported(ctx, "the gradients of a layer normalisation")); }
	eps = kept_eps(dtype, eps);
	tcg_device_scope device(ctx);
	if (0 == rows)
	{
		// sums over no rows
		int rc = dweight ? tcg_fill_zero(ctx, dweight, cols * tcg_type_size(dtype)) : TCG_OK;
		return rc == TCG_OK && dbias ? tcg_fill_zero(ctx, dbias, cols * tcg_type_size(dtype)) : rc;
	}
	return dtype == TCG_FLOAT ?
		grad_run<float>(ctx, rows, cols, dy, lddy, x, ldx, weight, mean, rstd, eps, dx, lddx, dweight, dbias) :
		grad_run<double>(ctx, rows, cols, dy, lddy, x, ldx, weight, mean, rstd, eps, dx, lddx, dweight, dbias);
}

} // extern "C"
