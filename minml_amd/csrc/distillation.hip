/*
 * distillation.hip — the distillation of a teacher into a last dense layer over many classes, from the layer's input and the teacher's top logits of every row, and its gradients. Neither the logits of the student nor a
 * distribution over all classes is ever kept.
 *
 *   z = (x W^T + b) / t,   lse[i] = log sum_j exp z[i, j],   log p[i, k] = z[i, c[i, k]] - lse[i]
 *   q[i, k] = softmax over k of v[i, k] / t,   loss[i] = sum_k q[i, k] (log q[i, k] - log p[i, k])
 *   d[i, j] = (exp(z[i, j] - lse[i]) - sum over k with c[i, k] = j of q[i, k]) dloss[i] / t,   dx = d W,   dW = d^T x,   db[j] = sum_i d[i, j]
 *
 * q is of (v - largest v) / t: of v / t the rounding alone would be off by |v / t| 2^-24, and at a small t it is no number of fp32.
 * A place k whose class c is none of the layer's, or whose logit v is -inf, does not count; a row without any that does has loss 0 and no gradient. A class that a row names twice has the sum of both probabilities.
 * The passes are the cross entropy's (vocabulary_loss.hpp). What is new is that a row has many classes of its own, spread over the tiles of logits. A launch before sorts every row's classes and notes where each column of tiles
 * begins among them; then one thread of a tile has a row's few in that tile, and they meet the logits in LDS, through which the tile goes anyway in the backward pass, and in the forward pass where it has any.
 * In the backward pass the student's probability at these places is known from the forward pass's log p, so that d there is p - q in fp32, rounded once, however close p and q are. In fp16, what rounding takes from d's rows is given back to the row of W with the teacher's largest share, as much as is its own, and
 * the rest to the mean of rows that teachers name: dx is 2.3e-4 to 2.8e-4 off (norm), of which its own rounding is 2.1e-4; 2 to 4 us more than all of it to one class (3964 / 3974 of 4096 x 2048 x 65536, 135.7 / 139.5 of 400 x 1024 x 10000).
 * Up to 64 rows d's low parts are kept (see LOW_ROWS).
 * fp16, what it takes beside the cross entropy of the same size: 2048 rows of 1024 x 50001, 32 classes a row, 245 to 267 us, card to card (the products 257 / 246, sorting 8); 4096 of 2048 x 65536, 64 classes, loss and gradients
 * 3.96 to 4.05 ms (products 1030 / 1003, making d 562 / 560 twice, sorting 12 twice). 3 rows of 1024 x 32000 18.5 us (14.2 at 4.6 TB/s, 5.2 to join). What bounds the rest is said there.
 */
#include "vocabulary_loss.hpp"

#include <cmath>

namespace
{
	using namespace mlhip;

	constexpr int MOST_CLASSES_OF_ROW = 1024;

	/* ---- the teacher's classes ---------------------------------------------------------------------------------------------- */
	/* what a row's classes look like in order */
	struct Teaching
	{
			int *classes; /* [rows][count], ascending; those that do not count behind all others */
			uint16_t *places; /* [rows][count]: where they stand in the caller's order */
			float *shares; /* [rows][count]: the class's probability, at its first place if the row names it twice, else 0 */
			float *known; /* backward, [rows][count]: the student's probability */
			uint16_t *begins; /* [rows][column tiles + 1]: how many of them lie before a column of tiles */
			int *anchors; /* [rows]: the class with the largest share, -1 where none counts */
			float *entropies; /* forward, [rows]: sum of q log q */
			float *own, *there; /* backward in fp16, [rows] and one: zeros, and whether there is a common row */
			half_t *common; /* [features in whole tiles]: what rows of the weights have in common */
	};
	/* whole vectors of four */
	__host__ __device__ inline int places_in_lds(int count)
	{
		return (count + 3) / 4 * 4;
	}
	template<typename V>
	__device__ __forceinline__ V lanes_max(V v)
	{
#pragma unroll
		for (int offset = 32; offset >= 1; offset >>= 1)
			v = max(v, __shfl_xor(v, offset));
		return v;
	}
	/*
	 * The mean of up to 64 of the teacher's classes' rows of weights, taken evenly over what it names; one of four places that counts, for each. A class that the teacher names is one that the model is trained for, whose row of W
	 * looks like those that d is large at. It is kept in fp16, where a row of W is: whatever row it is, what is given back to it is taken from it as it stands, so its own rounding is no error of dx. Columns behind the features: zeros. 64 columns to a workgroup, 16 rows to a wavefront
	 */
	constexpr int COMMON_ROWS = 64, COMMON_COLUMNS = 256; /* COMMON_COLUMNS: the widest tile's, which reads them without asking where they end */
	template<typename L>
	__device__ __forceinline__ void common_row(const int *classes_in, const L *logits, size_t places, int classes, const half_t *w, int features, int column0, half_t *common, float *there)
	{
		__shared__ int named[4][COMMON_ROWS];
		__shared__ float sums[4][64];
		const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
		const size_t asked = min(places, static_cast<size_t>(4 * COMMON_ROWS));
		named[wave][lane] = -1;
		if (threadIdx.x < asked)
		{
			const size_t place = threadIdx.x * places / asked;
			const int c = classes_in[place];
			if (c >= 0 && c < classes && !(static_cast<float>(logits[place]) == -std::numeric_limits<float>::infinity()))
				named[wave][lane] = c;
		}
		__syncthreads();
		int mine = -1; /* of the lane's four places */
#pragma unroll
		for (int k = 3; k >= 0; k--)
			mine = named[k][lane] >= 0 ? named[k][lane] : mine;
		const int rows = __popcll(__ballot(mine >= 0)), column = column0 + lane;
		float v[COMMON_ROWS / 4];
#pragma unroll
		for (int u = 0; u < COMMON_ROWS / 4; u++)
		{
			const int c = __shfl(mine, wave * (COMMON_ROWS / 4) + u);
			v[u] = c >= 0 && column < features ? static_cast<float>(w[static_cast<size_t>(c) * features + column]) : 0.0f;
		}
		float sum = 0.0f;
#pragma unroll
		for (int u = 0; u < COMMON_ROWS / 4; u++)
			sum += v[u];
		sums[wave][lane] = sum;
		__syncthreads();
		if (wave == 0)
			common[column] = static_cast<half_t>((sums[0][lane] + sums[1][lane] + sums[2][lane] + sums[3][lane]) / static_cast<float>(max(rows, 1)));
		if (column0 == 0 && threadIdx.x == 0)
			*there = rows > 0 ? 1.0f : 0.0f;
	}
	/* a wavefront per row from first_row on; workgroups behind the rows': common_row. What a class's place is, is counted: as many classes are smaller, or equal and named before. L: type of the logits */
	template<typename L>
	__global__ __launch_bounds__(256) void kernel_sort_teacher(const int *classes_in, const L *logits, const float *log_probabilities, int first_row, int groups, int rows, int count, int classes, float temperature, int width, int tiles, const half_t *w,
			int features, Teaching out)
	{
		extern __shared__ __attribute__((aligned(16))) int memory[];
		if (static_cast<int>(blockIdx.x) >= groups)
			return common_row(classes_in, logits, static_cast<size_t>(rows) * count, classes, w, features, (static_cast<int>(blockIdx.x) - groups) * 64, out.common, out.there);
		const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = first_row + static_cast<int>(blockIdx.x) * 4 + wave;
		if (row >= rows)
			return;
		const int stride = places_in_lds(count);
		int *named = memory + wave * 4 * stride, *sorted = named + stride;
		float *values = reinterpret_cast<float*>(sorted + stride), *shares = values + stride;
		const size_t base = static_cast<size_t>(row) * count;
		float top = -std::numeric_limits<float>::infinity();
		int there = 0, missing = 0;
		for (int k0 = 0; k0 < stride; k0 += 64)
		{
			const int k = k0 + lane;
			const int c = k < count ? classes_in[base + k] : -1;
			const float v = k < count ? static_cast<float>(logits[base + k]) : 0.0f;
			const bool counts = c >= 0 && c < classes && !(v == -std::numeric_limits<float>::infinity());
			const uint64_t all = __ballot(counts), none = __ballot(k < count && !counts);
			if (k < stride)
			{
				named[k] = counts ? c : 0x7fffffff;
				/* of one that does not count: how many others before do not either */
				values[k] = counts ? v : __int_as_float(missing + __popcll(none & ((1ull << lane) - 1)));
			}
			top = counts ? fmaxf(top, v) : top;
			there += __popcll(all);
			missing += __popcll(none);
		}
		top = lanes_max(top);
		__builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
		float sum = 0.0f;
		for (int k = lane; k < count; k += 64)
			if (named[k] != 0x7fffffff)
			{
				values[k] = expf((values[k] - top) / temperature);
				sum += values[k];
			}
		sum = lanes_sum<64>(sum);
		__builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
		for (int k = lane; k < count; k += 64)
		{
			const int c = named[k];
			int place = 0;
#pragma unroll 4
			for (int other = 0; other < stride; other += 4)
			{
				typedef int int4_t __attribute__((ext_vector_type(4)));
				const int4_t n = *reinterpret_cast<const int4_t*>(named + other);
#pragma unroll
				for (int e = 0; e < 4; e++)
					place += static_cast<uint32_t>(n[e]) < static_cast<uint32_t>(c) + (other + e < k ? 1 : 0) ? 1 : 0;
			}
			if (c == 0x7fffffff)
				place = there + __float_as_int(values[k]);
			sorted[place] = c;
			shares[place] = c == 0x7fffffff ? 0.0f : values[k] / sum;
			out.places[base + place] = static_cast<uint16_t>(k);
			if (log_probabilities != nullptr)
				out.known[base + place] = expf(log_probabilities[base + k]);
		}
		__builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
		float entropy = 0.0f, best = -1.0f;
		int best_at = there > 0 ? 0 : -1;
		for (int p = lane; p < count; p += 64)
		{
			const int c = sorted[p];
			float share = 0.0f;
			if (p < there)
			{
				if (p == 0 || sorted[p - 1] != c)
				{
					for (int e = p; e < there && sorted[e] == c; e++)
						share += shares[e];
					entropy += share > 0.0f ? share * logf(share) : share;
					if (share > best)
					{
						best = share;
						best_at = p;
					}
				}
			}
			out.classes[base + p] = c;
			out.shares[base + p] = share;
		}
		entropy = lanes_sum<64>(entropy);
		const float largest = lanes_max(best);
		const uint64_t has = __ballot(best == largest && best >= 0.0f);
		best_at = has != 0 ? __shfl(best_at, __ffsll(static_cast<unsigned long long>(has)) - 1) : best_at;
		if (lane == 0)
		{
			out.anchors[row] = best_at >= 0 ? sorted[best_at] : -1;
			if (log_probabilities == nullptr)
				out.entropies[row] = entropy;
			if (w != nullptr)
				out.own[row] = 0.0f;
		}
		/* several columns of tiles at a time, by halves of the row's classes: no read of LDS waits for another column's */
		constexpr int AT_A_TIME = 8;
		for (int t0 = lane; t0 <= tiles; t0 += 64 * AT_A_TIME)
		{
			int first[AT_A_TIME];
#pragma unroll
			for (int u = 0; u < AT_A_TIME; u++)
				first[u] = 0;
			for (int step = MOST_CLASSES_OF_ROW; step > 0; step >>= 1)
				if (step <= there)
#pragma unroll
					for (int u = 0; u < AT_A_TIME; u++)
					{
						const int t = t0 + 64 * u, next = first[u] + step;
						const bool below = sorted[min(next, there) - 1] < (t < tiles ? t * width : 0x7fffffff);
						first[u] = next <= there && below ? next : first[u];
					}
#pragma unroll
			for (int u = 0; u < AT_A_TIME; u++)
				if (t0 + 64 * u <= tiles)
					out.begins[static_cast<size_t>(row) * (tiles + 1) + t0 + 64 * u] = static_cast<uint16_t>(first[u]);
		}
	}

	/* ---- the goal: several classes of every row ------------------------------------------------------------------------------ */
	struct TopClasses
	{
			static constexpr bool ONE = false;
			static constexpr int FIXED_BITS = 38;
			const int *targets; /* none here */
			const int *classes;
			const float *shares, *known;
			const uint16_t *begins; /* from the piece's first column of tiles on */
			float *logits; /* forward: [rows][count] */
			int count, stride; /* stride: of begins */
			float slope; /* 1 / t */
			const int *anchors; /* backward: of every row the class whose part of what rounding took is kept for itself, in own; own null: of none */
			float *own;
			bool low; /* backward, of up to LOW_ROWS rows: d's low parts behind them */

			/*
			 * A thread's row of the tile and its classes there: first .. last - 1 of the row's, the first two of them with what is known of them. Asked for when the tile is complete, before anything is computed of it: the
			 * tile's end would wait for one load after another (us, so / when they are used: 2048 x 1024 x 50001 267 / 271, gradients of 4096 x 2048 x 65536 4050 / 4078)
			 */
			static constexpr int AHEAD = 2;
			struct OfTile
			{
					int row, m, first, last, anchor, named[AHEAD];
					float share[AHEAD], probability[AHEAD], factor;
			};
			template<bool BACKWARD, int BM, int BN>
			__device__ __forceinline__ OfTile classes_of(const TilePlace<BM, BN> &at, int rows, const float *factors) const
			{
				OfTile t;
				t.row = threadIdx.x;
				t.m = at.tile_m * BM + t.row;
				t.first = t.last = 0;
				t.anchor = -1;
				t.factor = 0.0f;
				if (t.row < BM && t.m < rows)
				{
					const uint16_t *of_row = begins + static_cast<size_t>(t.m) * stride + at.tile_n;
					t.first = of_row[0];
					t.last = of_row[1];
					if (BACKWARD)
					{
						t.factor = factors[t.m];
						t.last = t.factor != 0.0f ? t.last : t.first;
						if (own != nullptr)
							t.anchor = anchors[t.m];
					}
				}
#pragma unroll
				for (int u = 0; u < AHEAD; u++)
				{
					t.named[u] = 0;
					t.share[u] = t.probability[u] = 0.0f;
					if (t.first + u < t.last)
					{
						const size_t place = static_cast<size_t>(t.m) * count + t.first + u;
						t.named[u] = classes[place];
						if (BACKWARD)
						{
							t.share[u] = shares[place];
							t.probability[u] = known[place];
						}
					}
				}
				return t;
			}
			/* f(place of the row, class, probabilities of teacher and student) for all of them */
			template<bool BACKWARD, typename F>
			__device__ __forceinline__ void for_classes(const OfTile &t, F &&f) const
			{
#pragma unroll
				for (int u = 0; u < AHEAD; u++)
					if (t.first + u < t.last)
						f(static_cast<size_t>(t.m) * count + t.first + u, t.named[u], t.share[u], t.probability[u]);
				/* many in a tile: so many on their way at a time. us, one / 4 / 8: gradients of 532 x 421 of 421 classes, 105 a row 184 / 147 / 141, 2048 x 512 of 1000, 64 a row 126 / 112 / 111 */
				constexpr int MORE = 8;
				for (int k = t.first + AHEAD; k < t.last; k += MORE)
				{
					int named[MORE];
					float share[MORE], probability[MORE];
#pragma unroll
					for (int u = 0; u < MORE; u++)
					{
						const size_t place = static_cast<size_t>(t.m) * count + min(k + u, t.last - 1);
						named[u] = classes[place];
						share[u] = BACKWARD ? shares[place] : 0.0f;
						probability[u] = BACKWARD ? known[place] : 0.0f;
					}
					__builtin_amdgcn_sched_barrier(0);
#pragma unroll
					for (int u = 0; u < MORE; u++)
						if (k + u < t.last)
							f(static_cast<size_t>(t.m) * count + k + u, named[u], share[u], probability[u]);
				}
			}
			template<int BLOCKS>
			struct Rows
			{
					__device__ __forceinline__ void begin(const TopClasses&, int, int, int, int)
					{
					}
					template<typename Columns>
					__device__ __forceinline__ void take_row(const TopClasses&, int, int, const Columns&, const float (&)[2][16]) const
					{
					}
			};
			__device__ __forceinline__ float scaled(float z) const
			{
				return z * slope;
			}
			__device__ __forceinline__ float less(float z, float norm) const
			{
				return fmaf(z, slope, -norm);
			}
			template<int BM, int BN>
			static constexpr int loss_lds()
			{
				return Stage<float, BN>::bytes(rows_at_a_time(BM));
			}
			template<int BM, int BN>
			__device__ __forceinline__ OfTile begin_loss(const TilePlace<BM, BN> &at, int rows) const
			{
				return classes_of<false>(at, rows, nullptr);
			}
			/* the logits of the rows' classes, through LDS in fp32, a part of the rows at a time */
			template<int BM, int BN, typename Acc, typename Columns>
			__device__ __forceinline__ void take_tile(const Acc (&acc)[TilePlace<BM, BN>::BLOCKS][2], const Columns &columns, const TilePlace<BM, BN> &at, const OfTile &of_tile, uint8_t *lds) const
			{
				constexpr int ROWS = rows_at_a_time(BM), BLOCKS = ROWS / 64;
				typedef Stage<float, BN> TileStage;
				const TileStage stage { reinterpret_cast<float*>(lds) };
				if (__syncthreads_or(of_tile.first < of_tile.last) == 0)
					return;
				static_for<BM / ROWS>([&](auto part)
				{
					constexpr int h = decltype(part)::value;
					if (h > 0)
						__syncthreads();
#pragma unroll
					for (int i = h * BLOCKS; i < (h + 1) * BLOCKS; i++)
#pragma unroll
						for (int j = 0; j < 2; j++)
#pragma unroll
							for (int q = 0; q < 4; q++)
							{
								float z[4];
#pragma unroll
								for (int e = 0; e < 4; e++)
									z[e] = scaled(acc[i][j][4 * q + e] + columns.bias[j][4 * q + e]);
								stage.put(at.row(i) - h * ROWS, at.column(j) + at.lane_column(q), z[0], z[1], z[2], z[3]);
							}
					__syncthreads();
					if (of_tile.row >= h * ROWS && of_tile.row < (h + 1) * ROWS)
						for_classes<false>(of_tile, [&](size_t place, int n, float, float) __attribute__((always_inline))
						{
							logits[place] = stage.place[(of_tile.row - h * ROWS) * TileStage::STRIDE + n - at.tile_n * BN];
						});
				});
			}

			/* behind the tile: what is taken from the sums of the columns, in whole numbers of 2^-38, whose sum no order changes; whether it is no number; what rounding took from the rows beside what the tile's threads counted */
			template<int BM, int BN>
			static constexpr int gradient_lds()
			{
				return BN * 12 + BM * 4;
			}
			template<int BM, int BN>
			struct Extra
			{
					unsigned long long *columns;
					int *no_number;
					float *lost;
					__device__ __forceinline__ explicit Extra(uint8_t *lds) :
							columns(reinterpret_cast<unsigned long long*>(lds)),
							no_number(reinterpret_cast<int*>(lds + BN * 8)),
							lost(reinterpret_cast<float*>(lds + BN * 12))
					{
					}
			};
			template<int BM, int BN>
			__device__ __forceinline__ OfTile begin_gradient(const TilePlace<BM, BN> &at, int rows, const float *factors) const
			{
				return classes_of<true>(at, rows, factors);
			}
			/* the place may be an operand's until every wavefront is through with the product */
			template<int BM, int BN>
			__device__ __forceinline__ void begin_sums(uint8_t *lds) const
			{
				for (int i = threadIdx.x; i < gradient_lds<BM, BN>() / 4; i += TilePlace<BM, BN>::THREADS)
					reinterpret_cast<int*>(lds)[i] = 0;
			}
			/* the places of the rows' classes in a tile that lies in LDS, written again with p - q instead of p; a thread has a row's, so what rounding takes of them is added up in order */
			template<int BM, int BN, int ROWS, typename TileStage>
			__device__ __forceinline__ void correct(const TileStage &stage, uint8_t *lds, const TilePlace<BM, BN> &at, const OfTile &of_tile, int first_row, int first_class) const
			{
				typedef typename std::remove_pointer<decltype(stage.place)>::type T;
				const Extra<BM, BN> extra(lds);
				const int row = of_tile.row - first_row;
				if (row >= 0 && row < ROWS)
				{
					float taken = 0.0f;
					int before = -1;
					for_classes<true>(of_tile, [&](size_t, int n, float share, float probability) __attribute__((always_inline))
					{
						const int column = n - first_class - at.tile_n * BN;
						if (column == before) /* its share is at the class's first place */
							return;
						before = column;
						const float pf = probability * of_tile.factor, qf = share * of_tile.factor, d = pf - qf;
						T *stored = stage.place + row * TileStage::STRIDE + column;
						const T rounded = static_cast<T>(d);
						taken += (d - static_cast<float>(rounded)) - (pf - static_cast<float>(*stored));
						*stored = rounded;
						if (sizeof(T) == 2 && BM == 2 * LOW_ROWS && low)
							stored[LOW_ROWS * TileStage::STRIDE] = low_part(d, rounded);
						if (n == of_tile.anchor)
							own[of_tile.m] = d - static_cast<float>(rounded);
						if (fabsf(qf) < std::numeric_limits<float>::infinity())
							atomicAdd(&extra.columns[column], static_cast<unsigned long long>(__double2ll_rn(static_cast<double>(qf) * static_cast<double>(1ll << FIXED_BITS))));
						else
							extra.no_number[column] = 1;
					});
					extra.lost[of_tile.row] = taken;
				}
				__syncthreads();
			}
			template<int BM, int BN>
			__device__ __forceinline__ float column_sum(float sum, uint8_t *lds) const
			{
				const Extra<BM, BN> extra(lds);
				const double taken = static_cast<double>(static_cast<long long>(extra.columns[threadIdx.x])) / static_cast<double>(1ll << FIXED_BITS);
				return extra.no_number[threadIdx.x] != 0 ? std::numeric_limits<float>::quiet_NaN() : static_cast<float>(static_cast<double>(sum) - taken);
			}
			template<int BM, int BN>
			__device__ __forceinline__ float row_lost(float sum, uint8_t *lds) const
			{
				return sum + Extra<BM, BN>(lds).lost[threadIdx.x];
			}
	};

	/* ---- forward ------------------------------------------------------------------------------------------------------------ */
	/* few rows: all their logits are kept, which is little beside the weights (at most 64 of them), and whoever joins the tiles' sums finds the teacher's classes there */
	template<typename T, int MB, bool STREAM>
	__global__ __launch_bounds__(256) void kernel_distillation_few_rows(const T *x, const T *w, const T *bias, int rows, int features, int classes, float slope, Partial *partials, float *logits)
	{
		extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
		float (*sums)[2][16 * MB][16] = reinterpret_cast<float (*)[2][16 * MB][16]>(lds);
		const int n0 = blockIdx.x * FEW_CLASSES;
		const T *first = w + static_cast<size_t>(n0) * features;
		const bool second = n0 + 16 < classes; /* else the first block stands in for it */
		const int last_first = min(15, classes - 1 - n0), last_second = second ? min(15, classes - 1 - n0 - 16) : last_first;
		const T *next = second ? first + static_cast<size_t>(16) * features : first;
		if constexpr (STREAM)
			few_rows_stream<T, MB>(x, rows, first, next, last_first, last_second, features, lds);
		else
			few_rows_sums<T, MB>(x, rows, first, next, last_first, last_second, features, sums);
		const int c = threadIdx.x & 15;
		for (int row = threadIdx.x >> 4; row < 16 * MB; row += 16)
			if (row < rows)
			{
				float z[2];
				bool there[2];
#pragma unroll
				for (int i = 0; i < 2; i++)
				{
					const int n = n0 + 16 * i + c;
					there[i] = n < classes;
					z[i] = slope * (sums[0][i][row][c] + ((bias != nullptr && there[i]) ? static_cast<float>(bias[n]) : 0.0f));
					if (there[i])
						logits[static_cast<size_t>(row) * classes + n] = z[i];
				}
				const Partial p = lanes_join<16>(partial_of(z, there));
				if (c == 0)
					partials[static_cast<size_t>(row) * gridDim.x + blockIdx.x] = p;
			}
	}
	/*
	 * A workgroup to a row: lse, log p, and the loss with the teacher's probabilities made here. Of a class that stands there twice every place counts its own probability times the logarithm of their sum, which adds up to the
	 * same as the sum times its logarithm.
	 */
	template<typename L>
	__global__ __launch_bounds__(256) void kernel_join_few_rows(const Partial *partials, int tiles, const int *classes_in, const L *taught, const float *logits, int count, int classes, float temperature, float *loss,
			float *lse, float *log_probabilities)
	{
		__shared__ Partial waves[4];
		__shared__ float numbers[4];
		__shared__ int named[MOST_CLASSES_OF_ROW];
		__shared__ float shares[MOST_CLASSES_OF_ROW];
		const size_t row = blockIdx.x, base = row * count;
		float top = -std::numeric_limits<float>::infinity();
		for (int k = threadIdx.x; k < count; k += 256)
		{
			const int c = classes_in[base + k];
			const float v = static_cast<float>(taught[base + k]);
			const bool counts = c >= 0 && c < classes && !(v == -std::numeric_limits<float>::infinity());
			named[k] = counts ? c : -1;
			shares[k] = v;
			top = counts ? fmaxf(top, v) : top;
		}
		const Partial p = join_row<256>(partials + row * tiles, tiles, waves);
		const float value = p.top + logf(p.sum);
		const auto of_all = [&](float v, auto &&join)
		{
#pragma unroll
			for (int offset = 32; offset >= 1; offset >>= 1)
				v = join(v, __shfl_xor(v, offset));
			__syncthreads();
			if ((threadIdx.x & 63) == 0)
				numbers[threadIdx.x >> 6] = v;
			__syncthreads();
			return join(join(numbers[0], numbers[1]), join(numbers[2], numbers[3]));
		};
		const auto add = [](float a, float b)
		{
			return a + b;
		};
		top = of_all(top, [](float a, float b)
		{
			return fmaxf(a, b);
		});
		float sum = 0.0f;
		for (int k = threadIdx.x; k < count; k += 256)
			if (named[k] >= 0)
			{
				shares[k] = expf((shares[k] - top) / temperature);
				sum += shares[k];
			}
		sum = of_all(sum, add); /* behind its barriers every share is there for all */
		float divergence = 0.0f;
		for (int k = threadIdx.x; k < count; k += 256)
		{
			const int c = named[k];
			float log_p = 0.0f;
			if (c >= 0)
			{
				float together = 0.0f;
#pragma unroll 8
				for (int other = 0; other < count; other++)
					together += named[other] == c ? shares[other] : 0.0f;
				log_p = logits[row * classes + c] - value;
				const float share = shares[k] / sum;
				divergence += share == 0.0f ? 0.0f : share * (logf(together / sum) - log_p);
			}
			log_probabilities[base + k] = log_p;
		}
		divergence = of_all(divergence, add);
		if (threadIdx.x == 0)
		{
			lse[row] = value;
			loss[row] = divergence;
		}
	}
	/* as the cross entropy's, then the row's own classes: log p in the caller's order, and the loss */
	template<int THREADS>
	__global__ __launch_bounds__(256) void kernel_join_distillation(const Partial *partials, int tiles, const Teaching teaching, const float *logits, int rows, int count, float *loss, float *lse, float *log_probabilities)
	{
		__shared__ Partial waves[4];
		__shared__ float crosses[4];
		for (int row = blockIdx.x * (256 / THREADS) + threadIdx.x / THREADS; row < rows; row += gridDim.x * (256 / THREADS))
		{
			const Partial p = join_row<THREADS>(partials + static_cast<size_t>(row) * tiles, tiles, waves);
			const float value = p.top + logf(p.sum);
			const size_t base = static_cast<size_t>(row) * count;
			const int there = teaching.begins[static_cast<size_t>(row) * (tiles + 1) + tiles];
			float cross = 0.0f;
			for (int k = threadIdx.x % THREADS; k < count; k += THREADS)
			{
				float log_p = 0.0f;
				if (k < there)
				{
					const float share = teaching.shares[base + k];
					log_p = logits[base + k] - value;
					cross += share == 0.0f ? 0.0f : share * log_p;
				}
				log_probabilities[base + teaching.places[base + k]] = log_p;
			}
			cross = lanes_sum<64>(cross);
			if constexpr (THREADS > 64)
			{
				if ((threadIdx.x & 63) == 0)
					crosses[threadIdx.x >> 6] = cross;
				__syncthreads();
				cross = (crosses[0] + crosses[1]) + (crosses[2] + crosses[3]);
			}
			if (threadIdx.x % THREADS == 0)
			{
				lse[row] = value;
				loss[row] = there > 0 ? teaching.entropies[row] - cross : 0.0f;
			}
			if (THREADS > 64)
				return; /* one row, the meeting places are in use */
		}
	}

	/* ---- backward of few rows ------------------------------------------------------------------------------------------------ */
	/*
	 * Up to 16 rows: tiles would be empty but for a few rows, and each of three products would read or write the weights' size for itself on them. Here d is kept in fp32, [classes][rows], 64 bytes of a class at most; making it
	 * reads the weights once, past the rows, as the forward pass does; dx = d W reads them once more, every thread with its columns of all rows in registers; dW = d^T x writes as much, with its columns of x in registers. Rows of
	 * any width and alignment are read as they lie. Memory bounds all three. us of loss and gradients, so / on tiles: 1 row fp16 of 2048 x 65536 226 / 270, 1024 x 32000 68 / 98, 1023 x 32000 106 / 144, 1024 x 4000 34 / 53,
	 * 128 x 100000 80 / 149; 8 rows 262 / 278, 80 / 99, 136 / 152, 46 / 59, 106 / 150; fp32 1024 x 32000 1 row 106 / 202, 16 rows 127 / 205. (dW past the caches since: 8 rows of 2048 x 65536 227.) The second read of the weights, 54 of those 227 us, is
	 * there because a class's row has left the registers by the time its d is known; a run of classes that stays in LDS until then would spare it
	 */
	constexpr int FEW_GRADIENT_ROWS = 16;
	template<typename T, bool STREAM>
	__global__ __launch_bounds__(256) void kernel_few_gradient(const T *x, const T *w, const T *bias, TopClasses goal, const int *anchors, const float *lse, const float *dloss, int rows, int features, int classes, int stride, float *d,
			void *db, bool db_half, float beta)
	{
		extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
		__shared__ float tile[FEW_CLASSES][FEW_GRADIENT_ROWS + 1];
		float (*sums)[2][16][16] = reinterpret_cast<float (*)[2][16][16]>(lds);
		const int n0 = blockIdx.x * FEW_CLASSES;
		const T *first = w + static_cast<size_t>(n0) * features;
		const bool second = n0 + 16 < classes; /* else the first block stands in for it */
		const int last_first = min(15, classes - 1 - n0), last_second = second ? min(15, classes - 1 - n0 - 16) : last_first;
		const T *next = second ? first + static_cast<size_t>(16) * features : first;
		const int c = threadIdx.x & 15, row = threadIdx.x >> 4, m = min(row, rows - 1);
		/* a row without gradient has none, whatever its logits are */
		const float factor = row < rows && anchors[m] >= 0 ? dloss[m] * goal.slope : 0.0f, norm = lse[m];
		int from = 0, to = 0;
		if (factor != 0.0f)
		{
			const uint16_t *of_row = goal.begins + static_cast<size_t>(m) * goal.stride + blockIdx.x;
			from = of_row[0];
			to = of_row[1];
		}
		if constexpr (STREAM)
			few_rows_stream<T, 1>(x, rows, first, next, last_first, last_second, features, lds);
		else
			few_rows_sums<T, 1>(x, rows, first, next, last_first, last_second, features, sums);
#pragma unroll
		for (int i = 0; i < 2; i++)
		{
			const int n = n0 + 16 * i + c;
			const bool there = factor != 0.0f && n < classes;
			const float z = sums[0][i][row][c] + ((bias != nullptr && there) ? static_cast<float>(bias[n]) : 0.0f);
			tile[16 * i + c][row] = there ? factor * expf(goal.less(z, norm)) : 0.0f;
		}
		__syncthreads();
		/* 16 threads share a row's classes; of those that stand there twice the first place has the share */
		for (int k = from + c; k < to; k += 16)
		{
			const size_t place = static_cast<size_t>(m) * goal.count + k;
			const int n = goal.classes[place];
			if (k == from || goal.classes[place - 1] != n)
				tile[n - n0][row] = factor * (goal.known[place] - goal.shares[place]);
		}
		__syncthreads();
		for (int i = threadIdx.x; i < FEW_CLASSES * stride; i += 256)
			if (n0 + i / stride < classes)
				d[static_cast<size_t>(n0) * stride + i] = tile[i / stride][i % stride];
		const int n = n0 + static_cast<int>(threadIdx.x);
		if (db != nullptr && threadIdx.x < FEW_CLASSES && n < classes)
		{
			float sum = 0.0f;
			for (int r = 0; r < rows; r++)
				sum += tile[threadIdx.x][r];
			if (db_half)
			{
				half_t *out = reinterpret_cast<half_t*>(db) + n;
				*out = static_cast<half_t>(beta != 0.0f ? fmaf(beta, static_cast<float>(*out), sum) : sum);
			}
			else
			{
				float *out = reinterpret_cast<float*>(db) + n;
				*out = beta != 0.0f ? fmaf(beta, *out, sum) : sum;
			}
		}
	}
	/* a thread's columns of a row, of which `lanes` threads (a power of two from 64 on) take one; the workgroup's other threads take other classes. Whole wavefronts have the same class, so its row of d comes by scalar loads */
	template<int VEC>
	struct FewColumns
	{
			int group, groups;
			bool inside;
			RowPlace place;

			__device__ __forceinline__ FewColumns(int columns, int lanes) :
					group(__builtin_amdgcn_readfirstlane(threadIdx.x / lanes)),
					groups(256 / lanes)
			{
				const int column = (blockIdx.y * lanes + static_cast<int>(threadIdx.x) % lanes) * VEC;
				inside = column < columns;
				place = place_in_row<VEC>(min(column, columns - 1), columns);
			}
	};
	template<int ROWS>
	struct ClassRow
	{
			float d[ROWS];

			__device__ __forceinline__ void load(const float *src, int n)
			{
#pragma unroll
				for (int r = 0; r < ROWS; r++)
					d[r] = src[static_cast<size_t>(n) * ROWS + r];
			}
	};
	/* partial[part][row][column]: the part's classes */
	template<typename T, int VEC, int ROWS>
	__global__ __launch_bounds__(256) void kernel_few_input(const T *w, const float *d, int rows, int columns, int classes, int classes_of_part, int lanes, float *partial)
	{
		constexpr int AHEAD = 4;
		__shared__ float meeting[256][VEC];
		const FewColumns<VEC> column(columns, lanes);
		const int first = blockIdx.x * classes_of_part, last = first + min(classes_of_part, classes - first);
		float sums[ROWS][VEC];
#pragma unroll
		for (int r = 0; r < ROWS; r++)
#pragma unroll
			for (int e = 0; e < VEC; e++)
				sums[r][e] = 0.0f;
		const auto add = [&](const Elements<T, VEC> &weights, int n) __attribute__((always_inline))
		{
			ClassRow<ROWS> of_class;
			of_class.load(d, n);
#pragma unroll
			for (int r = 0; r < ROWS; r++)
#pragma unroll
				for (int e = 0; e < VEC; e++)
					sums[r][e] = fmaf(of_class.d[r], weights[e], sums[r][e]);
		};
		int n = first + column.group;
		for (; n + (AHEAD - 1) * column.groups < last; n += AHEAD * column.groups)
		{
			Elements<T, VEC> weights[AHEAD];
#pragma unroll
			for (int u = 0; u < AHEAD; u++)
				weights[u].load(column.place.in(w + static_cast<size_t>(n + u * column.groups) * columns));
			__builtin_amdgcn_sched_barrier(0); /* all on their way before one is waited for */
#pragma unroll
			for (int u = 0; u < AHEAD; u++)
				add(weights[u], n + u * column.groups);
		}
		for (; n < last; n += column.groups)
		{
			Elements<T, VEC> weights;
			weights.load(column.place.in(w + static_cast<size_t>(n) * columns));
			add(weights, n);
		}
#pragma unroll
		for (int r = 0; r < ROWS; r++)
		{
			if (column.groups > 1)
			{
				__syncthreads();
#pragma unroll
				for (int e = 0; e < VEC; e++)
					meeting[threadIdx.x][e] = sums[r][e];
				__syncthreads();
				if (column.group == 0)
					for (int t = threadIdx.x + lanes; t < 256; t += lanes)
#pragma unroll
						for (int e = 0; e < VEC; e++)
							sums[r][e] += meeting[t][e];
			}
			if (r < rows && column.group == 0 && column.inside)
				store_nearest<VEC>(column.place.in(partial + (static_cast<size_t>(blockIdx.x) * rows + r) * columns), sums[r], column.place.skip);
		}
	}
	template<typename T, typename Out, int VEC, int ROWS>
	__global__ __launch_bounds__(256) void kernel_few_weights(const T *x, const float *d, int rows, int columns, int classes, int classes_of_group, int lanes, Out *out, float beta, bool past)
	{
		const FewColumns<VEC> column(columns, lanes);
		Elements<T, VEC> of_row[ROWS];
#pragma unroll
		for (int r = 0; r < ROWS; r++)
			of_row[r].load(column.place.in(x + static_cast<size_t>(min(r, rows - 1)) * columns)); /* of rows that are not there d is zero */
		if (!column.inside)
			return;
		const int first = blockIdx.x * classes_of_group, last = first + min(classes_of_group, classes - first);
		for (int n = first + column.group; n < last; n += column.groups)
		{
			ClassRow<ROWS> of_class;
			of_class.load(d, n);
			Out *dst = column.place.in(out + static_cast<size_t>(n) * columns);
			Elements<Out, VEC> old;
			if (beta != 0.0f)
				old.load(dst);
			float v[VEC];
#pragma unroll
			for (int e = 0; e < VEC; e++)
				v[e] = 0.0f;
#pragma unroll
			for (int r = 0; r < ROWS; r++)
#pragma unroll
				for (int e = 0; e < VEC; e++)
					v[e] = fmaf(of_class.d[r], of_row[r][e], v[e]);
			if (beta != 0.0f)
#pragma unroll
				for (int e = 0; e < VEC; e++)
					v[e] = fmaf(beta, old[e], v[e]);
			if (past)
				store_past_caches<VEC>(dst, v, column.place.skip);
			else
				store_nearest<VEC>(dst, v, column.place.skip);
		}
	}

	/* ---- sizes ---------------------------------------------------------------------------------------------------------------- */
	/*
	 * The cross entropy's rule, but that 17 to 32 rows of large weights in fp16 go on tiles: they fill two blocks of 16 rows, and their logits are kept. us of a forward pass, so / on tiles: 24 rows fp16 of 2048 x 65536 67 / 56,
	 * 1024 x 32000 29 / 28, 1023 x 32000 68 / 50, 256 x 100000 55 / 31, 1024 x 8000 12 / 26; fp32 1024 x 32000 47 / 54; 16 rows fp16 47 / 55, 20 / 27, 46 / 50, 27 / 31, 11 / 25
	 */
	bool few_logits(const LossShape &s)
	{
		return few_rows(s) && (s.rows <= 16 || s.element_size == 4 || static_cast<size_t>(s.classes) * s.features * s.element_size <= (size_t(1) << 24));
	}
	/* beyond, 16 rows in fp16 (us of loss and gradients, so / on tiles: 2048 x 65536 332 / 281, 1024 x 32000 101 / 100), the vector units bound the products, which take an element of the weights times every row */
	bool few_gradients(const LossShape &s)
	{
		return s.rows <= (s.element_size == 2 ? 8 : FEW_GRADIENT_ROWS);
	}
	struct FewGradientPlan
	{
			int stride, vector, lanes, spans; /* rows of d's layout, a power of two; elements of a thread; threads and workgroups of a row */
			int parts, classes_of_part; /* of dx */
			int classes_of_group; /* of dW */
	};
	FewGradientPlan few_gradient_plan(const LossShape &s)
	{
		FewGradientPlan plan { };
		plan.stride = 1;
		while (plan.stride < s.rows)
			plan.stride *= 2;
		plan.vector = s.features >= 16 / s.element_size ? 16 / s.element_size : 1;
		plan.lanes = 64;
		while (plan.lanes < 256 && plan.lanes * plan.vector < s.features)
			plan.lanes *= 2;
		plan.spans = ceil_div(s.features, plan.lanes * plan.vector);
		/* a workgroup to every compute unit and a second one, whatever the width; no less than four classes to a group of threads */
		plan.classes_of_part = std::max(4 * 256 / plan.lanes, ceil_div(s.classes, std::max(1, 512 / plan.spans)));
		plan.parts = ceil_div(s.classes, plan.classes_of_part);
		plan.classes_of_group = std::max(256 / plan.lanes, ceil_div(s.classes, std::max(1, 2048 / plan.spans)));
		return plan;
	}
	struct DistillationSpace
	{
			LossSpace loss;
			size_t classes, places, shares, known, begins, anchors, entropies, logits, own, common, there;
			size_t d, partial; /* backward of few rows */
			size_t total;
	};
	DistillationSpace distillation_space(const LossShape &s, int count, bool backward)
	{
		DistillationSpace space { };
		const bool few = backward && few_gradients(s);
		if (!few)
			space.loss = loss_space(s, backward, few_logits(s), backward && may_keep_low(s));
		size_t at = space.loss.total;
		const auto take = [&](size_t bytes)
		{
			const size_t begin = at;
			at += round_up(bytes, 256);
			return begin;
		};
		const size_t rows = s.rows, places = rows * count;
		if (s.rows > 0 && !backward && few_logits(s))
			space.logits = take(sizeof(float) * rows * s.classes);
		else if (s.rows > 0)
		{
			space.classes = take(sizeof(int) * places);
			space.places = take(sizeof(uint16_t) * places);
			space.shares = take(sizeof(float) * places);
			space.logits = space.known = take(sizeof(float) * places);
			space.begins = take(sizeof(uint16_t) * rows * (ceil_div(s.classes, few ? FEW_CLASSES : tile_width(s, backward ? classes_of_piece(s) : s.classes)) + 1));
			if (few)
			{
				const FewGradientPlan plan = few_gradient_plan(s);
				space.d = take(sizeof(float) * s.classes * plan.stride);
				space.partial = take(sizeof(float) * plan.parts * rows * s.features);
			}
			space.anchors = take(sizeof(int) * rows);
			space.entropies = take(sizeof(float) * rows);
			if (backward && !few && s.element_size == 2 && !may_keep_low(s))
			{
				space.own = take(sizeof(float) * rows);
				space.there = take(sizeof(float));
				space.common = take(sizeof(half_t) * round_up(s.features, COMMON_COLUMNS));
			}
		}
		space.total = at;
		return space;
	}
	template<typename V>
	V* at(uint8_t *workspace, size_t offset)
	{
		return reinterpret_cast<V*>(workspace + offset);
	}
	Teaching teaching_of(uint8_t *workspace, const DistillationSpace &space)
	{
		return Teaching { at<int>(workspace, space.classes), at<uint16_t>(workspace, space.places), at<float>(workspace, space.shares), at<float>(workspace, space.known), at<uint16_t>(workspace, space.begins),
				at<int>(workspace, space.anchors), at<float>(workspace, space.entropies), at<float>(workspace, space.own), at<float>(workspace, space.there), at<half_t>(workspace, space.common) };
	}
	/* w: for the common row, else null */
	void sort_teacher(hipStream_t stream, const LossShape &s, const mlTensor_t &classes, const mlTensor_t &logits, const float *log_probabilities, int count, float temperature, int width, const half_t *w,
			const Teaching &out)
	{
		const int tiles = ceil_div(s.classes, width), bytes = 4 * 4 * static_cast<int>(sizeof(int)) * places_in_lds(count);
		/* a launch has less than 2^32 threads, so 2^26 rows and more go out in several (a loop over the rows in the kernel would take 2 us of every call); the common row in the last one */
		constexpr int MOST_ROWS = 1 << 25;
		const auto launch = [&](auto kernel, auto values)
		{
			ensure_dynamic_lds(reinterpret_cast<const void*>(kernel), bytes);
			for (int first = 0; first < s.rows; first += MOST_ROWS)
			{
				const int groups = ceil_div(std::min(MOST_ROWS, s.rows - first), 4);
				const int others = w != nullptr && s.rows - first <= MOST_ROWS ? static_cast<int>(round_up(s.features, COMMON_COLUMNS)) / 64 : 0;
				hipLaunchKernelGGL(kernel, dim3(groups + others), dim3(256), bytes, stream, ptr<int>(classes), values, log_probabilities, first, groups, s.rows, count, s.classes, temperature, width, tiles, w,
						s.features, out);
				MLHIP_CHECK(hipGetLastError());
			}
		};
		if (logits.dtype == DTYPE_FLOAT16)
			launch(kernel_sort_teacher<half_t>, static_cast<const half_t*>(ptr<half_t>(logits)));
		else
			launch(kernel_sort_teacher<float>, static_cast<const float*>(ptr<float>(logits)));
	}
	template<typename T>
	void distillation_forward(hipStream_t stream, const LossShape &s, const T *x, const T *w, const T *bias, const mlTensor_t &classes, const mlTensor_t &logits, int count, float temperature, float *loss,
			float *lse, float *log_probabilities, uint8_t *workspace)
	{
		const DistillationSpace space = distillation_space(s, count, false);
		Partial *partials = at<Partial>(workspace, space.loss.partials);
		float *kept = at<float>(workspace, space.logits);
		if (few_logits(s))
		{
			const int columns = ceil_div(s.classes, FEW_CLASSES);
			with_few_rows<T>(s.rows, s.features, [&](auto blocks, auto streamed)
			{
				constexpr int MB = decltype(blocks)::value, bytes = few_rows_lds<MB>(decltype(streamed)::value);
				auto kernel = kernel_distillation_few_rows<T, MB, decltype(streamed)::value>;
				ensure_dynamic_lds(reinterpret_cast<const void*>(kernel), bytes);
				hipLaunchKernelGGL(kernel, dim3(columns), dim3(256), bytes, stream, x, w, bias, s.rows, s.features, s.classes, 1.0f / temperature, partials, kept);
			});
			MLHIP_CHECK(hipGetLastError());
			const auto join = [&](auto kernel, auto taught)
			{
				hipLaunchKernelGGL(kernel, dim3(s.rows), dim3(256), 0, stream, partials, columns, ptr<int>(classes), taught, kept, count, s.classes, temperature, loss, lse, log_probabilities);
			};
			if (logits.dtype == DTYPE_FLOAT16)
				join(kernel_join_few_rows<half_t>, static_cast<const half_t*>(ptr<half_t>(logits)));
			else
				join(kernel_join_few_rows<float>, static_cast<const float*>(ptr<float>(logits)));
			MLHIP_CHECK(hipGetLastError());
			return;
		}
		const Teaching teaching = teaching_of(workspace, space);
		const int width = tile_width(s, s.classes), columns = ceil_div(s.classes, width), padded = padded_columns<T>(s.features);
		sort_teacher(stream, s, classes, logits, nullptr, count, temperature, width, nullptr, teaching);
		const TopClasses goal { nullptr, teaching.classes, teaching.shares, nullptr, teaching.begins, kept, count, columns + 1, 1.0f / temperature, nullptr, nullptr, false };
		x = pad_rows(stream, x, at<T>(workspace, space.loss.x), s.rows, s.features);
		w = pad_rows(stream, w, at<T>(workspace, space.loss.w), s.classes, s.features);
		const ProductPlan plan = logits_plan(s, s.classes);
		const Operand a { reinterpret_cast<const uint8_t*>(x), padded * sizeof(T), s.rows, padded };
		const Operand b { reinterpret_cast<const uint8_t*>(w), padded * sizeof(T), s.classes, padded };
		launch_product<T, Side::ROWS, Side::ROWS, false>(stream, plan, a, b, s.rows, LossEpilogue<T, TopClasses> { bias, goal, partials, s.classes, columns });
		MLHIP_CHECK(hipGetLastError());
		if (s.rows <= 1024)
			hipLaunchKernelGGL((kernel_join_distillation<256>), dim3(s.rows), dim3(256), 0, stream, partials, columns, teaching, kept, s.rows, count, loss, lse, log_probabilities);
		else
			hipLaunchKernelGGL((kernel_join_distillation<64>), dim3(std::min(ceil_div(s.rows, 4), 1 << 20)), dim3(256), 0, stream, partials, columns, teaching, kept, s.rows, count, loss, lse,
					log_probabilities);
		MLHIP_CHECK(hipGetLastError());
	}
	/* f(rows of d's layout, a power of two) as a compile-time constant */
	template<typename T, typename F>
	void with_stride(int stride, F &&f)
	{
		switch (stride)
		{
			case 1:
				return f(std::integral_constant<int, 1>());
			case 2:
				return f(std::integral_constant<int, 2>());
			case 4:
				return f(std::integral_constant<int, 4>());
			case 8:
				return f(std::integral_constant<int, 8>());
			default:
				if constexpr (sizeof(T) == 4)
					return f(std::integral_constant<int, 16>());
				else
					fail_logic("HIP backend: d of 16 rows is for fp32");
		}
	}
	template<typename T>
	void few_gradients(hipStream_t stream, const LossShape &s, const T *x, const T *w, const T *bias, const TopClasses &goal, const Teaching &teaching, const float *lse, const float *dloss, float beta_dx, T *dx,
			float beta_weights, const mlTensor_t &dw, const mlTensor_t &db, float *d, float *partial)
	{
		const FewGradientPlan plan = few_gradient_plan(s);
		const bool stream_rows = (s.features * sizeof(T)) % 16 == 0;
		const int bytes = few_rows_lds<1>(stream_rows);
		auto kernel = stream_rows ? kernel_few_gradient<T, true> : kernel_few_gradient<T, false>;
		ensure_dynamic_lds(reinterpret_cast<const void*>(kernel), bytes);
		hipLaunchKernelGGL(kernel, dim3(ceil_div(s.classes, FEW_CLASSES)), dim3(256), bytes, stream, x, w, bias, goal, teaching.anchors, lse, dloss, s.rows, s.features, s.classes, plan.stride, d, db.data,
				db.dtype == DTYPE_FLOAT16, beta_weights);
		MLHIP_CHECK(hipGetLastError());
		const auto products = [&](auto vector, auto stride)
		{
			constexpr int VEC = decltype(vector)::value, ROWS = decltype(stride)::value;
			if (dx != nullptr)
			{
				hipLaunchKernelGGL((kernel_few_input<T, VEC, ROWS>), dim3(plan.parts, plan.spans), dim3(256), 0, stream, w, d, s.rows, s.features, s.classes, plan.classes_of_part, plan.lanes, partial);
				MLHIP_CHECK(hipGetLastError());
				const int outputs = s.rows * s.features;
				launch_sum_partials(stream, partial, plan.parts, outputs, dx, sizeof(T) == 2 ? DTYPE_FLOAT16 : DTYPE_FLOAT32, outputs, beta_dx);
			}
			const dim3 grid(ceil_div(s.classes, plan.classes_of_group), plan.spans);
			if (dw.data != nullptr && dw.dtype == DTYPE_FLOAT32)
				hipLaunchKernelGGL((kernel_few_weights<T, float, VEC, ROWS>), grid, dim3(256), 0, stream, x, d, s.rows, s.features, s.classes, plan.classes_of_group, plan.lanes, ptr<float>(dw), beta_weights,
						past_caches(s.classes, s.features * sizeof(float)));
			else if constexpr (sizeof(T) == 2)
				if (dw.data != nullptr)
					hipLaunchKernelGGL((kernel_few_weights<T, T, VEC, ROWS>), grid, dim3(256), 0, stream, x, d, s.rows, s.features, s.classes, plan.classes_of_group, plan.lanes, ptr<T>(dw), beta_weights,
							past_caches(s.classes, s.features * sizeof(T)));
			MLHIP_CHECK(hipGetLastError());
		};
		with_stride<T>(plan.stride, [&](auto stride)
		{
			if (plan.vector == 1)
				products(std::integral_constant<int, 1>(), stride);
			else
				products(std::integral_constant<int, 16 / sizeof(T)>(), stride);
		});
	}
	template<typename T>
	void distillation_backward(hipStream_t stream, const LossShape &s, const T *x, const T *w, const T *bias, const mlTensor_t &classes, const mlTensor_t &logits, int count, float temperature, const float *lse,
			const float *log_probabilities, const float *dloss, float beta_dx, T *dx, float beta_weights, const mlTensor_t &dw, const mlTensor_t &db, uint8_t *workspace)
	{
		const DistillationSpace space = distillation_space(s, count, true);
		const Teaching teaching = teaching_of(workspace, space);
		const bool few = few_gradients(s), low = !few && may_keep_low(s);
		const int width = few ? FEW_CLASSES : tile_width(s, classes_of_piece(s)), tiles = ceil_div(s.classes, width);
		GivenBack<T> to { teaching.anchors, nullptr, nullptr, nullptr };
		const half_t *for_common = nullptr;
		if constexpr (sizeof(T) == 2)
			if (!few && !low && dx != nullptr)
			{
				to = GivenBack<T> { teaching.anchors, teaching.own, teaching.common, teaching.there };
				for_common = w;
			}
		sort_teacher(stream, s, classes, logits, log_probabilities, count, temperature, width, for_common, teaching);
		const auto goal = [&](int first_tile)
		{
			return TopClasses { nullptr, teaching.classes, teaching.shares, teaching.known, teaching.begins + first_tile, nullptr, count, tiles + 1, 1.0f / temperature, teaching.anchors,
					for_common != nullptr ? teaching.own : nullptr, low };
		};
		if (few)
			few_gradients(stream, s, x, w, bias, goal(0), teaching, lse, dloss, beta_dx, dx, beta_weights, dw, db, at<float>(workspace, space.d), at<float>(workspace, space.partial));
		else
			loss_backward(stream, s, x, w, bias, to, goal, 1.0f / temperature, lse, dloss, beta_dx, dx, beta_weights, dw, db, few_logits(s), low, workspace);
	}

	/* the rows' shape with another last dimension */
	bool places_of_rows(const mlTensor_t &t, const LossShape &s, int count)
	{
		return t.rank >= 1 && last_dim(t) == count && volume(t) == static_cast<size_t>(s.rows) * count && (s.rows == 0 || t.data != nullptr) && on_elements(t);
	}
	LossShape check_distillation(const mlTensor_t &x, const mlTensor_t &w, const mlTensor_t &b, const mlTensor_t &classes, const mlTensor_t &logits, float temperature, int &count, const char *name)
	{
		const std::string who(name);
		const LossShape s = loss_shape(shape_of(x), shape_of(w), x.dtype, name);
		MLHIP_REQUIRE(w.dtype == x.dtype, who + ": weights must have the input's type");
		MLHIP_REQUIRE(b.data == nullptr || (b.dtype == x.dtype && volume(b) == static_cast<size_t>(s.classes) && on_elements(b)), who + ": the bias must be [classes] of the input's type");
		count = last_dim(classes);
		MLHIP_REQUIRE(count >= 1 && count <= MOST_CLASSES_OF_ROW, who + ": the teacher must name 1 to 1024 classes for every row");
		MLHIP_REQUIRE(classes.dtype == DTYPE_INT32 && places_of_rows(classes, s, count), who + ": the teacher's classes must be int32, as many for every row");
		MLHIP_REQUIRE((logits.dtype == x.dtype || logits.dtype == DTYPE_FLOAT32) && places_of_rows(logits, s, count), who + ": there must be one logit of the input's type or fp32 for every class of the teacher");
		MLHIP_REQUIRE(temperature > 0.0f && std::isfinite(temperature) && std::isfinite(1.0f / temperature), who + ": the temperature must be positive and finite");
		MLHIP_REQUIRE(s.rows == 0 || (x.data != nullptr && w.data != nullptr), who + ": null pointer");
		MLHIP_REQUIRE(reinterpret_cast<uintptr_t>(x.data) % 16 == 0 && reinterpret_cast<uintptr_t>(w.data) % 16 == 0, who + ": input and weights must be aligned to 16 bytes");
		return s;
	}
}

extern "C"
{
	using namespace mlhip;

	size_t hip_linear_distillation_get_workspace_size(mlShape_t input_shape, mlShape_t weights_shape, int count, mlDataType_t dtype, bool backward)
	try
	{
		const char *name = "linear_distillation_get_workspace_size";
		MLHIP_REQUIRE(count >= 1 && count <= MOST_CLASSES_OF_ROW, std::string(name) + ": the teacher must name 1 to 1024 classes for every row");
		const LossShape s = loss_shape(input_shape, weights_shape, dtype, name);
		/* the forward pass may have the backward pass's workspace */
		return backward ? std::max(distillation_space(s, count, true).total, distillation_space(s, count, false).total) : distillation_space(s, count, false).total;
	}
	catch (...)
	{
		return mlhip::entry_failed<size_t>();
	}

	void hip_linear_distillation_forward(mlContext_t context, const mlTensor_t x, const mlTensor_t w, const mlTensor_t b, const mlTensor_t classes, const mlTensor_t logits, float temperature, mlTensor_t loss,
			mlTensor_t lse, mlTensor_t log_probabilities, void *workspace, size_t workspace_size)
	try
	{
		const char *name = "linear_distillation_forward";
		int count;
		const LossShape s = check_distillation(x, w, b, classes, logits, temperature, count, name);
		MLHIP_REQUIRE(per_row(loss, s, DTYPE_FLOAT32) && per_row(lse, s, DTYPE_FLOAT32), "linear_distillation_forward: loss and lse must be fp32 with one element per row");
		MLHIP_REQUIRE(log_probabilities.dtype == DTYPE_FLOAT32 && places_of_rows(log_probabilities, s, count), "linear_distillation_forward: the log probabilities must be fp32, one for every class of the teacher");
		if (s.rows == 0)
			return;
		check_space(workspace, workspace_size, distillation_space(s, count, false).total, name);
		require_apart( { loss, lse, log_probabilities, Extent(workspace, workspace_size) }, { x, w, b, classes, logits }, name);
		const OnDeviceOf on(context);
		if (x.dtype == DTYPE_FLOAT16)
			distillation_forward(on.stream, s, ptr<half_t>(x), ptr<half_t>(w), ptr<half_t>(b), classes, logits, count, temperature, ptr<float>(loss), ptr<float>(lse), ptr<float>(log_probabilities),
					reinterpret_cast<uint8_t*>(workspace));
		else
			distillation_forward(on.stream, s, ptr<float>(x), ptr<float>(w), ptr<float>(b), classes, logits, count, temperature, ptr<float>(loss), ptr<float>(lse), ptr<float>(log_probabilities),
					reinterpret_cast<uint8_t*>(workspace));
	}
	catch (...)
	{
		return mlhip::entry_failed<void>();
	}

	void hip_linear_distillation_backward(mlContext_t context, const mlTensor_t x, const mlTensor_t w, const mlTensor_t b, const mlTensor_t classes, const mlTensor_t logits, float temperature,
			const mlTensor_t lse, const mlTensor_t log_probabilities, const mlTensor_t dloss, float beta_dx, mlTensor_t dx, float beta_weights, mlTensor_t dw, mlTensor_t db, void *workspace, size_t workspace_size)
	try
	{
		const char *name = "linear_distillation_backward";
		int count;
		const LossShape s = check_distillation(x, w, b, classes, logits, temperature, count, name);
		MLHIP_REQUIRE(per_row(lse, s, DTYPE_FLOAT32) && per_row(dloss, s, DTYPE_FLOAT32), "linear_distillation_backward: lse and dloss must be fp32 with one element per row");
		MLHIP_REQUIRE(log_probabilities.dtype == DTYPE_FLOAT32 && places_of_rows(log_probabilities, s, count), "linear_distillation_backward: the log probabilities must be fp32, one for every class of the teacher");
		check_gradients(x, w, s, dx, dw, db, name);
		MLHIP_REQUIRE(on_elements(dx) && on_elements(dw) && on_elements(db), "linear_distillation_backward: the gradients must be aligned to an element");
		if (dx.data == nullptr && dw.data == nullptr && db.data == nullptr)
			return;
		if (s.rows == 0)
		{
			const OnDeviceOf on(context);
			sums_over_nothing(on.stream, dw, db, beta_weights);
			return;
		}
		check_space(workspace, workspace_size, distillation_space(s, count, true).total, name);
		require_apart( { dx, dw, db, Extent(workspace, workspace_size) }, { x, w, b, classes, logits, lse, log_probabilities, dloss }, name);
		const OnDeviceOf on(context);
		if (x.dtype == DTYPE_FLOAT16)
			distillation_backward(on.stream, s, ptr<half_t>(x), ptr<half_t>(w), ptr<half_t>(b), classes, logits, count, temperature, ptr<float>(lse), ptr<float>(log_probabilities), ptr<float>(dloss), beta_dx,
					ptr<half_t>(dx), beta_weights, dw, db, reinterpret_cast<uint8_t*>(workspace));
		else
			distillation_backward(on.stream, s, ptr<float>(x), ptr<float>(w), ptr<float>(b), classes, logits, count, temperature, ptr<float>(lse), ptr<float>(log_probabilities), ptr<float>(dloss), beta_dx,
					ptr<float>(dx), beta_weights, dw, db, reinterpret_cast<uint8_t*>(workspace));
	}
	catch (...)
	{
		return mlhip::entry_failed<void>();
	}
}
