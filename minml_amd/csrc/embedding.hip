/*
 * embedding.hip — rows of a table by token, and the table's gradient.
 *
 *   y[i] = scale table[token[i]]                                           a token that is none of the table's: zeros
 *   dtable[v] = scale sum over i with token[i] = v of dy[i] + beta dtable[v]     in fp32, always in the same order
 *
 * Forward: memory bounds it (a row of the table read for every row written, from the caches where tokens repeat): 57600 x 256 fp16 from 400 classes 7.8 us (3.8 TB/s, the stores of 29 MB alone take 6).
 * Backward: tokens are sorted first, stably, so that a class's rows stand in a list in the order they have in dy. Up to 15 rows of a class are added up in that order by one group of threads; of more, each of a workgroup's groups
 * takes every so many-th, in chunks of 32 or 64 rows where there are as many, and their sums are added up, groups and chunks in order. So no two threads write to the same row of the table, every element of dy is read once and
 * every row of the table written once, with zeros where there is no token, and the bits are the same on every run. us: 16384 x 4096 fp16 into 65536 classes 169 (4.0 TB/s: 22 for the order, 139 with 4.7 TB/s for the rows, 11 to
 * join the long classes), 57600 x 256 fp16 into 400 classes 25, 20011 x 1001 fp32 into 5003 classes 43 to 51: launches of 4 to 9 us, one after another, whose reads wait for each other. Many tokens: 131072 x 1024 fp16 into
 * 50000 classes 122, 28 of them for the order, 262144 x 256 99 and 37, 2^20 x 64 231.
 */
#include "training_utils.hpp"

#include <algorithm>
#include <cmath>
#include <tuple>
#include <utility>

namespace
{
	using namespace mlhip;

	/* ---- forward ------------------------------------------------------------------------------------------------------------ */
	/* EACH vectors of a thread, on their way at once */
	template<typename T, int VEC, int EACH>
	__global__ __launch_bounds__(256) void kernel_embedding_forward(const int *tokens, const T *table, T *y, int rows, int columns, int classes, int vectors, float scale)
	{
		const size_t count = static_cast<size_t>(rows) * vectors;
		for (size_t first = static_cast<size_t>(blockIdx.x) * 256 * EACH + threadIdx.x; first < count; first += static_cast<size_t>(gridDim.x) * 256 * EACH)
		{
			size_t row[EACH];
			int token[EACH];
			RowPlace place[EACH];
			Elements<T, VEC> of_table[EACH];
#pragma unroll
			for (int u = 0; u < EACH; u++)
			{
				int vector;
				row[u] = split_index(min(first + u * 256, count - 1), vectors, vector);
				place[u] = place_in_row<VEC>(vector * VEC, columns);
				token[u] = tokens[row[u]];
			}
#pragma unroll
			for (int u = 0; u < EACH; u++)
				of_table[u].load(place[u].in(table + static_cast<size_t>(token[u] >= 0 && token[u] < classes ? token[u] : 0) * columns));
#pragma unroll
			for (int u = 0; u < EACH; u++)
				if (first + u * 256 < count)
				{
					float v[VEC];
#pragma unroll
					for (int e = 0; e < VEC; e++)
						v[e] = token[u] >= 0 && token[u] < classes ? scale * of_table[u][e] : 0.0f;
					store_nearest<VEC>(place[u].in(y + row[u] * columns), v, place[u].skip);
				}
		}
	}

	/* ---- tokens in order ---------------------------------------------------------------------------------------------------- */
	/*
	 * A stable sort by digits, lowest first: an element's place is the number of elements with smaller digits and of equal ones before it. A wavefront looks at 64 elements at a time; the lanes with equal digits find one another by
	 * one ballot per bit. Tokens that are none of the table's are taken for class `classes`, so they end up last.
	 */
	__device__ __forceinline__ uint64_t lanes_alike(int digit, int bits, bool there)
	{
		uint64_t same = __ballot(there);
		for (int b = 0; b < bits; b++)
		{
			const bool one = (digit >> b) & 1;
			const uint64_t ones = __ballot(one);
			same &= one ? ones : ~ones;
		}
		return same;
	}
	__device__ __forceinline__ int lanes_below(uint64_t mask)
	{
		return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
	}
	/* what the lanes of a wavefront wrote to LDS before is there for all of them behind it: LDS serves a wavefront in order, the compiler has to */
	__device__ __forceinline__ void wave_in_order()
	{
		__builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
		__builtin_amdgcn_wave_barrier();
	}
	__device__ __forceinline__ int key_of(int token, int classes)
	{
		return static_cast<int>(min(static_cast<uint32_t>(token), static_cast<uint32_t>(classes)));
	}
	/* sum of the values of the threads before; of a workgroup of 64 WAVES threads. Every thread calls it */
	template<int WAVES>
	__device__ __forceinline__ int scan_exclusive(int value, int *waves)
	{
		const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
		int sum = value;
#pragma unroll
		for (int offset = 1; offset < 64; offset <<= 1)
		{
			const int below = __shfl_up(sum, offset);
			sum += lane >= offset ? below : 0;
		}
		if (lane == 63)
			waves[wave] = sum;
		__syncthreads();
		int before = sum - value;
#pragma unroll
		for (int w = 0; w < WAVES; w++)
			before += w < wave ? waves[w] : 0;
		__syncthreads();
		return before;
	}
	/*
	 * Few tokens: every one counts those that come before it, 64 tokens of a workgroup against all others, a sixteenth of them by each wavefront, which reads them through scalar registers.
	 */
	__global__ __launch_bounds__(1024) void kernel_sort_by_counting(const int *tokens, int count, int classes, int *keys_out, int *positions_out)
	{
		constexpr int WAVES = 16;
		__shared__ int counts[WAVES][64];
		const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
		const int first = blockIdx.x * 64, position = first + lane;
		const int key = position < count ? key_of(tokens[position], classes) : 0;
		const int each = (count + WAVES - 1) / WAVES, from = min(wave * each, count), to = min(from + each, count);
		int before = 0;
		/* neither of the workgroup's own tokens nor of those behind counts an equal one, of those before it does */
		const auto count_below = [&](int begin, int end, int limit) __attribute__((always_inline))
		{
#pragma unroll 16
			for (int i = begin; i < end; i++)
				before += key_of(tokens[i], classes) < limit ? 1 : 0;
		};
		count_below(from, min(to, first), key + 1);
		count_below(max(from, first + 64), to, key);
		for (int i = max(from, first); i < min(to, first + 64); i++)
			before += key_of(tokens[i], classes) < key + (i < position ? 1 : 0) ? 1 : 0;
		counts[wave][lane] = before;
		__syncthreads();
		if (wave == 0 && position < count)
		{
			int place = 0;
#pragma unroll
			for (int w = 0; w < WAVES; w++)
				place += counts[w][lane];
			keys_out[place] = key;
			positions_out[place] = position;
		}
	}
	/*
	 * More of them: a launch that counts the digits of every group's tokens and one that puts them in place, for every digit of up to 11 bits. At most 64 groups, so that each can add up the others' counts by itself (that it also
	 * counts the others' tokens, without the first launch, takes 16 us where the two take 12, at 16384 tokens). So from 65536 tokens on the groups grow instead, a quarter of the compute units sort, and tokens are read twice: a digit of
	 * 131072 takes 14 us, of 262144 19. `keys` null: the tokens themselves, which stand where they are
	 */
	constexpr int SORT_GROUPS = 64, SORT_WAVES = 8, SORT_THREADS = 64 * SORT_WAVES;
	struct SortPass
	{
			const int *tokens, *keys, *positions;
			int *keys_out, *positions_out;
			int *counts; /* [groups][2^bits] */
			int count, classes, shift, bits, per_group; /* per_group: a multiple of 512 */

			__device__ __forceinline__ int key(int i) const
			{
				return keys != nullptr ? keys[i] : key_of(tokens[i], classes);
			}
			__device__ __forceinline__ int digit(int key) const
			{
				return (key >> shift) & ((1 << bits) - 1);
			}
			/* counters[digit] of the tokens of [first, last); several tokens of a thread on their way at a time */
			template<int THREADS>
			__device__ __forceinline__ void count_digits(int *counters, int first, int last, int thread) const
			{
				constexpr int AHEAD = 8;
				for (int i = first + thread; i < last; i += AHEAD * THREADS)
				{
					int k[AHEAD];
#pragma unroll
					for (int u = 0; u < AHEAD; u++)
						k[u] = key(min(i + u * THREADS, last - 1));
#pragma unroll
					for (int u = 0; u < AHEAD; u++)
						if (i + u * THREADS < last)
							atomicAdd(&counters[digit(k[u])], 1);
				}
			}
	};
	__global__ __launch_bounds__(SORT_THREADS) void kernel_sort_count(SortPass p)
	{
		extern __shared__ int counters[];
		const int digits = 1 << p.bits;
		for (int d = threadIdx.x; d < digits; d += SORT_THREADS)
			counters[d] = 0;
		__syncthreads();
		const int first = blockIdx.x * p.per_group, last = first + min(p.per_group, p.count - first);
		p.count_digits<SORT_THREADS>(counters, first, last, threadIdx.x);
		__syncthreads();
		for (int d = threadIdx.x; d < digits; d += SORT_THREADS)
			p.counts[blockIdx.x * digits + d] = counters[d];
	}
	/* KEPT: a wavefront's share is at most 128 tokens, which it reads once */
	template<bool KEPT>
	__global__ __launch_bounds__(SORT_THREADS) void kernel_sort_place(SortPass p)
	{
		extern __shared__ int counters[]; /* [wavefronts][digits]; of the groups before [digits], of those behind */
		__shared__ int waves[SORT_WAVES];
		const int digits = 1 << p.bits, groups = gridDim.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
		int *before = counters + SORT_WAVES * digits, *behind = before + digits, *mine = counters + wave * digits;
		/* a wavefront has an eighth of the group's tokens, in their order */
		const int group_first = blockIdx.x * p.per_group, group_last = group_first + min(p.per_group, p.count - group_first), share = p.per_group / SORT_WAVES;
		const int first = group_first + wave * share, here = max(0, min(share, group_last - first));
		constexpr int ROUNDS = 2, AHEAD = 8;
		int keys[ROUNDS], positions[ROUNDS];
		if constexpr (KEPT)
#pragma unroll
			for (int u = 0; u < ROUNDS; u++)
			{
				const int from = min(first + 64 * u + lane, p.count - 1);
				keys[u] = p.key(from);
				positions[u] = p.keys != nullptr ? p.positions[from] : from;
			}
		for (int d = threadIdx.x; d < (SORT_WAVES + 2) * digits; d += SORT_THREADS)
			counters[d] = 0;
		__syncthreads();
		if constexpr (KEPT)
		{
#pragma unroll
			for (int u = 0; u < ROUNDS; u++)
				if (64 * u + lane < here)
					atomicAdd(&mine[p.digit(keys[u])], 1);
		}
		else
			p.count_digits<64>(mine, first, first + here, lane);
		/* the groups' counts of four digits by a thread, every team of threads those of other groups: few reads wait for one another. us of embedding gradients, so / a digit of all
		   groups by a thread: 57600 x 256 of 400 classes 24.7 / 26.4, 40000 x 64 of 1500 32.9 / 39.0, 65536 x 64 of 131072 45.9 / 48.9 */
		typedef int int4_t __attribute__((ext_vector_type(4)));
		const int lanes = digits / 4, teams = SORT_THREADS / lanes, team = threadIdx.x / lanes, digit = static_cast<int>(threadIdx.x) % lanes * 4;
		int4_t sum_before = { 0, 0, 0, 0 }, sum_behind = sum_before;
		for (int g = team; g < groups; g += AHEAD * teams)
		{
			int4_t c[AHEAD];
#pragma unroll
			for (int a = 0; a < AHEAD; a++)
				c[a] = *reinterpret_cast<const int4_t*>(p.counts + min(g + a * teams, groups - 1) * digits + digit);
#pragma unroll
			for (int a = 0; a < AHEAD; a++)
			{
				const int of = g + a * teams;
				if (of < static_cast<int>(blockIdx.x))
					sum_before += c[a];
				if (of > static_cast<int>(blockIdx.x) && of < groups)
					sum_behind += c[a];
			}
		}
		if (team < groups)
#pragma unroll
			for (int e = 0; e < 4; e++)
			{
				atomicAdd(&before[digit + e], sum_before[e]);
				atomicAdd(&behind[digit + e], sum_behind[e]);
			}
		__syncthreads();
		const int each = max(1, digits / SORT_THREADS); /* neighbouring digits of a thread */
		int sum = 0;
		for (int d = threadIdx.x * each; d < min(static_cast<int>(threadIdx.x + 1) * each, digits); d++)
		{
			sum += before[d] + behind[d];
#pragma unroll
			for (int w = 0; w < SORT_WAVES; w++)
				sum += counters[w * digits + d];
		}
		int smaller = scan_exclusive<SORT_WAVES>(sum, waves);
		for (int d = threadIdx.x * each; d < min(static_cast<int>(threadIdx.x + 1) * each, digits); d++)
		{
			int at = smaller + before[d];
#pragma unroll
			for (int w = 0; w < SORT_WAVES; w++)
			{
				const int n = counters[w * digits + d];
				counters[w * digits + d] = at;
				at += n;
			}
			smaller = at + behind[d];
		}
		__syncthreads();
		const auto place_tokens = [&](bool there, int key, int position) __attribute__((always_inline))
		{
			const int digit = p.digit(key);
			const uint64_t same = lanes_alike(digit, p.bits, there);
			const int below = lanes_below(same);
			const int place = mine[digit] + below;
			wave_in_order();
			if (there && below == 0)
				mine[digit] += __popcll(same);
			wave_in_order();
			if (there)
			{
				p.keys_out[place] = key;
				p.positions_out[place] = position;
			}
		};
		if constexpr (KEPT)
		{
#pragma unroll
			for (int u = 0; u < ROUNDS; u++)
				place_tokens(64 * u + lane < here, keys[u], positions[u]);
		}
		else
			for (int i = 0; i < here; i += 64)
			{
				const int from = first + min(i + lane, here - 1);
				place_tokens(i + lane < here, p.key(from), p.keys != nullptr ? p.positions[from] : from);
			}
	}

	/* ---- backward ----------------------------------------------------------------------------------------------------------- */
	/*
	 * A class's rows are added up by those who write its row of the table; but where one class has many (a few tokens are in every line), they would wait for it alone. The list is therefore cut into chunks of 64 places (32 where a row takes
	 * all threads of a workgroup, so that nothing adds up rows side by side: 20011 x 1001 of 5003 fp32 43.5 us, with 64 45), and a class of as many rows and more has every chunk that begins with it added up by a workgroup of its own, beside those
	 * that write the other classes' rows; a second launch adds these sums in fp32 and the rows before the class's first whole chunk, less than a chunk's, and writes the class's row. None asks more than the list to know who does
	 * what. (With the chunks in a launch of their own before all rows, which then joined them: us, so / that way, 16384 x 4096 of 65536 classes fp16 173 / 176, 20011 x 1001 of 5003 fp32 43.5 / 45.5.)
	 */
	constexpr int MOST_OF_CHUNK = 64;
	template<typename T, typename Out>
	struct TableGradient
	{
			const int *keys, *positions; /* in order */
			const T *dy;
			float *partial; /* [chunks][columns] */
			int *ranges; /* [classes][2], of those with chunks of their own: first place and the one behind the last */
			Out *out;
			int count, classes, columns, classes_of_group, lanes, spans, chunk, chunks; /* chunks: workgroups for them, or 0; lanes: threads of a row, a power of two; spans: that a row takes of them */
			float scale, beta;
			bool past; /* the caches */
	};
	/* the first place of [first, first + length) whose key is not below `key` */
	__device__ __forceinline__ int lower_bound(const int *keys, int first, int length, int key)
	{
		while (length > 0)
		{
			const int half = length / 2;
			const bool below = keys[first + half] < key;
			first = below ? first + half + 1 : first;
			length = below ? length - half - 1 : half;
		}
		return first;
	}
	/* the same by a whole wavefront, which looks at 64 places at a time: three reads one after another where halving takes 17 */
	__device__ __forceinline__ int lower_bound_by_wave(const int *keys, int length, int key)
	{
		const int lane = threadIdx.x & 63;
		int first = 0;
		while (length > 0)
		{
			const int step = (length + 63) / 64, at = (lane + 1) * step - 1;
			const bool below = at < length && keys[first + min(at, length - 1)] < key;
			const int whole = __popcll(__ballot(below));
			first += whole * step;
			length = min(step - 1, length - whole * step);
		}
		return first;
	}
	/*
	 * v += the rows of every `step`th place from `first` on, AHEAD of them on their way at a time. row(i): where the i-th lies. Places behind the last one read it once more and count for nothing by a selection: the compiler
	 * would move loads into a branch, where they wait for all others.
	 */
	template<typename T, int AHEAD, int VEC, typename Row>
	__device__ __forceinline__ void add_rows(float (&v)[VEC], int first, int last, int step, Row &&row)
	{
		for (int i = first; i < last; i += AHEAD * step)
		{
			Elements<T, VEC> x[AHEAD];
#pragma unroll
			for (int u = 0; u < AHEAD; u++)
				x[u].load(row(min(i + u * step, last - 1)));
			__builtin_amdgcn_sched_barrier(0); /* else they are asked for one by one, to spare registers */
#pragma unroll
			for (int u = 0; u < AHEAD; u++)
#pragma unroll
				for (int e = 0; e < VEC; e++)
					v[e] += i + u * step < last ? x[u][e] : 0.0f;
		}
	}
	/*
	 * The sums of a workgroup's 256 / lanes groups of threads in the first of them, always in the same order: those of a wavefront by exchange, the wavefronts' in LDS. Every thread calls it. (All of them in LDS, by the first
	 * group's threads one after another: us, embedding gradients so / that way, 31058 x 16 of 119601 classes 36 / 57, 57600 x 64 of 400 25 / 28, 65536 x 64 of 131072 49 / 54.)
	 */
	template<int VEC>
	__device__ __forceinline__ void join_groups(float (&v)[VEC], int lanes, float (*meeting)[VEC])
	{
		if (lanes == 256)
			return;
		for (int offset = 32; offset >= lanes; offset >>= 1)
#pragma unroll
			for (int e = 0; e < VEC; e++)
				v[e] += __shfl_xor(v[e], offset);
		__syncthreads();
		if (static_cast<int>(threadIdx.x & 63) < lanes)
#pragma unroll
			for (int e = 0; e < VEC; e++)
				meeting[threadIdx.x][e] = v[e];
		__syncthreads();
		const int step = max(lanes, 64);
		if (static_cast<int>(threadIdx.x) < lanes)
			for (int t = threadIdx.x + step; t < 256; t += step)
#pragma unroll
				for (int e = 0; e < VEC; e++)
					v[e] += meeting[t][e];
	}
	/* whether the chunk at `first` begins with a class of a chunk's rows and more: as many neighbouring places are the class's with `first` among them. Of a wavefront; the same in all of them */
	template<typename T, typename Out>
	__device__ __forceinline__ bool begins_with_many(const TableGradient<T, Out> &p, int first, int key)
	{
		const int lane = threadIdx.x & 63, from = first - lane, to = from + p.chunk - 1;
		const bool all = lane < p.chunk && from >= 0 && to < p.count && p.keys[max(from, 0)] == key && p.keys[min(to, p.count - 1)] == key;
		return key < p.classes && __ballot(all) != 0;
	}
	/* a thread's column of a row, and where it lies */
	template<typename T, typename Out, int VEC>
	struct Column
	{
			int group, groups;
			bool inside;
			RowPlace place;

			__device__ __forceinline__ Column(const TableGradient<T, Out> &p, int span) :
					group(threadIdx.x / p.lanes),
					groups(256 / p.lanes)
			{
				const int column = (span * p.lanes + static_cast<int>(threadIdx.x) % p.lanes) * VEC;
				inside = column < p.columns;
				place = place_in_row<VEC>(min(column, p.columns - 1), p.columns);
			}
			__device__ __forceinline__ const T* of_list(const TableGradient<T, Out> &p, int i) const
			{
				return place.in(p.dy + static_cast<size_t>(p.positions[i]) * p.columns);
			}
			__device__ __forceinline__ Out* of_table(const TableGradient<T, Out> &p, int c) const
			{
				return place.in(p.out + static_cast<size_t>(c) * p.columns);
			}
			__device__ __forceinline__ float* of_chunk(const TableGradient<T, Out> &p, int i) const
			{
				return place.in(p.partial + static_cast<size_t>(i) * p.columns);
			}
			/* old: what is added to, if anything is */
			__device__ __forceinline__ void write(const TableGradient<T, Out> &p, int c, float (&v)[VEC], const Elements<Out, VEC> &old) const
			{
#pragma unroll
				for (int e = 0; e < VEC; e++)
					v[e] = p.beta != 0.0f ? fmaf(p.beta, old[e], p.scale * v[e]) : p.scale * v[e];
				if (p.past)
					store_past_caches<VEC>(of_table(p, c), v, place.skip);
				else
					store_nearest<VEC>(of_table(p, c), v, place.skip);
			}
	};
	constexpr int AHEAD = 8;
	template<int VEC>
	__device__ __forceinline__ void clear(float (&v)[VEC])
	{
#pragma unroll
		for (int e = 0; e < VEC; e++)
			v[e] = 0.0f;
	}
	template<typename T, typename Out, int VEC>
	__device__ __forceinline__ void sum_chunk(const TableGradient<T, Out> &p, int chunk, int span, float (*meeting)[VEC])
	{
		const int first = chunk * p.chunk, lane = threadIdx.x & 63, key = p.keys[first];
		if (!begins_with_many(p, first, key))
			return;
		const bool mine = lane < p.chunk && first + lane < p.count && p.keys[min(first + lane, p.count - 1)] == key;
		const int here = __popcll(__ballot(mine));
		const Column<T, Out, VEC> column(p, span);
		float v[VEC];
		clear(v);
		add_rows<T, AHEAD>(v, first + column.group, first + here, column.groups, [&](int i) __attribute__((always_inline))
		{
			return column.of_list(p, i);
		});
		join_groups<VEC>(v, p.lanes, meeting);
		if (column.group == 0 && column.inside)
			store_nearest<VEC>(column.of_chunk(p, chunk), v, column.place.skip);
	}
	/* of the class that has its first whole chunk here: that chunk's sum, the others', and the rows before */
	template<typename T, typename Out, int VEC>
	__global__ __launch_bounds__(256) void kernel_join_chunks(TableGradient<T, Out> p)
	{
		__shared__ float meeting[256][VEC];
		const int chunk = blockIdx.x / p.spans, span = blockIdx.x % p.spans, first = chunk * p.chunk, key = p.keys[first];
		if (!begins_with_many(p, first, key) || (chunk > 0 && p.keys[first - p.chunk] == key))
			return;
		const int begin = p.ranges[2 * key], end = p.ranges[2 * key + 1];
		const Column<T, Out, VEC> column(p, span);
		Elements<Out, VEC> old;
		if (p.beta != 0.0f && column.group == 0)
			old.load(column.of_table(p, key));
		float v[VEC];
		clear(v);
		add_rows<T, AHEAD>(v, begin + column.group, first, column.groups, [&](int i) __attribute__((always_inline))
		{
			return column.of_list(p, i);
		});
		add_rows<float, AHEAD>(v, chunk + column.group, (end + p.chunk - 1) / p.chunk, column.groups, [&](int i) __attribute__((always_inline))
		{
			return static_cast<const float*>(column.of_chunk(p, i));
		});
		join_groups<VEC>(v, p.lanes, meeting);
		if (column.group == 0 && column.inside)
			column.write(p, key, v, old);
	}
	constexpr int MOST_CLASSES_OF_GROUP = 1024;
	/*
	 * A class of fewer rows is one group's of threads, which may be a small part of the workgroup; of more, the whole workgroup's. us with 8 / 16 / 32: 57600 x 256 of 400 classes 26.3 / 26.3 / 28.6, 65536 x 64 of 131072 50.7 / 49.1 / 46.9, 31058 x 16 of 119601 38.8 / 36.2 / 36.6
	 */
	constexpr int ROWS_OF_ALL = 16;
	template<typename T, typename Out, int VEC>
	__global__ __launch_bounds__(256) void kernel_table_gradient(TableGradient<T, Out> p)
	{
		__shared__ int bounds[MOST_CLASSES_OF_GROUP + 1], large[MOST_CLASSES_OF_GROUP], ends[2], large_ones;
		__shared__ float meeting[256][VEC];
		const int unit = static_cast<int>(blockIdx.x / p.spans) - p.chunks, span = blockIdx.x % p.spans;
		if (unit < 0)
			return sum_chunk<T, Out, VEC>(p, unit + p.chunks, span, meeting);
		const int first_class = unit * p.classes_of_group, classes = min(p.classes_of_group, p.classes - first_class);
		if (threadIdx.x < 128)
		{
			const int wave = threadIdx.x >> 6, bound = lower_bound_by_wave(p.keys, p.count, first_class + wave * classes);
			if ((threadIdx.x & 63) == 0)
				ends[wave] = bound;
		}
		__syncthreads();
		if (threadIdx.x == 0)
			large_ones = 0;
		/* where every class begins: between two neighbours of the list all classes up to the second one's begin there; a long list is searched instead */
		const int list_first = ends[0], list_last = ends[1];
		if (list_last - list_first <= 4 * 256)
		{
			for (int i = list_first + threadIdx.x; i <= list_last; i += 256)
			{
				const int before = i > list_first ? p.keys[i - 1] - first_class : -1, here = i < list_last ? p.keys[i] - first_class : classes;
				for (int c = before + 1; c <= here; c++)
					bounds[c] = i;
			}
		}
		else
			for (int c = threadIdx.x; c <= classes; c += 256)
				bounds[c] = c == 0 ? list_first : c == classes ? list_last : lower_bound(p.keys, list_first, list_last - list_first, first_class + c);
		__syncthreads();
		const Column<T, Out, VEC> column(p, span);
		const int groups = column.groups, group = column.group;
		/* one group's of threads; the workgroup's; that of the chunks and their joining */
		const auto rows_of = [&](int c)
		{
			return bounds[c + 1] - bounds[c];
		};
		const auto of_group = [&](int c)
		{
			return rows_of(c) < (groups > 1 ? ROWS_OF_ALL : p.chunk);
		};
		for (int c = threadIdx.x; c < classes; c += 256)
			if (!of_group(c) && rows_of(c) < p.chunk)
				large[atomicAdd(&large_ones, 1)] = c; /* in any order: each has a row of its own */
			else if (rows_of(c) >= p.chunk && span == 0)
			{
				p.ranges[2 * (first_class + c)] = bounds[c];
				p.ranges[2 * (first_class + c) + 1] = bounds[c + 1];
			}
		float v[VEC];
		Elements<Out, VEC> old;
		if (column.inside)
		{
			/* neighbouring classes of a group of threads: first those without rows, which wait for nothing; then the others' rows in one go, whichever class they are of */
			const int each = (classes + groups - 1) / groups, begin = min(group * each, classes), end = min(begin + each, classes);
			if (p.beta != 1.0f)
				for (int c = begin; c < end; c++)
					if (rows_of(c) == 0)
					{
						clear(v);
						if (p.beta != 0.0f)
							old.load(column.of_table(p, first_class + c));
						column.write(p, first_class + c, v, old);
					}
			for (int c = begin; c < end;)
			{
				if (!of_group(c))
				{
					c++;
					continue;
				}
				const int first = bounds[c];
				while (c < end && of_group(c))
					c++;
				const int last = bounds[c];
				int current = -1;
				for (int i = first; i < last; i += AHEAD)
				{
					Elements<T, VEC> x[AHEAD];
					int key[AHEAD];
#pragma unroll
					for (int u = 0; u < AHEAD; u++)
					{
						key[u] = p.keys[min(i + u, last - 1)];
						x[u].load(column.of_list(p, min(i + u, last - 1)));
					}
					__builtin_amdgcn_sched_barrier(0);
#pragma unroll
					for (int u = 0; u < AHEAD; u++)
					{
						if (key[u] != current)
						{
							if (current >= 0)
								column.write(p, current, v, old);
							current = key[u];
							if (p.beta != 0.0f)
								old.load(column.of_table(p, current));
							clear(v);
						}
#pragma unroll
						for (int e = 0; e < VEC; e++)
							v[e] += i + u < last ? x[u][e] : 0.0f; /* behind the last place: its class, nothing more */
					}
				}
				if (current >= 0)
					column.write(p, current, v, old);
			}
		}
		__syncthreads();
		for (int i = 0; i < large_ones; i++)
		{
			const int c = large[i];
			clear(v);
			if (p.beta != 0.0f && group == 0)
				old.load(column.of_table(p, first_class + c));
			add_rows<T, AHEAD>(v, bounds[c] + group, bounds[c + 1], groups, [&](int at) __attribute__((always_inline))
			{
				return column.of_list(p, at);
			});
			join_groups<VEC>(v, p.lanes, meeting);
			if (group == 0 && column.inside)
				column.write(p, first_class + c, v, old);
		}
	}

	/* ---- sizes ---------------------------------------------------------------------------------------------------------------- */
	struct EmbeddingShape
	{
			int rows, classes, columns;
	};
	EmbeddingShape embedding_shape(const mlShape_t &tokens, const mlShape_t &table, mlDataType_t dtype, const char *name)
	{
		const std::string who(name);
		MLHIP_REQUIRE(dtype == DTYPE_FLOAT16 || dtype == DTYPE_FLOAT32, who + ": unsupported data type");
		MLHIP_REQUIRE(tokens.rank >= 1 && tokens.rank <= 6 && table.rank == 2, who + ": tokens need one to six dimensions, the table must be [classes, features]");
		for (int i = 0; i < tokens.rank; i++)
			MLHIP_REQUIRE(tokens.dim[i] >= 0, who + ": negative dimension");
		MLHIP_REQUIRE(table.dim[0] > 0 && table.dim[1] > 0, who + ": there must be classes and features");
		const size_t rows = volume(tokens);
		MLHIP_REQUIRE(rows <= (1 << 28) && table.dim[0] <= (1 << 28) && table.dim[1] <= (1 << 18), who + ": too many tokens, classes or features");
		return EmbeddingShape { static_cast<int>(rows), table.dim[0], table.dim[1] };
	}
	struct SortPlan
	{
			int bits, passes, digit_bits, groups, per_group;
	};
	SortPlan sort_plan(const EmbeddingShape &s)
	{
		SortPlan plan { };
		while ((s.classes >> plan.bits) > 0)
			plan.bits++;
		plan.passes = ceil_div(plan.bits, 11);
		plan.digit_bits = std::max(2, ceil_div(plan.bits, plan.passes)); /* counts are read four at a time */
		plan.per_group = std::max(1024, static_cast<int>(round_up(ceil_div(s.rows, SORT_GROUPS), 512)));
		plan.groups = ceil_div(s.rows, plan.per_group);
		return plan;
	}
	/*
	 * Counting takes longer the more tokens there are, a digit about as long for all up to 65536, longer ones longer. us of gradients of rows of 64, counted / by digits: 400 classes, 3000, 4096 and 6000 tokens 19.7 / 20.3,
	 * 20.9 / 20.0, 24.3 / 20.4; 1500 classes, 4096, 6000 and 8192 22.9 / 25.6, 26.2 / 26.4, 29.6 / 26.9; 8000 classes, 6000, 8192 and 12000 26.0 / 28.3, 29.2 / 29.4, 34.8 / 30.0; 100000 classes 30.5 / 33.4, 32.2 / 34.0, 38.0 / 34.2
	 */
	bool sorted_by_counting(const EmbeddingShape &s)
	{
		return s.rows <= (s.classes < 512 ? 3500 : s.classes < 2048 ? 6000 : 8192);
	}
	/* threads that a row takes, a power of two */
	int lanes_of_row(const EmbeddingShape &s, int vector)
	{
		int lanes = 1;
		while (lanes < 256 && lanes * vector < s.columns)
			lanes *= 2;
		return lanes;
	}
	int chunk_of(const EmbeddingShape &s, int vector)
	{
		return lanes_of_row(s, vector) == 256 ? 32 : MOST_OF_CHUNK;
	}
	/* elements of dy that a thread takes at a time */
	int vector_of(const EmbeddingShape &s, mlDataType_t dtype)
	{
		const int vector = 16 / size_of(dtype);
		return s.columns >= vector ? vector : 1;
	}
	struct EmbeddingSpace
	{
			size_t keys[2], positions[2], counts, partial, ranges, total;
	};
	EmbeddingSpace embedding_space(const EmbeddingShape &s, mlDataType_t dtype)
	{
		EmbeddingSpace space { };
		size_t at = 0;
		const auto take = [&](size_t bytes)
		{
			const size_t begin = at;
			at += round_up(bytes, 256);
			return begin;
		};
		if (s.rows > 0)
		{
			const SortPlan plan = sort_plan(s);
			const bool small = sorted_by_counting(s);
			for (int i = 0; i < (small || plan.passes == 1 ? 1 : 2); i++)
			{
				space.keys[i] = take(sizeof(int) * s.rows);
				space.positions[i] = take(sizeof(int) * s.rows);
			}
			space.counts = take(small ? 0 : (sizeof(int) * plan.groups << plan.digit_bits));
			const int chunk = chunk_of(s, vector_of(s, dtype));
			space.partial = take(s.rows >= chunk ? sizeof(float) * ceil_div(s.rows, chunk) * s.columns : 0);
			space.ranges = take(s.rows >= chunk ? 2 * sizeof(int) * s.classes : 0);
		}
		space.total = at;
		return space;
	}

	template<typename T, int VEC>
	void embedding_forward(hipStream_t stream, const EmbeddingShape &s, const int *tokens, const T *table, T *y, float scale)
	{
		const int vectors = ceil_div(s.columns, VEC);
		const size_t count = static_cast<size_t>(s.rows) * vectors;
		const auto launch = [&](auto kernel, int each)
		{
			const size_t groups = std::min<size_t>((count + 256 * each - 1) / (256 * each), 1 << 20);
			hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned int>(groups)), dim3(256), 0, stream, tokens, table, y, s.rows, s.columns, s.classes, vectors, scale);
		};
		/* a vector to a thread / four of them, us on the device: 4096 x 256 fp16 2.7 / 3.3, 16384 x 256 4.6 / 4.6, 32768 x 256 6.5 / 6.1, 65536 x 256 9.9 / 9.1 */
		if (count < (1 << 19))
			launch(kernel_embedding_forward<T, VEC, 1>, 1);
		else
			launch(kernel_embedding_forward<T, VEC, 4>, 4);
		MLHIP_CHECK(hipGetLastError());
	}
	/* the tokens in order: keys and positions */
	std::pair<const int*, const int*> sort_tokens(hipStream_t stream, const EmbeddingShape &s, const EmbeddingSpace &space, const int *tokens, uint8_t *workspace)
	{
		const SortPlan plan = sort_plan(s);
		const auto keys = [&](int i)
		{
			return reinterpret_cast<int*>(workspace + space.keys[i]);
		};
		const auto positions = [&](int i)
		{
			return reinterpret_cast<int*>(workspace + space.positions[i]);
		};
		if (sorted_by_counting(s))
		{
			hipLaunchKernelGGL(kernel_sort_by_counting, dim3(ceil_div(s.rows, 64)), dim3(1024), 0, stream, tokens, s.rows, s.classes, keys(0), positions(0));
			MLHIP_CHECK(hipGetLastError());
			return { keys(0), positions(0) };
		}
		for (int pass = 0; pass < plan.passes; pass++)
		{
			const int from = (pass + 1) & 1, to = pass & 1;
			const SortPass p { tokens, pass == 0 ? nullptr : keys(from), pass == 0 ? nullptr : positions(from), keys(to), positions(to), reinterpret_cast<int*>(workspace + space.counts), s.rows, s.classes,
					pass * plan.digit_bits, plan.digit_bits, plan.per_group };
			const int bytes = static_cast<int>(sizeof(int)) << plan.digit_bits;
			hipLaunchKernelGGL(kernel_sort_count, dim3(plan.groups), dim3(SORT_THREADS), bytes, stream, p);
			auto place = plan.per_group <= 2 * SORT_THREADS ? kernel_sort_place<true> : kernel_sort_place<false>;
			ensure_dynamic_lds(reinterpret_cast<const void*>(place), (SORT_WAVES + 2) * bytes);
			hipLaunchKernelGGL(place, dim3(plan.groups), dim3(SORT_THREADS), (SORT_WAVES + 2) * bytes, stream, p);
			MLHIP_CHECK(hipGetLastError());
		}
		const int last = (plan.passes - 1) & 1;
		return { keys(last), positions(last) };
	}
	template<typename T, typename Out, int VEC>
	void table_gradient(hipStream_t stream, const EmbeddingShape &s, const int *keys, const int *positions, const T *dy, float *partial, int *ranges, float scale, float beta, Out *out)
	{
		const int lanes = lanes_of_row(s, VEC);
		const int spans = ceil_div(s.columns, lanes * VEC);
		const size_t units = static_cast<size_t>(s.classes) * spans;
		/* classes of a workgroup: their search is its beginning, but four workgroups to a compute unit come first. us with 16 / 32 / 64 at most for wide rows: 16384 x 4096 of 65536 174 / 172 / 176 */
		const int most = static_cast<int>(std::min<size_t>(std::max(32, 1024 / lanes), std::max<size_t>(1, units / 1024)));
		const int chunk = chunk_of(s, VEC), chunks = s.rows >= chunk ? ceil_div(s.rows, chunk) : 0;
		const TableGradient<T, Out> p { keys, positions, dy, partial, ranges, out, s.rows, s.classes, s.columns, most, lanes, spans, chunk, chunks, scale, beta,
				past_caches(s.classes, s.columns * sizeof(Out)) };
		hipLaunchKernelGGL((kernel_table_gradient<T, Out, VEC>), dim3((static_cast<unsigned int>(ceil_div(s.classes, most)) + chunks) * spans), dim3(256), 0, stream, p);
		if (chunks > 0)
		{
			/* several groups of threads to a row, however wide it is: a class's chunks wait for one another otherwise */
			TableGradient<T, Out> joined = p;
			joined.lanes = std::min(lanes, 64);
			joined.spans = ceil_div(s.columns, joined.lanes * VEC);
			hipLaunchKernelGGL((kernel_join_chunks<T, Out, VEC>), dim3(static_cast<unsigned int>(chunks) * joined.spans), dim3(256), 0, stream, joined);
		}
		MLHIP_CHECK(hipGetLastError());
	}
	template<typename T, typename Out>
	void embedding_backward(hipStream_t stream, const EmbeddingShape &s, const int *tokens, const T *dy, float scale, float beta, Out *out, const EmbeddingSpace &space, uint8_t *workspace)
	{
		constexpr int VEC = 16 / sizeof(T);
		const int *keys = nullptr, *positions = nullptr;
		float *partial = reinterpret_cast<float*>(workspace + space.partial);
		int *ranges = reinterpret_cast<int*>(workspace + space.ranges);
		if (s.rows > 0)
			std::tie(keys, positions) = sort_tokens(stream, s, space, tokens, workspace);
		if (s.columns >= VEC)
			table_gradient<T, Out, VEC>(stream, s, keys, positions, dy, partial, ranges, scale, beta, out);
		else
			table_gradient<T, Out, 1>(stream, s, keys, positions, dy, partial, ranges, scale, beta, out);
	}
	void check_tokens(const mlTensor_t &tokens, const EmbeddingShape &s, const char *name)
	{
		MLHIP_REQUIRE(tokens.dtype == DTYPE_INT32, std::string(name) + ": tokens must be int32");
		MLHIP_REQUIRE((s.rows == 0 || tokens.data != nullptr) && on_elements(tokens), std::string(name) + ": null or misaligned tokens");
	}
	/* one row of features for every token, aligned to an element */
	bool rows_of(const mlTensor_t &t, const EmbeddingShape &s)
	{
		return t.rank >= 1 && last_dim(t) == s.columns && volume(t) == static_cast<size_t>(s.rows) * s.columns && (s.rows == 0 || t.data != nullptr) && on_elements(t);
	}
}

extern "C"
{
	using namespace mlhip;

	void hip_embedding_forward(mlContext_t context, const mlTensor_t tokens, const mlTensor_t table, float scale, mlTensor_t y)
	try
	{
		const char *name = "embedding_forward";
		const EmbeddingShape s = embedding_shape(shape_of(tokens), shape_of(table), table.dtype, name);
		check_tokens(tokens, s, name);
		MLHIP_REQUIRE(std::isfinite(scale), "embedding_forward: the scale must be finite");
		MLHIP_REQUIRE(y.dtype == table.dtype && rows_of(y, s), "embedding_forward: the result must hold a row of the table's type and width for every token");
		if (s.rows == 0)
			return;
		MLHIP_REQUIRE(table.data != nullptr && on_elements(table), "embedding_forward: null or misaligned table");
		require_apart( { y }, { tokens, table }, name);
		const OnDeviceOf on(context);
		if (table.dtype == DTYPE_FLOAT16)
		{
			if (s.columns >= 8)
				embedding_forward<half_t, 8>(on.stream, s, ptr<int>(tokens), ptr<half_t>(table), ptr<half_t>(y), scale);
			else
				embedding_forward<half_t, 1>(on.stream, s, ptr<int>(tokens), ptr<half_t>(table), ptr<half_t>(y), scale);
		}
		else if (s.columns >= 4)
			embedding_forward<float, 4>(on.stream, s, ptr<int>(tokens), ptr<float>(table), ptr<float>(y), scale);
		else
			embedding_forward<float, 1>(on.stream, s, ptr<int>(tokens), ptr<float>(table), ptr<float>(y), scale);
	}
	catch (...)
	{
		return mlhip::entry_failed<void>();
	}

	size_t hip_embedding_get_workspace_size(mlShape_t tokens_shape, mlShape_t table_shape, mlDataType_t dtype)
	try
	{
		return embedding_space(embedding_shape(tokens_shape, table_shape, dtype, "embedding_get_workspace_size"), dtype).total;
	}
	catch (...)
	{
		return mlhip::entry_failed<size_t>();
	}

	void hip_embedding_backward(mlContext_t context, const mlTensor_t tokens, const mlTensor_t dy, float scale, float beta_weights, mlTensor_t dtable, void *workspace, size_t workspace_size)
	try
	{
		const char *name = "embedding_backward";
		if (dtable.data == nullptr)
			return;
		const EmbeddingShape s = embedding_shape(shape_of(tokens), shape_of(dtable), dy.dtype, name);
		check_tokens(tokens, s, name);
		MLHIP_REQUIRE(std::isfinite(scale), "embedding_backward: the scale must be finite"); /* classes without tokens get zeros, not zero times it */
		MLHIP_REQUIRE(rows_of(dy, s), "embedding_backward: there must be a gradient of the table's width for every token");
		MLHIP_REQUIRE(dtable.dtype == dy.dtype || dtable.dtype == DTYPE_FLOAT32, "embedding_backward: the table's gradient must be of the gradients' type or fp32");
		MLHIP_REQUIRE(on_elements(dtable), "embedding_backward: the table's gradient must be aligned to an element");
		const EmbeddingSpace space = embedding_space(s, dy.dtype);
		MLHIP_REQUIRE(space.total == 0 || (workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 256 == 0 && workspace_size >= space.total),
				"embedding_backward: the workspace is too small or not aligned to 256 bytes");
		require_apart( { dtable, Extent(workspace, workspace_size) }, { tokens, dy }, name);
		const OnDeviceOf on(context);
		uint8_t *memory = reinterpret_cast<uint8_t*>(workspace);
		if (dy.dtype == DTYPE_FLOAT32)
			embedding_backward<float, float>(on.stream, s, ptr<int>(tokens), ptr<float>(dy), scale, beta_weights, ptr<float>(dtable), space, memory);
		else if (dtable.dtype == DTYPE_FLOAT32)
			embedding_backward<half_t, float>(on.stream, s, ptr<int>(tokens), ptr<half_t>(dy), scale, beta_weights, ptr<float>(dtable), space, memory);
		else
			embedding_backward<half_t, half_t>(on.stream, s, ptr<int>(tokens), ptr<half_t>(dy), scale, beta_weights, ptr<half_t>(dtable), space, memory);
	}
	catch (...)
	{
		return mlhip::entry_failed<void>();
	}
}
