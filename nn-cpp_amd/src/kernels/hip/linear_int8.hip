// linear_int8.hip - which kernel a product of 8-bit codes takes (linear_int8_tile.hpp).
#include "linear_int8_tile.hpp"

#include <algorithm>

namespace nnh {

namespace i8 {

using Large = g16::Tile<256, 256, 128, 64>;
using Small = g16::Tile<128, 128, 64, 64>;

template <class S>
static int64_t tiles(int64_t V, int64_t rows) { return ((V + S::BM - 1) / S::BM) * ((rows + S::BN - 1) / S::BN); }

// 256 x 256 tiles from 200 of them on, a workgroup a CU; else 128 x 128 ones, two a CU, and the depth in runs, of 1024 codes at
// least, where these are fewer than 512.
struct Cut {
	bool large;
	int64_t parts, units;  // runs, and the depth of one in units of two codes
};
static Cut cut_of(int64_t rows, int64_t D, int64_t V) {
	const int64_t depth = (D + 15) / 16 * 8;
	if (tiles<Large>(V, rows) >= 200) return {true, 1, depth};
	const int64_t t = std::max<int64_t>(1, tiles<Small>(V, rows));
	Cut c{false, std::max<int64_t>(1, std::min(512 / t, depth / 512)), depth};
	c.units = ((depth + c.parts - 1) / c.parts + g16::BK - 1) / g16::BK * g16::BK;
	if (c.units > 0) c.parts = std::max<int64_t>(1, (depth + c.units - 1) / c.units);
	return c;
}

template <typename T>
static hipError_t tile_of_type(const LinearInt8Args& given, hipStream_t s) {
	const Cut c = cut_of(given.rows, given.D, given.V);
	LinearInt8Args a = given;
	a.part_units = (int)c.units;
	if (c.parts == 1) a.parts = nullptr;
	if (c.large) linear_int8_tile_kernel<Large, T><<<dim3((unsigned)tiles<Large>(a.V, a.rows)), Large::kThreads, 0, s>>>(a);
	else linear_int8_tile_kernel<Small, T><<<dim3((unsigned)tiles<Small>(a.V, a.rows), (unsigned)c.parts), Small::kThreads, 0, s>>>(a);
	hipError_t e = hipGetLastError();
	if (e != hipSuccess || c.parts == 1) return e;
	linear_int8_join_kernel<T><<<(unsigned)(((int64_t)a.rows * a.V + 255) / 256), 256, 0, s>>>(a, (int)c.parts);
	return hipGetLastError();
}

template <int I, int J, int NW, typename T>
static hipError_t few_launch(const LinearInt8Args& a, hipStream_t s) {
	const unsigned blocks = (unsigned)((a.V + 16 * I - 1) / (16 * I));
	if constexpr (J == 1) {
		if (a.whole) {
			linear_int8_few_kernel<I, J, NW, T, true><<<blocks, 64 * NW, 0, s>>>(a);
			return hipGetLastError();
		}
	}
	linear_int8_few_kernel<I, J, NW, T, false><<<blocks, 64 * NW, 0, s>>>(a);
	return hipGetLastError();
}
template <int J, typename T>
static hipError_t few_of(const LinearInt8Args& a, hipStream_t s) {
	if constexpr (J == 1) {
		// 32 columns to a workgroup where that still makes 512 of them (the rows' codes are then read half as often), else 16; the depth
		// over as many waves as bring 2048 together
		if (a.V >= 32 * 512) return few_launch<2, J, 4, T>(a, s);
		if (a.V >= 16 * 512) return few_launch<1, J, 4, T>(a, s);
	} else {
		// the rows' codes are as many bytes as those of 32 or 64 columns: the fewest columns that make one round of the 256 CUs, 64 at most
		// (32 rows, 4096 deep, 10240 columns: 64 to a workgroup 27 us, 32 31; 64 rows: 32 and 39; 8192 columns: 26 and 22 us, 32 and 26)
		if (a.V > 32 * 256) return few_launch<4, J, 4, T>(a, s);
		if (a.V > 16 * 256) return few_launch<2, J, 8, T>(a, s);
	}
	return few_launch<1, J, 8, T>(a, s);
}
template <typename T>
static hipError_t few(const LinearInt8Args& a, hipStream_t s) {
	if (a.rows <= 16) return few_of<1, T>(a, s);
	if (a.rows <= 32) return few_of<2, T>(a, s);
	return few_of<4, T>(a, s);
}

}  // namespace i8

// (64 rows, 4096 deep: 16384 columns 35 us here and 41 in tiles, 24576 55 and 46)
bool linear_int8_few(int64_t rows, int64_t V) { return rows <= 32 || (rows <= 64 && V <= 64 * 256); }
bool linear_int8_whole(int64_t rows, int64_t D) { return rows <= 16 && rows * i8::whole_pitch(D) <= i8::kWhole; }

size_t linear_int8_parts(int64_t rows, int64_t D, int64_t V) {
	if (linear_int8_few(rows, V)) return 0;
	const i8::Cut c = i8::cut_of(rows, D, V);
	return c.parts > 1 ? (size_t)(c.parts * rows * V) : 0;
}

hipError_t linear_int8(const LinearInt8Args& a, int type, hipStream_t s) {
	if (a.rows == 0 || a.V == 0) return hipSuccess;
	if (linear_int8_few(a.rows, a.V)) return type == kF32 ? i8::few<float>(a, s) : i8::few<__bf16>(a, s);
	return type == kF32 ? i8::tile_of_type<float>(a, s) : i8::tile_of_type<__bf16>(a, s);
}

}  // namespace nnh
