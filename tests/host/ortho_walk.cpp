// The walk over a round's items (ortho_walk.h) against the tiles themselves, for lists of shapes and for how far their tiles are split: every
// part of every tile is one item's, parts lie in places of their own, and whoever asks for an item or a tile that the round does not
// have is told so, without a look behind the last matrix.  Status 0: all lists sound.
#include "ortho_walk.h"

#include <cstdio>
#include <cstdlib>
#include <random>
#include <set>
#include <tuple>
#include <vector>

using namespace glb;

// The launch's parameters as the walk reads them; an index behind the last one ends the program.
template <class T>
struct Checked
{
	std::vector<T> v;
	const T& operator[](int i) const
	{
		if (i < 0 || i >= (int)v.size())
		{
			printf("element %d of %d\n", i, (int)v.size());
			exit(2);
		}
		return v[i];
	}
};
struct Shape
{
	int p, q;
};
struct Params
{
	struct
	{
		Checked<OrOp> op;
	} prog;
	Checked<Shape> mat;
	Checked<Checked<unsigned char>> split;
	int count;
};

static int failures = 0;
static void expect(bool ok, const char* what, const Params& P, int round, int bn)
{
	if (ok) return;
	if (++failures < 10) printf("%s: round %d, tiles of %d columns, %d matrices, first %d x %d\n", what, round, bn, P.count, P.mat[0].p, P.mat[0].q);
}

template <int BN>
static void walk(const Params& P, int round)
{
	const OrOp& o = P.prog.op[round];
	const bool symmetric = op_symmetric(o);
	int items = 0, splits = 0, slots = 0;
	for (int i = 0; i < P.count; ++i)
	{
		const int n = op_tiles(o, P.mat[i].p, P.mat[i].q, BN), s = P.split[i][round];
		items += n * s;
		if (s > 1) splits += n, slots += n * s;
	}
	std::set<std::tuple<int, int, int>> tiles;                // matrix and origin
	std::set<std::tuple<int, int, int, int>> parts;          // and where the part's k begins
	std::vector<int> taken(slots, 0);
	std::vector<long long> covered(P.count, 0);               // stages of all parts
	for (int t = 0; t < items; ++t)
	{
		OrItem it;
		if (!find_item<BN>(P, round, t, it))
		{
			expect(false, "an item is missing", P, round, BN);
			return;
		}
		const int p = P.mat[it.mat].p, q = P.mat[it.mat].q, kb = op_kb(o, p, q);
		expect(it.m0 >= 0 && it.m0 < p && it.m0 % OR_BM == 0 && it.n0 >= 0 && it.n0 < (symmetric ? p : q) && it.n0 % BN == 0, "a tile outside its matrix", P, round, BN);
		expect(!symmetric || it.n0 <= it.m0 + OR_BM - 1, "a tile above the diagonal", P, round, BN);
		expect(it.kb0 >= 0 && it.kb0 < it.kb1 && it.kb1 <= kb, "a part without its k", P, round, BN);
		expect(parts.insert({it.mat, it.m0, it.n0, it.kb0}).second, "a part twice", P, round, BN);
		tiles.insert({it.mat, it.m0, it.n0});
		covered[it.mat] += it.kb1 - it.kb0;
		if (it.split > 1)
		{
			expect(it.slot >= 0 && it.slot < slots && !taken[it.slot], "a part's place", P, round, BN);
			if (it.slot >= 0 && it.slot < slots) taken[it.slot] = 1;
		}
	}
	long long all = 0;
	for (int i = 0; i < P.count; ++i)
	{
		const int p = P.mat[i].p, q = P.mat[i].q;
		long long n = 0;
		for (int m0 = 0; m0 < p; m0 += OR_BM)
			for (int n0 = 0; n0 < (symmetric ? p : q); n0 += BN) n += !symmetric || n0 <= m0 + OR_BM - 1;
		all += n;
		expect(covered[i] == n * op_kb(o, p, q), "k of all parts", P, round, BN);
	}
	expect((long long)tiles.size() == all, "tiles of all matrices", P, round, BN);
	for (int t = 0; t < splits; ++t)
	{
		OrItem it;
		if (!find_split<BN>(P, round, t, it))
		{
			expect(false, "a split tile is missing", P, round, BN);
			return;
		}
		// its parts are those that the items wrote
		expect(it.split > 1 && it.slot >= 0 && it.slot + it.split <= slots && tiles.count({it.mat, it.m0, it.n0}), "a split tile", P, round, BN);
	}
	OrItem it;
	for (int beyond : {0, 1, 147, 1 << 20})
	{
		expect(!find_item<BN>(P, round, items + beyond, it), "an item behind the last one", P, round, BN);
		expect(!find_split<BN>(P, round, splits + beyond, it), "a split tile behind the last one", P, round, BN);
	}
}

int main()
{
	std::mt19937 rng(1);
	const int sizes[] = {1, 2, 63, 64, 65, 127, 128, 129, 200, 255, 256, 257, 300, 512, 640, 1000, 1025, 2048};
	auto size = [&]() { return sizes[rng() % (sizeof sizes / sizeof *sizes)]; };
	for (int list = 0; list < 400; ++list)
	{
		Params P;
		P.count = list < 18 ? 1 : 1 + (int)(rng() % 16);
		P.prog.op.v = {{ID_X, ID_X, ID_NONE, ID_A, 1, 0, 1}, {ID_A, ID_A, ID_A, ID_R, 1, 1, 1}, {ID_R, ID_X, ID_X, ID_X + 1, 1, 1, 1}};
		for (int i = 0; i < P.count; ++i)
		{
			const int a = list < 18 ? sizes[list] : size(), b = list < 18 ? sizes[list] : size();
			P.mat.v.push_back({a < b ? a : b, a < b ? b : a});
			Checked<unsigned char> split;
			for (const OrOp& o : P.prog.op.v)
			{
				const int kb = op_kb(o, P.mat.v.back().p, P.mat.v.back().q);
				split.v.push_back((unsigned char)(rng() % 2 ? 1 : 1 + rng() % (kb < 9 ? kb : 9)));
			}
			P.split.v.push_back(split);
		}
		for (int round = 0; round < 3; ++round)
		{
			walk<128>(P, round);
			walk<64>(P, round);
		}
	}
	printf("%d failures\n", failures);
	return failures != 0;
}
