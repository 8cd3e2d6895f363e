// Which tile of which matrix an item of a round is (orthogonalize.cu).
//
// The host counts a round's items and split tiles, the kernel's warps walk them.  A walk ends behind the last matrix, whatever number it is
// asked for: where the two ever disagreed, a warp gives up its round and says so, instead of reading on behind the launch's parameters.
//
// No device code, so that the walk can be run on the CPU (tests/host/ortho_walk.cpp).
#pragma once

#ifdef __CUDACC__
#define GL_WALK __host__ __device__ __forceinline__
#else
#define GL_WALK inline
#endif

namespace glb {

constexpr int OR_BM = 128;  // rows of a tile
// k per pipeline stage.  A stage costs the multiplying warp two waits and a commit, about 350 clocks, whatever its MMAs take: with
// stages of 32 k that bounded both tiles (530 clocks per 32 k on 128 columns, 350 to 400 now).
constexpr int OR_BK = 64;

// Matrices of parts that an operation names: two p x p, and the two X.
enum { ID_A = 0, ID_R = 1, ID_X = 2, ID_NONE = -1 };
// out = f (A B^T or A B) + w E; the factors hold the parts' scales
struct OrOp
{
	signed char a, b, e, out;  // out ID_NONE: the result
	float f, w, so;
};

// An operation's tiles of one matrix, of a symmetric product only those that reach the diagonal.
GL_WALK bool op_symmetric(const OrOp& o) { return o.b < ID_X || o.a >= ID_X; }
GL_WALK int op_kb(const OrOp& o, int p, int q) { return ((o.a >= ID_X ? q : p) + OR_BK - 1) / OR_BK; }
GL_WALK int tiles_of_row(int mt, int tn, int bn)
{
	const int c = (mt * OR_BM + OR_BM - 1) / bn + 1;
	return c < tn ? c : tn;
}
GL_WALK int op_tiles(const OrOp& o, int p, int q, int bn)
{
	const int tm = (p + OR_BM - 1) / OR_BM;
	if (!op_symmetric(o)) return tm * ((q + bn - 1) / bn);
	const int tn = (p + bn - 1) / bn;
	int n = 0;
	for (int mt = 0; mt < tm; ++mt) n += tiles_of_row(mt, tn, bn);
	return n;
}

struct OrItem
{
	int mat, m0, n0, kb0, kb1, split, slot;  // slot: of a split tile's first part
};
// the tile t of operation o
template <int BN>
GL_WALK void tile_origin(const OrOp& o, int p, int q, int t, int& m0, int& n0)
{
	const int tm = (p + OR_BM - 1) / OR_BM;
	if (!op_symmetric(o))
	{
		m0 = (t % tm) * OR_BM;
		n0 = (t / tm) * BN;
		return;
	}
	const int tn = (p + BN - 1) / BN;
	for (int mt = tm - 1;; --mt)
	{
		const int n = tiles_of_row(mt, tn, BN);
		if (t < n || mt == 0)
		{
			m0 = mt * OR_BM;
			n0 = t * BN;
			return;
		}
		t -= n;
	}
}
// Item t of a round: t < P.items[round].  False: there is none.  (PARAMS: prog.op[round], count, mat[i].p and .q, split[i][round])
template <int BN, class PARAMS>
GL_WALK bool find_item(const PARAMS& P, int round, int t, OrItem& it)
{
	const OrOp& o = P.prog.op[round];
	int slot = 0;
	for (int i = 0; i < P.count; ++i)
	{
		const int p = P.mat[i].p, q = P.mat[i].q, s = P.split[i][round];
		const int n = op_tiles(o, p, q, BN) * s;
		if (t < n)
		{
			const int tile = t / s, part = t - tile * s;
			const int kb = op_kb(o, p, q);
			it.mat = i;
			it.split = s;
			it.kb0 = kb * part / s;
			it.kb1 = kb * (part + 1) / s;
			it.slot = slot + t;
			tile_origin<BN>(o, p, q, tile, it.m0, it.n0);
			return true;
		}
		t -= n;
		if (s > 1) slot += n;
	}
	return false;
}
// Tile t of a round's split matrices: t < P.splits[round].  False: there is none.
template <int BN, class PARAMS>
GL_WALK bool find_split(const PARAMS& P, int round, int t, OrItem& it)
{
	const OrOp& o = P.prog.op[round];
	int slot = 0;
	for (int i = 0; i < P.count; ++i)
	{
		const int p = P.mat[i].p, q = P.mat[i].q, s = P.split[i][round];
		if (s < 2) continue;
		const int n = op_tiles(o, p, q, BN);
		if (t < n)
		{
			it.mat = i;
			it.split = s;
			it.slot = slot + t * s;
			tile_origin<BN>(o, p, q, t, it.m0, it.n0);
			return true;
		}
		t -= n;
		slot += n * s;
	}
	return false;
}

}  // namespace glb
