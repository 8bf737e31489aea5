"""Chunks over the 4-bit cache whose keys and values differ by large powers of two, against what each row sees."""
import numpy as np
import pytest

from glint_amd import glint_hip as H
from tests import bounded_util as R
from tests import serve_util as S
from tests.gpu_util import torch_cuda
from tests.test_gpu_kv4 import bf16, gpu
from tests.test_gpu_kv4_chunk import bound, many
from tests.test_gpu_window import paged, values

pytestmark = pytest.mark.gpu

HEADS, G = 2, 2


class Chunk:
    """n tokens of which nq are new: positive queries, small keys, and so weights that are alike, and positive values,
    so that a row's output is as large as the sum of its parts and what is lost shows."""

    def __init__(self, n, nq, D, own, seed):
        rng = np.random.default_rng(seed)
        self.n, self.nq, self.D, self.own = n, nq, D, own
        self.planes, self.table, _ = paged(rng, [n], HEADS, D)
        self.planes[2] |= 0x88
        self.planes[1] *= np.float32(0.05)
        self.planes[3] *= np.float32(0.25)
        self.q = bf16(np.abs(rng.normal(0, 1, (nq, HEADS * G, D))) + 0.1)
        self.k, self.v = (rng.normal(0, 1, (nq, HEADS, D)).astype(np.float32) for _ in range(2))
        self.k, self.v = self.k * np.float32(0.05), (np.abs(self.v) + np.float32(0.1)) * np.float32(0.25)

    def place(self, j):
        return self.table[0, j // 64], slice(None), slice(None), j % 64

    def key(self, j, size):
        """Key j: `size` in every dimension; its score is some 10 of it (7 for 64 dimensions) away from the others'."""
        if self.own and j >= self.n - self.nq:
            self.k[j - self.n + self.nq] = size
        else:
            page, _, _, t = self.place(j)
            self.planes[0][page, :, t] = 0xFF if size > 0 else 0  # PARENT's ends are -1 and 1
            self.planes[1][self.place(j)] = abs(size)

    def times(self, which, j, by):
        """Key or value j times a power of two."""
        if self.own and j >= self.n - self.nq:
            (self.k, self.v)[which][j - self.n + self.nq] *= np.float32(by)
        else:
            self.planes[2 * which + 1][self.place(j)] *= np.float32(by)

    def run(self, window=0, sinks=0):
        self.at = bf16(self.k), bf16(self.v)
        wide, max_q = many(self.table, self.nq)
        k, v = self.at if self.own else (None, None)
        self.got = values(H.kv4_attend_chunk(
            self.q, tuple(gpu(p) for p in self.planes), gpu(wide), gpu(np.array([self.n], np.int32)), max_q=max_q,
            cu_q=gpu(np.array([0, self.nq], np.int32)), k=k, v=v, window=window or None, sinks=sinks))

    def check(self, leave=(), rows=slice(None), window=0, sinks=0):
        """Rows against what they see, without the positions `leave`: those have no weight there that counts, and no
        part in what the others' roundings may add up to."""
        j = np.arange(self.n)
        k, v = S.held(self.planes, self.table[0][j // 64].astype(np.int64) * 64 + j % 64)
        if self.own:
            k[self.n - self.nq:], v[self.n - self.nq:] = (values(x) for x in self.at)
        ok = R.seen(np.arange(self.nq) + self.n - self.nq, self.n, window, sinks) & ~np.isin(j, leave)
        q = values(self.q)
        for h in range(HEADS * G):
            z = R.attend(q[rows, h], k[:, h // G], v[:, h // G], ok[rows], self.D ** -0.5)
            with np.errstate(over="ignore"):  # a key past every bound of f32 scores: finite is all that is asked
                worst = R.far(self.got[rows, h], *z, bound(self.own))
            assert worst <= 0, (h, worst)


@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("power", [8, 18, 26, 36, 60])
def test_a_large_value_that_weighs_nothing(power, D, own):
    """A first token (of the cache's, or of the chunk's own) whose value is 2^power times the others'; its weight and those of
    its tile's others are below 2^-100. Every row's output is what the other tiles give, where one token weighs 2^7 to 2^10
    times what each of many does."""
    torch_cuda()
    print(f"power={power} D={D} own={own}", flush=True)
    for n, nq in ((500, 70), (3000, 150)):
        c = Chunk(n, nq, D, own, power + D)
        j = n - nq if own else 0
        for i in range(j, j + 64):
            c.key(i, -30.0)
        c.times(1, j, 2.0 ** power)
        c.key(100, 0.7)
        c.run()
        c.check(range(j, j + 64))


@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("power", [14, 27, 36, 100])
def test_a_later_token_takes_nothing_from_earlier_rows(power, D, own):
    """A key or value of 2^power times the others' in the middle of the chunk: rows before it do not see it, however near
    their own tokens lie to it. Rows from it on hold what it gives them."""
    torch_cuda()
    for n, nq in ((300, 100), (3000, 100)):
        for which in (0, 1):
            print(f"power={power} D={D} own={own} n={n} which={which}", flush=True)
            c = Chunk(n, nq, D, own, power + D + which)
            j = n - nq + 37
            c.times(which, j, 2.0 ** power)
            c.key(100, 0.7)
            c.run()
            c.check(rows=slice(0, 37))
            c.check(rows=slice(37, nq))


@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("power", [14, 26, 100])
def test_one_large_value_beside_others(power, D, own):
    """As above for a value that every row sees and that weighs nothing: the tokens of its own tile keep theirs. A power of 100
    also leaves the tiles behind it more than f32 could carry an output up by."""
    torch_cuda()
    for n, nq, window, sinks in ((500, 70, 0, 0), (3000, 150, 0, 0), (900, 200, 400, 70)):
        print(f"power={power} D={D} own={own} n={n} window={window}", flush=True)
        c = Chunk(n, nq, D, own, power + n)
        j = n - nq if own else 20 if sinks else 0
        c.key(j, -30.0)
        c.times(1, j, 2.0 ** power)
        c.key(50, 0.7)
        c.run(window, sinks)
        c.check([j], window=window, sinks=sinks)


@pytest.mark.parametrize("own", [False, True])
def test_blocks_of_unlike_size(own):
    """128 dimensions whose first 64 are 2^40 times the others', where the queries hold nothing there; values likewise."""
    torch_cuda()
    c = Chunk(400, 90, 128, own, 3)
    c.q[..., :64] = 0
    c.planes[1][:, :, 0] *= np.float32(2.0 ** 40)
    c.planes[3][:, :, 1] *= np.float32(2.0 ** -40)
    c.k[..., :64] *= np.float32(2.0 ** 40)
    c.v[..., 64:] *= np.float32(2.0 ** -40)
    c.run()
    c.check()


@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("power", [-60, -34, 30, 41, 90])
def test_values_far_from_one(power, own):
    """All values 2^power, but for a tile of zeros and one of ordinary size with no weight."""
    torch_cuda()
    for D, n, nq in ((64, 500, 100), (128, 3000, 40)):
        c = Chunk(n, nq, D, own, 1000 + power)
        c.planes[3] *= np.float32(2.0 ** power)
        c.v *= np.float32(2.0 ** power)
        for j in range(64, 128):
            c.planes[3][c.place(j)] = 0
        for j in range(192, 256):
            c.times(1, j, 2.0 ** -power)
            c.key(j, -30.0)
        c.run()
        c.check(range(192, 256))


@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("D", [64, 128])
def test_the_largest_values(D, own):
    """Sums of some 500 weights times 2^116: in f32 as long as no weight counts as more than 1."""
    torch_cuda()
    c = Chunk(500, 100, D, own, 77)
    c.planes[3] *= np.float32(2.0 ** 116)
    c.v *= np.float32(2.0 ** 116)
    c.run()
    c.check()
