"""The paged cache and its operators: pages (``kv_*``), norm + rotation + append (``map_qk_norm_rope_kv_dev``) and attention
(``map_attn_kv_dev``), against the 64-bit forms of kv_oracle.py."""
import numpy as np
import pytest

import adam_b200 as A
from tests import kv_oracle as ko

pytestmark = pytest.mark.gpu
ACT, WT = 41, 42
U = 2.0 ** -24                                     # half a step of float32
HALF = {"f16": np.float16, "f32": np.float32}


class Cache:
    """A cache of the library and what its sequences should hold: per sequence [positions][n_layer, 2, heads, dim]."""

    def __init__(self, gpu, layers, kv_heads, dim, page, seqs, max_pages, n_pages, dtype):
        self.gpu, self.page, self.dtype, self.shape = gpu, page, HALF[dtype], (layers, 2, kv_heads, dim)
        self.id = gpu.kv_create(layers, kv_heads, dim, n_pages, seqs, max_pages, page, dtype)
        self.handles = []

    def pool(self):
        import torch
        self.gpu.sync()
        return torch.as_tensor(self.gpu.kv_array(self.id, "pool"), device="cuda")

    def fill(self, rng, lens, poison=False):
        """Sequences 0 .. grown in turns to ``lens`` with random contents; everything else NaN with ``poison``."""
        import torch
        left = np.array(lens)
        while left.any():
            who = np.flatnonzero(left)
            n = np.minimum(left[who], self.page)
            self.gpu.kv_extend(self.id, who, n)
            left[who] -= n
        pool, table = self.pool(), self.gpu.kv_table(self.id)
        if poison:
            pool.fill_(float("nan"))
        self.held = []
        for s, n in enumerate(lens):
            x = rng.standard_normal((n,) + self.shape).astype(self.dtype)
            p = np.arange(n)
            pool[torch.from_numpy(table[s][p // self.page].astype(np.int64)).cuda(), :, :, :, torch.from_numpy(p % self.page).cuda()] = torch.from_numpy(x).cuda()
            self.held.append(x)
        torch.cuda.synchronize()

    def read(self, seq):
        n, pool, table = self.gpu.kv_lens(self.id)[seq], self.pool(), self.gpu.kv_table(self.id)[seq]
        p = np.arange(n)
        return pool.cpu().numpy()[table[p // self.page], :, :, :, p % self.page]

    def batch(self, seqs, starts):
        hs = [self.gpu.upload_dev(np.array(v, np.uint32))[0] for v in (seqs, starts)]
        self.handles += hs
        return hs

    def close(self):
        for h in self.handles:
            self.gpu.free_handle(h)
        self.gpu.kv_destroy(self.id)


def up(c, values):
    h = c.gpu.upload_dev(np.array(values, np.uint32))[0]
    c.handles.append(h)
    return h


# ---- pages -----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,layers,kv_heads,dim,page", [("f16", 3, 2, 64, 16), ("f32", 1, 1, 32, 7), ("f16", 2, 1, 256, 64), ("f32", 2, 3, 128, 1)])
def test_fork_extend_truncate_compact(gpu, dtype, layers, kv_heads, dim, page):
    rng = np.random.default_rng(page)
    lens = [3 * page + page // 2 + 1, page + 1, 2 * page]
    c = Cache(gpu, layers, kv_heads, dim, page, 12, 8, 40, dtype)
    c.fill(rng, lens + [0] * 9)
    want = [x.copy() for x in c.held]

    def agree():
        import torch
        table, lens_now = (torch.as_tensor(gpu.kv_array(c.id, k), device="cuda").cpu().numpy() for k in ("table", "lens"))
        assert np.array_equal(table, gpu.kv_table(c.id)) and np.array_equal(lens_now, gpu.kv_lens(c.id))
        for s, x in enumerate(want):
            got = c.read(s)
            assert len(got) >= len(x) and np.array_equal(got[:len(x)], x), s

    gpu.kv_fork(c.id, 0, [3, 4, 5, 6])
    gpu.kv_fork(c.id, 0, [7], page + 1)
    for s in (3, 4, 5, 6):
        want[s] = want[0]
    want[7] = want[0][:page + 1]
    agree()
    assert gpu.kv_free_pages(c.id) == 40 - sum(-(-n // page) for n in lens)
    gpu.kv_extend(c.id, [3, 0, 4, 7], [1, 1, page + 2, 1])                # copies of the shared last pages
    agree()
    # what a continuation writes behind the fork is nobody else's
    pool, table = c.pool(), gpu.kv_table(c.id)
    for s in (3, 0, 4):
        p = lens[0]
        pool[int(table[s, p // page]), :, :, :, p % page] = float(s + 1)
        want[s] = np.concatenate([want[s], np.full((1,) + c.shape, s + 1, c.dtype)])
    agree()
    gpu.kv_truncate(c.id, [0, 1, 5], [page, 0, 2])
    want[0], want[1], want[5] = want[0][:page], want[1][:0], want[5][:2]
    agree()
    live = gpu.kv_compact(c.id)
    agree()
    table = gpu.kv_table(c.id)
    assert live == 40 - gpu.kv_free_pages(c.id) == len(set(table[table >= 0].tolist())) and table.max() == live - 1
    assert gpu.kv_compact(c.id) == live
    gpu.kv_truncate(c.id, np.arange(12))
    assert gpu.kv_free_pages(c.id) == 40 and (gpu.kv_table(c.id) == -1).all()
    c.close()


def test_many_records_and_copies_in_one_call(gpu):
    """More changes than the parameters of one launch hold."""
    rng = np.random.default_rng(3)
    c = Cache(gpu, 1, 1, 32, 3, 1300, 4, 4000, "f16")
    c.fill(rng, [5] + [0] * 1299)
    others = np.arange(1, 1300)
    gpu.kv_fork(c.id, 0, others)
    gpu.kv_extend(c.id, others, rng.integers(1, 4, 1299))
    pool, table = c.pool().cpu().numpy(), gpu.kv_table(c.id)
    assert len(set(table[:, 1].tolist())) == 1300 and (table[:, 0] == 0).all()
    assert (pool[table[1:, 1], :, :, :, :2] == pool[table[0, 1], :, :, :, :2]).all()
    gpu.kv_truncate(c.id, others[::2])
    assert gpu.kv_compact(c.id) == 4000 - gpu.kv_free_pages(c.id)
    for s in (0, 2, 600, 1298):
        assert np.array_equal(c.read(s)[:5], c.held[0])
    c.close()


def test_page_refusals(gpu):
    for bad in (dict(head_dim=48), dict(kv_heads=0), dict(n_pages=0), dict(page=1025), dict(seqs=0), dict(max_pages=1 << 31)):
        k = dict(layers=1, kv_heads=1, head_dim=32, page=4, seqs=2, max_pages=3, n_pages=4)
        k.update(bad)
        with pytest.raises(RuntimeError, match="code -3"):
            gpu.kv_create(k["layers"], k["kv_heads"], k["head_dim"], k["n_pages"], k["seqs"], k["max_pages"], k["page"])
    with pytest.raises(RuntimeError, match="code -2"):
        gpu.kv_create(64, 16, 256, 1 << 27, 1, 1, 64, "f32")
    with pytest.raises(ValueError):
        gpu.kv_create(1, 1, 32, 4, 2, 3, kv_dtype="bf16")
    c = Cache(gpu, 1, 1, 32, 4, 2, 3, 4, "f32")
    gpu.kv_extend(c.id, [0], 9)
    for call, code in [(lambda: gpu.kv_extend(c.id, [0], 4), -3), (lambda: gpu.kv_extend(c.id, [1], 5), -2), (lambda: gpu.kv_extend(c.id, [1, 1], 1), -3),
                       (lambda: gpu.kv_fork(c.id, 0, [0]), -3), (lambda: gpu.kv_truncate(c.id, [1], 1), -3), (lambda: gpu.kv_extend(63, [0], 1), -4),
                       (lambda: gpu.kv_compact(77), -4)]:
        with pytest.raises(RuntimeError, match=f"code {code}"):
            call()
    with pytest.raises(ValueError):
        gpu.kv_extend(c.id, [0, 1], [1, 2, 3])
    gpu.capture_begin()
    for call in (lambda: gpu.kv_extend(c.id, [0], 1), lambda: gpu.kv_compact(c.id), lambda: gpu.kv_destroy(c.id), lambda: gpu.kv_create(1, 1, 32, 4, 2, 3)):
        with pytest.raises(RuntimeError, match="captured"):
            call()
    gpu.graph_destroy(gpu.capture_end())
    assert gpu.kv_lens(c.id).tolist() == [9, 0] and gpu.kv_free_pages(c.id) == 1
    c.close()


def test_pages_stay_while_the_owner_of_a_lent_stream_captures(gpu):
    """Another program's capture of the stream that the library works on: operators are recorded, page calls are refused."""
    import torch
    rng = np.random.default_rng(31)
    heads, KV, D = 4, 2, 64
    c = Cache(gpu, 1, KV, D, 8, 3, 10, 12, "f16")
    c.fill(rng, [30, 0, 0])
    gpu.map_create_typed(ACT, A.DTYPE_F32, 1, 2 * heads * D)
    q_h, o_h, (seq, start) = up(c, [0]), up(c, [heads * D]), c.batch([0], [0, 1])
    act = torch.as_tensor(gpu.map_array(ACT), device="cuda")
    st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    gpu.set_stream(st.cuda_stream)
    gpu.batch_begin()
    try:
        with torch.cuda.graph(graph, stream=st):
            gpu.map_attn_kv_dev(ACT, c.id, 0, q_h, o_h, seq, start, 1, 1, heads, scale=D ** -0.5)
            for call in (lambda: gpu.kv_extend(c.id, [0], 1), lambda: gpu.kv_fork(c.id, 0, [1], 30), lambda: gpu.kv_truncate(c.id, [0], 3),
                         lambda: gpu.kv_compact(c.id), lambda: gpu.kv_create(1, 1, 32, 4, 2, 3), lambda: gpu.kv_destroy(c.id)):
                with pytest.raises(RuntimeError, match="captured"):
                    call()
        assert gpu.kv_lens(c.id).tolist() == [30, 0, 0] and gpu.kv_free_pages(c.id) == 8
        q = torch.from_numpy(rng.standard_normal(heads * D).astype(np.float32)).cuda()
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            act[:heads * D] = q
            graph.replay()
            gpu.kv_fork(c.id, 0, [1])                              # and are as ever afterwards
        torch.cuda.synchronize()
    finally:
        gpu.batch_end()
        gpu.set_stream(0)
    assert gpu.kv_lens(c.id).tolist() == [30, 30, 0]
    want, most = ko.attend(q.view(heads, D).cpu().numpy(), c.held[0][:, 0, 0], c.held[0][:, 0, 1], 29, 0, 0, D ** -0.5, 0.0)
    near(act[heads * D:].view(heads, D).cpu().numpy(), want, most)
    c.close()


# ---- norm + rotation + append ------------------------------------------------------------------------------------------

SHAPES = [(4, 1, 256), (32, 16, 128), (14, 2, 64), (9, 3, 32), (5, 5, 64), (3, 1, 128), (10, 2, 256)]


def append(gpu, c, rng, seqs, new, heads, layer, norm=(True, True), in_place=False, skew=0, base=1e6, eps=1e-6, pads=(0, 0)):
    """Rows of the batch through the operator: (map contents before and after, offsets of q, k, v, q_dst, weights).  ``pads``:
    rows ahead of the first entry and behind the last; ``skew``: how far the offsets are off four values."""
    _, _, KV, D = c.shape
    n, (ahead, behind) = sum(new), pads
    rows = ahead + n + behind
    starts = ahead + np.cumsum([0] + list(new))
    oq = skew + np.arange(rows) * (heads * D + 3 * skew)
    ok = oq[-1] + heads * D + np.arange(rows) * (KV * D + skew)
    ov = ok[-1] + KV * D + rng.permutation(rows) * KV * D
    od = oq if in_place else ov.max() + KV * D + skew + np.arange(rows) * heads * D
    end = int(max(od.max() + heads * D, ov.max() + KV * D))
    gpu.map_create_typed(ACT, A.DTYPE_F32, 1, end)
    gpu.map_create_typed(WT, A.DTYPE_F32, 1, 2 * D + skew)
    act, wt = (rng.standard_normal(end) * 3).astype(np.float32), (1 + 0.1 * rng.standard_normal(2 * D + skew)).astype(np.float32)
    gpu.scatter_contiguous(ACT, 0, act)
    gpu.scatter_contiguous(WT, 0, wt)
    hs = [up(c, o) for o in (oq, ok, ov)]
    w = [up(c, [skew]) if norm[0] else 0, up(c, [skew + D]) if norm[1] else 0]
    gpu.map_qk_norm_rope_kv_dev(ACT, WT, c.id, layer, *hs, *w, up(c, od), *c.batch(seqs, starts), len(seqs), rows, heads, base, eps)
    got = gpu.gather(ACT, np.arange(end, dtype=np.uint32)).view(np.float32)
    return act, got, (oq, ok, ov, od), (wt[skew:skew + D] if norm[0] else None, wt[skew + D:skew + 2 * D] if norm[1] else None), starts


@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("kind", ["token", "ragged", "skewed", "plain", "in_place"])
def test_append(gpu, heads, kv_heads, dim, dtype, kind):
    rng = np.random.default_rng(heads + dim)
    page = {"token": 64, "ragged": 16, "skewed": 7, "plain": 5, "in_place": 1}[kind]
    new = {"token": [1] * 5, "ragged": [37, 0, 1, 64], "skewed": [3, 9], "plain": [20], "in_place": [2, 1, 3]}[kind]
    seqs, ctx = [3, 0, 4, 1, 2][:len(new)], [130, 0, 17, 900, 3]
    lens = [0] * 5
    for s, n, p in zip(seqs, new, ctx):
        lens[s] = n + p
    c = Cache(gpu, 2, kv_heads, dim, page, 5, -(-1000 // page), sum(-(-x // page) for x in lens) + 2, dtype)
    c.fill(rng, lens)
    norm = {"plain": (False, False), "in_place": (True, False)}.get(kind, (True, True))
    before, after, (oq, ok, ov, od), (qw, kw), starts = append(gpu, c, rng, seqs, new, heads, 1, norm, kind == "in_place", 1 if kind == "skewed" else 0,
                                                               pads=(2, 3) if kind == "ragged" else (0, 0))
    want_map = before.astype(np.float64)
    touched = np.zeros(len(before), bool)
    # Norm: ss of dim products and sums, its root, a quotient, the weight: (dim / 32 + 12) half-steps at most, as every lane
    # sums dim / 32 of them and the lanes meet in five steps.  Rotation: the sine and cosine of an angle known to 2^-24 of a
    # turn, 6.3 half-steps of 1 in all, and a product and a sum: 9 half-steps of the pair's length.
    tol = (dim / 32 + 24) * U
    for e, s in enumerate(seqs):
        got, held = c.read(s), c.held[s].astype(np.float64)
        for i in range(new[e]):
            r, pos = starts[e] + i, lens[s] - new[e] + i
            q, k, v = (before[o[r]:o[r] + h * dim].reshape(h, dim) for o, h in ((oq, heads), (ok, kv_heads), (ov, kv_heads)))
            y = ko.rotate_normed(q, qw, pos, 1e6, 1e-6)
            pair = np.hypot(y[:, :dim // 2], y[:, dim // 2:])
            at = slice(od[r], od[r] + heads * dim)
            assert (np.abs(after[at].reshape(heads, dim) - y) <= tol * np.concatenate([pair, pair], 1) + 1e-30).all()
            want_map[at], touched[at] = after[at], True
            y = ko.rotate_normed(k, kw, pos, 1e6, 1e-6)
            pair = np.hypot(y[:, :dim // 2], y[:, dim // 2:])
            half = 0 if dtype == "f32" else 2.0 ** -11
            assert (np.abs(got[pos, 1, 0] - y) <= tol * np.concatenate([pair, pair], 1) + half * (1 + tol) * np.abs(y) + 2.0 ** -25).all()
            assert np.array_equal(got[pos, 1, 1], v.astype(c.dtype))
            held[pos, 1] = got[pos, 1]
        assert np.array_equal(got, held.astype(c.dtype))         # nothing else in the cache changed
    assert np.array_equal(after, want_map.astype(np.float32))    # nor in the map
    assert gpu.device_error() == 0
    c.close()


def test_append_far_positions(gpu):
    """The rotation of a position of many turns (64-bit angles)."""
    rng = np.random.default_rng(5)
    c = Cache(gpu, 1, 1, 128, 1024, 1, 300, 300, "f32")
    gpu.kv_extend(c.id, [0], 300001)
    before, after, (oq, ok, _, od), (qw, kw), _ = append(gpu, c, rng, [0], [2], 2, 0, base=10000.0)
    for i, pos in enumerate((299999, 300000)):
        y = ko.rotate_normed(before[oq[i]:oq[i] + 256].reshape(2, 128), qw, pos, 10000.0, 1e-6)
        assert np.abs(after[od[i]:od[i] + 256].reshape(2, 128) - y).max() <= 30 * U * np.abs(y).max()
        got = c.pool()[int(gpu.kv_table(c.id)[0, pos // 1024]), 0, 0, 0, pos % 1024].cpu().numpy()
        y = ko.rotate_normed(before[ok[i]:ok[i] + 128].reshape(1, 128), kw, pos, 10000.0, 1e-6)[0]
        assert np.abs(got - y).max() <= 30 * U * np.abs(y).max()
    c.close()


@pytest.mark.parametrize("dim", [32, 64, 128, 256])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_append_rows_whose_squares_overflow_or_vanish(gpu, dtype, dim):
    """x / sqrt(mean(x^2) + eps) in 32 bits where the mean is infinite (0, and NaN for an infinite value), or 0 with eps = 0 (nothing
    finite)."""
    rng = np.random.default_rng(dim)
    H, KV, rows = 4, 2, 4
    c = Cache(gpu, 1, KV, dim, 8, 1, 1, 1, dtype)
    gpu.kv_extend(c.id, [0], rows)
    n, m = H * dim, KV * dim
    x = rng.standard_normal((rows, H + 2 * KV, dim)).astype(np.float32)
    x[0, :, :] *= np.float32(1e25)
    x[1, 0] *= np.float32(1e20)                                  # one head of the row; its neighbours are what they were
    x[1, H] *= np.float32(1e37)
    x[2, 1, 5], x[2, H + 1, dim - 1] = np.inf, -np.inf
    x[2, 2, 3], x[2, H, 1] = 3e38, -3e38
    x[3] *= np.float32(1e-30)
    x[:, H + KV:] = rng.standard_normal((rows, KV, dim))         # values: not normed
    w = (1 + 0.1 * rng.standard_normal((2, dim))).astype(np.float32)
    at = np.cumsum([0, rows * n, rows * m, rows * m, rows * n])
    gpu.map_create_typed(ACT, A.DTYPE_F32, 1, int(at[-1]) + 2 * dim)
    gpu.scatter_contiguous(ACT, 0, np.concatenate([x[:, :H].reshape(-1), x[:, H:H + KV].reshape(-1), x[:, H + KV:].reshape(-1)]))
    gpu.scatter_contiguous(ACT, int(at[-1]), w.reshape(-1))
    r = np.arange(rows)
    hs = [up(c, o + r * k) for o, k in zip(at, (n, m, m, n))]
    ws = up(c, [at[-1]]), up(c, [at[-1] + dim])
    for eps in (0.0, 1e-6):
        gpu.map_qk_norm_rope_kv_dev(ACT, ACT, c.id, 0, *hs[:3], *ws, hs[3], *c.batch([0], [0, rows]), 1, rows, H, 1e4, eps)
        got_q = gpu.gather(ACT, np.arange(at[3], at[4], dtype=np.uint32)).view(np.float32).reshape(rows, H, dim)
        got = c.read(0)
        with np.errstate(all="ignore"):
            for i in range(rows):
                for heads, out, wt in ((slice(0, H), got_q[i], w[0]), (slice(H, H + KV), got[i, 0, 0].astype(np.float32), w[1])):
                    v = x[i, heads]
                    y = v / np.sqrt((v * v).mean(-1, keepdims=True, dtype=np.float32) + np.float32(eps))
                    assert y.dtype == np.float32
                    want = ko.rotate_normed(y * wt, None, i, 1e4, 0.0)
                    fine = np.isfinite(want)
                    assert np.array_equal(np.isfinite(out), fine), (eps, i)
                    # as in test_append, and 2^-11 of the value in a 16-bit cache; the plain form's own norm adds dim / 32 + 12 half-steps
                    pair = np.hypot(want[:, :dim // 2], want[:, dim // 2:])
                    tol = (2 * (dim / 32 + 12) + 24) * U + (0 if dtype == "f32" or heads.start == 0 else 2.0 ** -11)
                    assert (np.abs(out - want)[fine] <= (tol * np.concatenate([pair, pair], 1) + 2.0 ** -25)[fine]).all()
        assert (got_q[0] == 0).all() and (got_q[1, 0] == 0).all() and (got[1, 0, 0, 0] == 0).all()
        assert np.array_equal(got[:, 0, 1], x[:, H + KV:].astype(c.dtype)) and gpu.device_error() == 0
    c.close()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_append_captured_while_sequences_grow(gpu, dtype):
    """Two graphs of one cache, each an append of two rows, replayed in turn at lengths, pages and values of their own time."""
    rng = np.random.default_rng(17)
    H, KV, D, page = 4, 2, 64, 5
    c = Cache(gpu, 2, KV, D, page, 2, 30, 60, dtype)
    c.fill(rng, [1, 7])
    n, m = H * D, KV * D
    at = np.cumsum([0, 4 * n, 4 * m, 4 * m, 4 * n, D, D])            # q, k, v, results of both graphs' rows; weights
    gpu.map_create_typed(ACT, A.DTYPE_F32, 1, int(at[-1]))
    w = (1 + 0.1 * rng.standard_normal((2, D))).astype(np.float32)
    ws = up(c, [at[4]]), up(c, [at[5]])
    graphs = []
    for g in range(2):                                            # graph g: the last two positions of sequence g
        hs = [up(c, o + (2 * g + np.arange(2)) * k) for o, k in zip(at, (n, m, m, n))]
        batch = c.batch([g], [0, 2])
        gpu.capture_begin()
        gpu.map_qk_norm_rope_kv_dev(ACT, ACT, c.id, 1, *hs[:3], *ws, hs[3], *batch, 1, 2, H, 1e4, 1e-6)
        graphs.append(gpu.capture_end())
    tol = (D / 32 + 24) * U                                          # as in test_append
    for step in range(3):
        for s, grow in enumerate((2 + 11 * step, 2 + 3 * step)):
            gpu.kv_extend(c.id, [s], grow)
        held, lens = [c.read(s) for s in range(2)], gpu.kv_lens(c.id)
        x = (rng.standard_normal(4 * (2 * n + 2 * m)) * 3).astype(np.float32)
        gpu.scatter_contiguous(ACT, 0, np.concatenate([x, w.reshape(-1)]))
        for g in graphs:
            gpu.graph_launch(g)
        after = gpu.gather(ACT, np.arange(at[4], dtype=np.uint32)).view(np.float32)
        for s in range(2):
            got = c.read(s)
            for i in range(2):
                r, pos = 2 * s + i, int(lens[s]) - 2 + i
                q, k, v = (x[at[j] + r * z:at[j] + (r + 1) * z].reshape(-1, D) for j, z in ((0, n), (1, m), (2, m)))
                for y, out, half in ((ko.rotate_normed(q, w[0], pos, 1e4, 1e-6), after[at[3] + r * n:at[3] + (r + 1) * n].reshape(H, D), 0.0),
                                     (ko.rotate_normed(k, w[1], pos, 1e4, 1e-6), got[pos, 1, 0], 0.0 if dtype == "f32" else 2.0 ** -11)):
                    pair = np.hypot(y[:, :D // 2], y[:, D // 2:])
                    assert (np.abs(out - y) <= tol * np.concatenate([pair, pair], 1) + half * (1 + tol) * np.abs(y) + 2.0 ** -25).all()
                assert np.array_equal(got[pos, 1, 1], v.astype(c.dtype))
                held[s][pos, 1] = got[pos, 1]
            assert np.array_equal(got, held[s])
    for g in graphs:
        gpu.graph_destroy(g)
    assert gpu.device_error() == 0
    c.close()


def test_append_leaves_out_what_it_may_not_write(gpu):
    """Padding entries, unknown sequences, positions that the sequence does not have or shares with another."""
    rng = np.random.default_rng(6)
    c = Cache(gpu, 1, 1, 32, 4, 6, 8, 20, "f32")
    c.fill(rng, [6, 5, 3, 0, 0, 0])
    gpu.kv_fork(c.id, 0, [3])
    gpu.kv_extend(c.id, [0], [1])
    held = [c.read(s) for s in range(4)]
    # sequence 0: rows for positions 5 (shared) and 6 (its own); 1: six rows of five positions; no sequence; one past the cache's
    before, after, (oq, ok, ov, od), _, starts = append(gpu, c, rng, [0, 1, A.KV_NO_SEQ, 9], [2, 6, 1, 1], 2, 0)
    assert gpu.device_error() == 1
    assert np.array_equal(c.read(3), held[3]) and np.array_equal(c.read(2), held[2]) and np.array_equal(c.read(0)[:6], held[0][:6])
    assert not np.array_equal(c.read(0)[6], held[0][6]) and not np.array_equal(c.read(1), held[1])
    for r, written in enumerate([False, True, False] + [True] * 5 + [False, False]):
        at = slice(od[r], od[r] + 64)
        assert np.array_equal(after[at], before[at]) != written, r
    # offsets outside the maps
    gpu.kv_extend(c.id, [1], [2])
    n = len(before)
    rows = [up(c, v) for v in ([0, n - 63], [0, 0], [0, 0], [64, 128])]
    gpu.map_qk_norm_rope_kv_dev(ACT, WT, c.id, 0, *rows[:3], up(c, [0]), up(c, [33]), rows[3], *c.batch([1], [0, 2]), 1, 2, 2)
    assert gpu.device_error() == 1
    c.close()


def test_operator_refusals(gpu):
    c = Cache(gpu, 2, 2, 32, 4, 3, 4, 8, "f16")
    gpu.map_create_typed(ACT, A.DTYPE_F32, 1, 1000)
    gpu.map_create_typed(WT, A.DTYPE_F32, 2, 100)
    h, w, (seq, start) = up(c, [0, 64]), up(c, [0]), c.batch([0], [0, 2])
    ok = dict(m=ACT, wt=ACT, kv=c.id, layer=1, h=h, w=w, seq=seq, start=start, n_seqs=1, n_rows=2, heads=4, base=1e4, eps=1e-6, window=0, scale=1.0, cap=0.0)
    for bad, code in [(dict(m=250), -4), (dict(m=WT), -3), (dict(kv=63), -4), (dict(layer=2), -3), (dict(heads=3), -3), (dict(heads=0), -3), (dict(n_rows=3), -4),
                      (dict(n_seqs=4), -3), (dict(n_seqs=2), -4), (dict(seq=0), -4), (dict(start=60000), -4), (dict(h=0), -4), (dict(n_rows=(1 << 24) + 1), -3)]:
        k = dict(ok, **bad)
        with pytest.raises(RuntimeError, match=f"code {code}"):
            gpu.map_attn_kv_dev(k["m"], k["kv"], k["layer"], k["h"], k["h"], k["seq"], k["start"], k["n_seqs"], k["n_rows"], k["heads"])
        with pytest.raises(RuntimeError, match=f"code {code}"):
            gpu.map_qk_norm_rope_kv_dev(k["m"], k["wt"], k["kv"], k["layer"], *[k["h"]] * 3, k["w"], k["w"], k["h"], k["seq"], k["start"], k["n_seqs"], k["n_rows"], k["heads"])
    for bad in (dict(scale=np.inf), dict(scale=np.nan), dict(cap=-1.0), dict(cap=np.inf), dict(cap=np.nan)):
        with pytest.raises(RuntimeError, match="code -3"):
            gpu.map_attn_kv_dev(ACT, c.id, 1, h, h, seq, start, 1, 2, 4, **bad)
    for bad in (dict(freq_base=0.0), dict(freq_base=np.inf), dict(freq_base=np.nan), dict(eps=-1.0), dict(eps=np.nan)):
        with pytest.raises(RuntimeError, match="code -3"):
            gpu.map_qk_norm_rope_kv_dev(ACT, ACT, c.id, 1, h, h, h, w, w, h, seq, start, 1, 2, 4, **bad)
    with pytest.raises(RuntimeError, match="code -3"):
        gpu.map_qk_norm_rope_kv_dev(ACT, WT, c.id, 1, h, h, h, w, w, h, seq, start, 1, 2, 4)
    gpu.map_attn_kv_dev(ACT, c.id, 1, h, h, seq, start, 0, 2, 4)
    gpu.map_attn_kv_dev(ACT, c.id, 1, h, h, seq, start, 1, 0, 4)
    assert gpu.device_error() == 0
    c.close()


# ---- attention ---------------------------------------------------------------------------------------------------------

def attention(gpu, c, seqs, starts, rows, heads, q, layer=1, window=0, n_sink=0, scale=None, cap=0.0, oq=None, oo=None, n_rows=None):
    """q [rows, heads, dim] through the operator; results likewise (what no row wrote is -7)."""
    D = c.shape[3]
    oq = np.arange(rows) * heads * D if oq is None else oq
    base = int(oq.max()) + heads * D
    oo = base + np.arange(rows) * heads * D if oo is None else oo
    end = int(oo.max()) + heads * D
    gpu.map_create_typed(ACT, A.DTYPE_F32, 1, end)
    data = np.full(end, -7, np.float32)
    for r in range(rows):
        data[oq[r]:oq[r] + heads * D] = q[r].reshape(-1)
    gpu.scatter_contiguous(ACT, 0, data)
    gpu.map_attn_kv_dev(ACT, c.id, layer, up(c, oq), up(c, oo), *c.batch(seqs, starts), len(seqs), rows if n_rows is None else n_rows, heads, window, n_sink,
                        D ** -0.5 if scale is None else scale, cap)
    got = gpu.gather(ACT, np.arange(end, dtype=np.uint32)).view(np.float32)
    return np.stack([got[o:o + heads * D].reshape(heads, D) for o in oo])


def near(got, want, most):
    """A score is off by a few half-steps of the largest one in the row (sums of head_dim products in 22 to 24 bits), a weight
    by that much of itself, and so is the weighted sum; sums of weights and values add a few half-steps of their own:
    8 (1 + largest score) half-steps in the mean over all outputs, and 16 times that for a single one."""
    tol = 8 * U * (1 + most)
    d, norm = got.astype(np.float64) - want, np.sqrt((want ** 2).mean())
    assert np.sqrt((d ** 2).mean()) <= tol * norm, (np.sqrt((d ** 2).mean()) / norm, tol)
    assert (np.abs(d) <= 16 * tol * np.maximum(norm, np.abs(want))).all()


def expect(c, lens, seqs, starts, q, heads, layer, window, n_sink, scale, cap):
    want, most, rows = [], 0.0, []
    for e, s in enumerate(seqs):
        n = starts[e + 1] - starts[e]
        for i in range(n):
            o, m = ko.attend(q[starts[e] + i], c.held[s][:, layer, 0], c.held[s][:, layer, 1], lens[s] - n + i, window, n_sink, scale, cap)
            want.append(o)
            most = max(most, m)
            rows.append(starts[e] + i)
    return rows, np.stack(want), most


CASES = {
    # new rows and earlier positions per sequence, page, window, sinks, cap
    "token": ([1, 1, 1], [130, 0, 63], 64, 0, 0, 0.0),
    "token_long": ([1], [3001], 16, 0, 0, 50.0),
    "chunk": ([70, 1, 33], [200, 64, 0], 64, 0, 0, 0.0),
    "ragged": ([5, 0, 130, 2], [7, 9, 300, 1], 7, 0, 0, 50.0),
    "window": ([3, 90], [500, 260], 48, 100, 0, 0.0),
    "window_sinks": ([1, 90, 200], [700, 40, 333], 16, 64, 5, 50.0),
    "window_one": ([4], [90], 5, 1, 0, 0.0),
    "sinks_beyond_window": ([40], [300], 64, 30, 200, 0.0),
    "wide_window": ([20], [20], 1, 1000, 3, 0.0),
    "many": ([1] * 40, [11 * i for i in range(40)], 64, 0, 0, 0.0),
}


@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("kind", list(CASES))
def test_attention(gpu, heads, kv_heads, dim, dtype, kind):
    new, ctx, page, window, n_sink, cap = CASES[kind]
    rng = np.random.default_rng(dim + len(kind))
    S = len(new)
    lens = [n + p for n, p in zip(new, ctx)]
    c = Cache(gpu, 2, kv_heads, dim, page, S, max(-(-x // page) for x in lens), sum(-(-x // page) for x in lens) + 1, dtype)
    c.fill(rng, lens, poison=True)                               # whatever no sequence holds is NaN
    seqs = rng.permutation(S).tolist()
    starts = np.cumsum([0] + [new[s] for s in seqs])
    q = (rng.standard_normal((starts[-1], heads, dim)) * 2.5).astype(np.float32)
    got = attention(gpu, c, seqs, starts, int(starts[-1]), heads, q, 1, window, n_sink, cap=cap)
    rows, want, most = expect(c, lens, seqs, starts, q, heads, 1, window, n_sink, dim ** -0.5, cap)
    near(got[rows], want, most)
    assert gpu.device_error() == 0
    c.close()


WIDE = [
    # what is chosen by how much there is: type, dims, query heads of a key head, page, new rows and earlier positions, window, sinks, cap
    ("f16", 64, 2, 16, [140, 1, 60], [900, 400, 1000], 0, 0, 0.0),
    ("f16", 64, 3, 12, [140, 1, 60], [900, 400, 1000], 0, 0, 50.0),
    ("f16", 128, 2, 64, [400, 33], [300, 900], 250, 5, 50.0),
    ("f16", 128, 1, 12, [400, 33], [300, 900], 250, 5, 0.0),
    ("f16", 128, 4, 8, [129, 128, 127], [1100, 0, 555], 0, 0, 0.0),
    ("f16", 256, 2, 64, [150], [1000], 0, 0, 50.0),
    ("f16", 256, 8, 64, [250], [1300], 0, 0, 0.0),
    ("f32", 128, 2, 64, [150, 20], [1000, 3], 0, 0, 0.0),
    ("f32", 128, 8, 16, [250], [1300], 0, 0, 50.0),
    ("f32", 256, 8, 64, [250], [1300], 0, 0, 0.0),
    ("f32", 256, 2, 5, [150], [1000], 0, 0, 0.0),
    ("f32", 64, 2, 16, [140, 1, 60], [900, 400, 1000], 64, 70, 0.0),
    ("f16", 32, 2, 16, [140, 1, 60], [900, 400, 1000], 100, 0, 0.0),
    ("f16", 32, 2, 16, [340, 1, 60], [900, 400, 1000], 0, 0, 0.0),
    ("f32", 32, 2, 16, [340, 1, 60], [900, 400, 1000], 0, 0, 50.0),
    ("f32", 64, 4, 16, [340, 1, 60], [900, 400, 1000], 0, 0, 50.0),
]


@pytest.mark.parametrize("dtype,dim,group,page,new,ctx,window,n_sink,cap", WIDE)
def test_attention_of_much(gpu, dtype, dim, group, page, new, ctx, window, n_sink, cap):
    rng = np.random.default_rng(dim + page)
    lens = [n + p for n, p in zip(new, ctx)]
    heads = 8 * group
    c = Cache(gpu, 1, 8, dim, page, len(new), max(-(-x // page) for x in lens), sum(-(-x // page) for x in lens) + 1, dtype)
    c.fill(rng, lens, poison=True)
    starts = np.cumsum([0] + new)
    q = (rng.standard_normal((starts[-1], heads, dim)) * 2.5).astype(np.float32)
    got = attention(gpu, c, list(range(len(new))), starts, int(starts[-1]), heads, q, 0, window, n_sink, cap=cap)
    assert np.isfinite(got).all()
    want, rows, most = [], [], 0.0
    for s, n in enumerate(new):
        for i in sorted({*range(0, n, 11), n - 1}):
            o, m = ko.attend(q[starts[s] + i], c.held[s][:, 0, 0], c.held[s][:, 0, 1], ctx[s] + i, window, n_sink, dim ** -0.5, cap)
            want.append(o), rows.append(starts[s] + i)
            most = max(most, m)
    near(got[rows], np.stack(want), most)
    assert gpu.device_error() == 0
    c.close()


@pytest.mark.parametrize("dtype,dim,rows", [("f16", 64, 1), ("f32", 64, 2), ("f16", 128, 7), ("f16", 64, 40), ("f32", 128, 40), ("f16", 256, 3)])
def test_attention_of_many_sequences(gpu, dtype, dim, rows):
    """More sequences than a CTA has threads, in any order, some without rows, some that are none."""
    rng = np.random.default_rng(dim + rows)
    S = 700
    new = [(i * 5 + 1) % (rows + 1) if i % 9 else 0 for i in range(S)] if rows > 1 else [1] * S
    lens = [n + (37 * i) % 190 for i, n in enumerate(new)]
    c = Cache(gpu, 1, 2, dim, 16, S, 16, sum(-(-x // 16) for x in lens) + 1, dtype)
    c.fill(rng, lens, poison=True)
    order = rng.permutation(S).tolist()
    starts = np.cumsum([0] + [new[s] for s in order])
    seqs = [A.KV_NO_SEQ if i % 50 == 7 else s for i, s in enumerate(order)]
    q = rng.standard_normal((starts[-1], 4, dim)).astype(np.float32)
    got = attention(gpu, c, seqs, starts, int(starts[-1]), 4, q, 0, 100, 3)
    want, at, most = [], [], 0.0
    for e, s in enumerate(seqs):
        n = starts[e + 1] - starts[e]
        if s == A.KV_NO_SEQ:
            assert (got[starts[e]:starts[e + 1]] == -7).all()
            continue
        for i in sorted({0, n - 1} if n else {}):
            o, m = ko.attend(q[starts[e] + i], c.held[s][:, 0, 0], c.held[s][:, 0, 1], lens[s] - n + i, 100, 3, dim ** -0.5, 0.0)
            want.append(o), at.append(starts[e] + i)
            most = max(most, m)
    near(got[at], np.stack(want), most)
    assert gpu.device_error() == 0
    c.close()


@pytest.mark.parametrize("dtype,dim,page", [("f16", 64, 12), ("f16", 128, 16), ("f32", 128, 16), ("f16", 256, 64)])
def test_attention_of_much_with_infinite_and_nan_values(gpu, dtype, dim, page):
    rng = np.random.default_rng(dim)
    n, new, window = 1200, 150, 900
    c = Cache(gpu, 1, 8, dim, page, 1, n // page + 1, n // page + 1, dtype)
    c.fill(rng, [n], poison=True)
    pool, table = c.pool(), gpu.kv_table(c.id)[0]
    for p, which, value in [(n - 1, 0, np.nan), (n - 1, 1, np.inf), (n - 4, 1, -np.inf), (60, 0, np.inf), (61, 1, np.nan), (n - new - window, 1, np.inf)]:
        c.held[0][p, 0, which, 0, 3] = value
        pool[int(table[p // page]), 0, which, 0, p % page, 3] = float(value)
    q = rng.standard_normal((new, 16, dim)).astype(np.float32)
    got = attention(gpu, c, [0], [0, new], new, 16, q, layer=0, window=window)
    rows = [*range(0, new - 8, 13), *range(new - 8, new)]
    with np.errstate(all="ignore"):
        want = np.stack([ko.attend(q[r], c.held[0][:, 0, 0], c.held[0][:, 0, 1], n - new + r, window, 0, dim ** -0.5, 0.0)[0] for r in rows])
    got, fine = got[rows], np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[np.isinf(want)], want[np.isinf(want)].astype(np.float32))
    assert (np.abs(got[fine] - want[fine]) <= 1e-4).all()
    c.close()


def test_attention_rows_anywhere(gpu):
    """Unaligned and permuted rows, results in the queries' place, rows outside every entry, padding entries."""
    rng = np.random.default_rng(9)
    heads, dim, lens = 6, 64, [100, 37, 5]
    c = Cache(gpu, 2, 2, dim, 16, 3, 8, 20, "f16")
    c.fill(rng, lens, poison=True)
    seqs, starts, rows = [2, A.KV_NO_SEQ, 0], [1, 3, 5, 40], 43
    q = rng.standard_normal((rows, heads, dim)).astype(np.float32)
    oq = 3 + rng.permutation(rows) * (heads * dim + 1)
    live = [0, 2]
    for oo in (None, oq):
        got = attention(gpu, c, seqs, starts, rows, heads, q, oq=oq, oo=oo)
        used = [(2, 1, 2), (0, 5, 35)]
        for s, first, n in used:
            for i in range(n):
                want, most = ko.attend(q[first + i], c.held[s][:, 1, 0], c.held[s][:, 1, 1], lens[s] - n + i, 0, 0, dim ** -0.5, 0.0)
                near(got[first + i], want, most)
        rest = [r for r in range(rows) if not (1 <= r < 3 or 5 <= r < 40)]
        assert np.array_equal(got[rest], q[rest] if oo is not None else np.full_like(q[rest], -7))
    assert live and gpu.device_error() == 0
    c.close()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("new", [1, 6, 150])
def test_attention_infinite_and_nan_values(gpu, dtype, new):
    """What a row does not see does not reach it: infinities and NaN in the keys and values of later positions and behind the
    window.  What it sees does."""
    rng = np.random.default_rng(new)
    heads, dim, n = 4, 64, 300
    c = Cache(gpu, 1, 1, dim, 16, 1, 20, 20, dtype)
    c.fill(rng, [n], poison=True)
    pool, table = c.pool(), gpu.kv_table(c.id)[0]
    window = 40
    for p, which, value in [(n - 1, 0, np.nan), (n - 1, 1, np.inf), (n - 4, 1, -np.inf), (60, 0, np.inf), (61, 1, np.nan), (n - new - window, 1, np.inf)]:
        c.held[0][p, 0, which, 0, 3] = value
        pool[int(table[p // 16]), 0, which, 0, p % 16, 3] = float(value)
    q = rng.standard_normal((new, heads, dim)).astype(np.float32)
    got = attention(gpu, c, [0], [0, new], new, heads, q, layer=0, window=window)
    with np.errstate(all="ignore"):
        rows, want, _ = expect(c, [n], [0], [0, new], q, heads, 0, window, 0, dim ** -0.5, 0.0)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[np.isinf(want)], want[np.isinf(want)].astype(np.float32))
    assert (np.abs(got[fine] - want[fine]) <= 1e-4).all()
    c.close()


# type, dims, query heads of a key head, key heads, page, new rows and all positions: tiles of 2 and 4, of 16, of 32 and 64, of 128 with
# and without tensor copies
SPECIAL = [("f16", 64, 2, 1, 16, 1, 300), ("f32", 128, 4, 1, 16, 1, 300), ("f16", 256, 4, 1, 64, 1, 700), ("f32", 32, 3, 2, 16, 6, 300), ("f16", 128, 4, 2, 7, 6, 300),
           ("f16", 32, 2, 8, 16, 150, 1200), ("f16", 64, 2, 8, 16, 150, 1200), ("f16", 64, 2, 8, 12, 150, 1200), ("f16", 128, 2, 8, 16, 150, 1200),
           ("f16", 128, 1, 16, 12, 150, 1200), ("f32", 64, 2, 8, 16, 150, 1200), ("f32", 128, 2, 8, 16, 150, 1200), ("f16", 256, 2, 8, 64, 150, 1200),
           ("f32", 256, 8, 8, 64, 150, 1200)]


def special(gpu, rng, dtype, dim, group, kv_heads, page, new, n, window, cap, scale, spoil):
    """Rows of one sequence against the 64-bit form: not finite where that is not, otherwise as near as scores up to 50 allow (near())."""
    c = Cache(gpu, 1, kv_heads, dim, page, 1, n // page + 1, n // page + 1, dtype)
    c.fill(rng, [n], poison=True)
    q = rng.standard_normal((new, kv_heads * group, dim)).astype(np.float32)
    pool, table = c.pool(), gpu.kv_table(c.id)[0]

    def put(p, which, head, d, value):
        c.held[0][p, 0, which, head, d] = value
        pool[int(table[p // page]), 0, which, head, p % page, d] = float(value)

    spoil(q, put)
    got = attention(gpu, c, [0], [0, new], new, kv_heads * group, q, layer=0, window=window, cap=cap, scale=scale)
    rows = sorted({*range(0, new, 13), *range(min(54, new), min(66, new)), new // 2, *range(max(new - 8, 0), new)})       # (54 ..: a tile's end)
    with np.errstate(all="ignore"):
        want = np.stack([ko.attend(q[r], c.held[0][:, 0, 0], c.held[0][:, 0, 1], n - new + r, window, 0, scale, cap)[0] for r in rows])
    got, fine = got[rows], np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[np.isinf(want)], want[np.isinf(want)].astype(np.float32))
    assert (np.abs(got[fine] - want[fine]) <= 16 * 8 * U * (1 + 50) * np.maximum(1, np.abs(want[fine]))).all()
    assert gpu.device_error() == 0
    c.close()
    return want


@pytest.mark.parametrize("cap", [0.0, 50.0])
@pytest.mark.parametrize("dtype,dim,group,kv_heads,page,new,n", SPECIAL)
def test_attention_special_queries_and_keys(gpu, dtype, dim, group, kv_heads, page, new, n, cap):
    """An infinite score is the cap with its sign where there is one, a NaN stays one: an infinite key with products of either sign,
    a NaN key, infinite and NaN queries, some seen by all rows and some by the last ones only."""
    def spoil(q, put):
        q[:, (kv_heads - 1) * group:, 9] = np.abs(q[:, (kv_heads - 1) * group:, 9])
        q[:, -1, 9] *= -1                                         # the last key head's last query head: scores of -infinity
        put(n - new, 0, kv_heads - 1, 9, np.inf)
        if kv_heads > 1:
            q[new // 2, 0, 3], q[new - 1, 0, dim - 1], q[0, 0, 7] = np.nan, np.inf, -np.inf
            put(n - new // 3, 0, 0, 5, -np.inf)
        else:
            q[0, 0, 3] = np.nan
        if kv_heads > 2:
            put(n - new // 3, 0, 1, 5, np.nan)

    want = special(gpu, np.random.default_rng(dim + new), dtype, dim, group, kv_heads, page, new, n, 0, cap, dim ** -0.5, spoil)
    assert np.isnan(want).any() and np.isfinite(want).any()


@pytest.mark.parametrize("cap", [0.0, 50.0])
@pytest.mark.parametrize("dtype,dim,group,kv_heads,page,new,n", SPECIAL + [("f16", 64, 2, 16, 16, 600, 1500), ("f16", 128, 2, 16, 12, 600, 1500)])
def test_attention_scale_of_zero(gpu, dtype, dim, group, kv_heads, page, new, n, cap):
    """The mean of what a row sees; rows that see nothing of a chunk of positions among others that do (the first of several, too)."""
    special(gpu, np.random.default_rng(new + dim), dtype, dim, group, kv_heads, page, new, n, 7 * n // 15, cap, 0.0, lambda q, put: None)


@pytest.mark.parametrize("cap", [0.0, 50.0])
@pytest.mark.parametrize("dtype,dim,group,kv_heads,page,new,n", SPECIAL)
def test_attention_negative_scale(gpu, dtype, dim, group, kv_heads, page, new, n, cap):
    """Scores with the other sign, and a query of zeros."""
    def spoil(q, put):
        q[new - 1, 0] = 0.0
        put(n - new, 0, 0, 1, 30000.0)                            # a key that decides

    special(gpu, np.random.default_rng(new + dim), dtype, dim, group, kv_heads, page, new, n, 0, cap, -1e-4, spoil)


@pytest.mark.parametrize("cap", [0.0, 50.0])
@pytest.mark.parametrize("dtype,dim,group,kv_heads,page,new,n", SPECIAL + [("f16", 128, 2, 16, 128, 333, 1111), ("f16", 64, 4, 8, 8, 333, 1111), ("f16", 128, 2, 16, 64, 600, 1501)])
@pytest.mark.parametrize("window,n_sink", [(0, 0), (300, 0), (300, 5), (130, 200)])
def test_attention_is_the_same_whatever_lies_where_no_row_sees(gpu, dtype, dim, group, kv_heads, page, new, n, cap, window, n_sink):
    """The same bits over pages whose other positions are NaN (an earlier holder's, say) and over zeros there: behind the sequence's
    end, between its first positions and its window."""
    rng = np.random.default_rng(dim + new)
    heads, n = kv_heads * group, n - 3
    c = Cache(gpu, 1, kv_heads, dim, page, 1, n // page + 1, n // page + 1, dtype)
    c.fill(rng, [n], poison=True)
    pool, table = c.pool(), gpu.kv_table(c.id)[0]
    if window:
        import torch
        p = np.arange(n_sink, max(n - new + 1 - window, n_sink))
        pool[torch.from_numpy(table[p // page].astype(np.int64)).cuda(), :, :, :, torch.from_numpy(p % page).cuda()] = float("nan")
    q = rng.standard_normal((new, heads, dim)).astype(np.float32)
    runs = []
    for _ in range(2):
        runs.append(attention(gpu, c, [0], [0, new], new, heads, q, 0, window, n_sink, cap=cap))
        pool[pool.isnan()] = 0.0
    assert np.isfinite(runs[0]).all() and np.array_equal(*runs)
    rows = [0, new // 2, new - 1]
    want, most = zip(*(ko.attend(q[r], c.held[0][:, 0, 0], c.held[0][:, 0, 1], n - new + r, window, n_sink, dim ** -0.5, cap) for r in rows))
    near(runs[0][rows], np.stack(want), max(most))
    assert gpu.device_error() == 0
    c.close()


def test_attention_leaves_out_what_is_not_there(gpu):
    rng = np.random.default_rng(4)
    c = Cache(gpu, 2, 1, 32, 4, 3, 4, 9, "f32")
    c.fill(rng, [6, 9, 0])
    q = rng.standard_normal((9, 2, 32)).astype(np.float32)
    # sequence 0: eight rows of six positions; one past the cache's; an empty sequence with a row
    got = attention(gpu, c, [0, 7, 2], [0, 7, 8, 9], 9, 2, q)
    assert gpu.device_error() == 1
    assert (got[0] == -7).all() and (got[7:] == -7).all()
    want, most = ko.attend(q[6], c.held[0][:, 1, 0], c.held[0][:, 1, 1], 5, 0, 0, 32 ** -0.5, 0.0)
    near(got[6], want, most)
    # starts that fall, or run past the rows: the entries are left out
    got = attention(gpu, c, [0, 1], [5, 2, 3], 9, 2, q)
    want, most = ko.attend(q[2], c.held[1][:, 1, 0], c.held[1][:, 1, 1], 8, 0, 0, 32 ** -0.5, 0.0)
    near(got[2], want, most)
    assert (got[[0, 1, 3, 4, 5]] == -7).all()
    gpu.device_error()
    got = attention(gpu, c, [1], [0, 1000000], 9, 2, q)
    assert (got == -7).all()
    gpu.device_error()
    c.close()


def test_attention_large_queries(gpu):
    """Scores of hundreds, far beyond what weights can hold beside each other, and queries near the end of the range."""
    rng = np.random.default_rng(14)
    for dtype in ("f16", "f32"):
        c = Cache(gpu, 1, 1, 64, 16, 1, 20, 20, dtype)
        c.fill(rng, [200])
        for size, scale in ((1e3, 0.125), (1e30, 1e-29), (1e-30, 1e29), (1e-30, 1.0)):
            q = (rng.standard_normal((3, 2, 64)) * size).astype(np.float32)
            got = attention(gpu, c, [0], [0, 3], 3, 2, q, layer=0, scale=scale)
            rows, want, most = expect(c, [200], [0], [0, 3], q, 2, 0, 0, 0, float(np.float32(scale)), 0.0)
            near(got, want, most)
        c.close()


def test_attention_captured_while_sequences_grow(gpu):
    """Two graphs of the same cache, recorded at short lengths and replayed in turn as the sequences grow."""
    rng = np.random.default_rng(10)
    heads, KV, D = 8, 2, 64
    c = Cache(gpu, 1, KV, D, 16, 2, 80, 120, "f16")
    c.fill(rng, [3, 20])
    n = heads * D
    gpu.map_create_typed(ACT, A.DTYPE_F32, 1, 6 * n)
    graphs = []
    for e in range(2):                                           # graph e: sequence e's last position
        hs = up(c, [e * n]), up(c, [(2 + e) * n]), *c.batch([e], [0, 1])
        gpu.capture_begin()
        gpu.map_attn_kv_dev(ACT, c.id, 0, *hs, 1, 1, heads, scale=D ** -0.5)
        graphs.append(gpu.capture_end())
    for step in range(3):
        grow = [200 * step, 333]
        gpu.kv_extend(c.id, [0, 1], grow)
        pool, table, lens = c.pool(), gpu.kv_table(c.id), gpu.kv_lens(c.id)
        import torch
        for s in range(2):
            x = rng.standard_normal((grow[s],) + c.shape).astype(np.float16)
            p = np.arange(lens[s] - grow[s], lens[s])
            if len(p):
                pool[torch.from_numpy(table[s][p // 16].astype(np.int64)).cuda(), :, :, :, torch.from_numpy(p % 16).cuda()] = torch.from_numpy(x).cuda()
            c.held[s] = np.concatenate([c.held[s], x])
        torch.cuda.synchronize()
        q = rng.standard_normal((2, heads, D)).astype(np.float32)
        gpu.scatter_contiguous(ACT, 0, q.reshape(-1))
        for g in graphs:
            gpu.graph_launch(g)
        got = gpu.gather(ACT, np.arange(2 * n, 4 * n, dtype=np.uint32)).view(np.float32).reshape(2, heads, D)
        for s in range(2):
            want, most = ko.attend(q[s], c.held[s][:, 0, 0], c.held[s][:, 0, 1], int(lens[s]) - 1, 0, 0, D ** -0.5, 0.0)
            near(got[s], want, most)
    for g in graphs:
        gpu.graph_destroy(g)
    assert gpu.device_error() == 0
    c.close()


def test_attention_on_a_lent_stream(gpu):
    """Queries written and results read by another program's stream, no wait in between; twice the same bits."""
    import torch
    rng = np.random.default_rng(12)
    heads, KV, D = 4, 1, 256
    c = Cache(gpu, 1, KV, D, 64, 1, 40, 40, "f16")
    c.fill(rng, [2000])
    gpu.map_create_typed(ACT, A.DTYPE_F32, 1, 2 * heads * D)
    q_h, o_h, (seq, start) = up(c, [0]), up(c, [heads * D]), c.batch([0], [0, 1])
    act = torch.as_tensor(gpu.map_array(ACT), device="cuda")
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    gpu.set_stream(st.cuda_stream)
    try:
        with torch.cuda.stream(st), gpu.batch():
            outs, qs = [], []
            for i in range(6):
                q = torch.randn(heads * D, device="cuda", generator=torch.Generator("cuda").manual_seed(i // 2))
                act[:heads * D] = q
                gpu.map_attn_kv_dev(ACT, c.id, 0, q_h, o_h, seq, start, 1, 1, heads, scale=D ** -0.5)
                outs.append(act[heads * D:].clone())
                qs.append(q)
    finally:
        gpu.set_stream(0)
    torch.cuda.synchronize()
    for i in range(0, 6, 2):
        assert torch.equal(outs[i], outs[i + 1])
        want, most = ko.attend(qs[i].view(heads, D).cpu().numpy(), c.held[0][:, 0, 0], c.held[0][:, 0, 1], 1999, 0, 0, D ** -0.5, 0.0)
        near(outs[i].view(heads, D).cpu().numpy(), want, most)
    c.close()


@pytest.mark.parametrize("page", [64, 60])
def test_pages_behind_4_billion_elements(gpu, page):
    """All operators on pages whose elements have numbers of more than 32 bits: append, attention in tiles of 2, 16 and 128, copies."""
    import torch
    rng = np.random.default_rng(page)
    KV, D, heads, n = 8, 128, 16, 1203
    low = -(-(1 << 32) // (2 * 2 * KV * page * D))                  # pages of 2^32 elements and more
    need = -(-n // page)
    c = Cache(gpu, 2, KV, D, page, 3, low, low + need + 2, "f16")
    gpu.kv_extend(c.id, [0], low * page)
    gpu.kv_extend(c.id, [1], n)
    table, pool = gpu.kv_table(c.id)[1], c.pool()
    assert int(table[:need].min()) * pool[0].numel() >= 1 << 32
    x = rng.standard_normal((n,) + c.shape).astype(np.float16)
    p = np.arange(n)

    def rows(seq):
        t = gpu.kv_table(c.id)[seq]
        return (torch.from_numpy(t[p // page].astype(np.int64)).cuda(), slice(None), slice(None), slice(None), torch.from_numpy(p % page).cuda())

    pool[rows(1)] = torch.from_numpy(x).cuda()
    c.held = [None, x, None]
    before, after, (oq, ok, ov, od), (qw, kw), starts = append(gpu, c, rng, [1], [3], heads, 1)
    got = pool[rows(1)].cpu().numpy()
    for i in range(3):
        k, v = (before[o[i]:o[i] + KV * D].reshape(KV, D) for o in (ok, ov))
        y = ko.rotate_normed(k, kw, n - 3 + i, 1e6, 1e-6)
        assert np.abs(got[n - 3 + i, 1, 0] - y).max() <= 2.0 ** -10 * np.abs(y).max() and np.array_equal(got[n - 3 + i, 1, 1], v.astype(np.float16))
        x[n - 3 + i, 1] = got[n - 3 + i, 1]
    assert np.array_equal(got, x)
    for new in (1, 6, 400):
        q = rng.standard_normal((new, heads, D)).astype(np.float32)
        out = attention(gpu, c, [1], [0, new], new, heads, q)
        at = sorted({0, new // 2, new - 1})
        want, most = zip(*(ko.attend(q[r], x[:, 1, 0], x[:, 1, 1], n - new + r, 0, 0, D ** -0.5, 0.0) for r in at))
        near(out[at], np.stack(want), max(most))
    gpu.kv_fork(c.id, 1, [2])
    gpu.kv_extend(c.id, [2], 1)                                      # a copy of the last page's positions
    assert np.array_equal(pool[rows(2)].cpu().numpy(), x)
    gpu.kv_truncate(c.id, [0])
    assert gpu.kv_compact(c.id) == need + 1 and gpu.kv_table(c.id).max() == need
    gpu.sync()
    for s in (1, 2):
        assert np.array_equal(pool[rows(s)].cpu().numpy(), x)
    assert gpu.device_error() == 0
    del pool
    c.close()


# ---- together ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_continuations_of_one_prompt(gpu, dtype):
    """A one-layer model as a host engine runs it: the prompt in two chunks, four continuations that share its pages, their
    tokens drawn from given random numbers, one of them ended and the pages moved together on the way; against the same model
    over plain lists.  The model: embedding rows as residual stream, q / k / v by fixed random matrices, logits = embedding
    table x attention output."""
    rng = np.random.default_rng(21)
    V, E, H, KV, D, page, window, n_sink, branches, steps = 97, 48, 4, 2, 32, 8, 11, 2, 4, 9
    emb = rng.standard_normal((V, E)).astype(np.float32)
    wq, wk, wv = ((rng.standard_normal((E, h * D)) / 4).astype(np.float32) for h in (H, KV, KV))
    wo = (rng.standard_normal((H * D, V)) / 2).astype(np.float32)
    qn, kn = (1 + 0.1 * rng.standard_normal((2, D))).astype(np.float32)
    prompt, u = rng.integers(0, V, 29), rng.random((steps, branches)).astype(np.float32)
    rule = [(0.9, 20, 0.9, 0.01), (1.2, 0, 0.8, 0.0), (0.7, 0, 1.0, 0.05), (0.0, 0, 1.0, 0.0)]
    kw = dict(base=1e4, eps=1e-6)

    # the plain program
    def plain():
        hist, out = [list(prompt) for _ in range(branches)], [[] for _ in range(branches)]
        margin = 1.0
        for t in range(steps):
            for b in range(branches):
                if b == 1 and t >= 5:
                    continue
                toks = hist[b]
                k = np.stack([ko.rotate_normed((emb[x] @ wk).reshape(KV, D), kn, i, **kw) for i, x in enumerate(toks)]).astype(HALF[dtype])
                v = np.stack([(emb[x] @ wv).reshape(KV, D) for x in toks]).astype(HALF[dtype])
                q = ko.rotate_normed((emb[toks[-1]] @ wq).reshape(H, D), qn, len(toks) - 1, **kw)
                o, _ = ko.attend(q, k, v, len(toks) - 1, window, n_sink, D ** -0.5, 0.0)
                tok, m = ko.sample((o.reshape(-1) @ wo).astype(np.float32), *rule[b], u[t, b])
                margin = min(margin, m)
                hist[b].append(tok)
                out[b].append(tok)
        return out, margin

    want, margin = plain()
    # the program on the operators
    c = Cache(gpu, 1, KV, D, page, branches, 8, 24, dtype)
    n_row = (H + 2 * KV) * D
    m = 64
    o_q, o_kv, o_out, o_log, o_u, o_tok, o_w = np.cumsum([0, m * H * D, m * 2 * KV * D, m * H * D, m * V, m, m]).tolist()
    assert n_row
    gpu.map_create_typed(ACT, A.DTYPE_F32, 1, o_w + 2 * D)
    gpu.scatter_contiguous(ACT, o_w, np.concatenate([qn, kn]))
    norm = up(c, [o_w]), up(c, [o_w + D])

    def forward(seqs, tokens):
        """Logits of the last row of every sequence; tokens[e]: the entry's new tokens."""
        new = [len(t) for t in tokens]
        starts, rows = np.cumsum([0] + new), sum(new)
        flat = np.concatenate(tokens)
        gpu.kv_extend(c.id, seqs, new)
        gpu.scatter_contiguous(ACT, o_q, np.ascontiguousarray(emb[flat] @ wq).reshape(-1))
        gpu.scatter_contiguous(ACT, o_kv, np.concatenate([(emb[flat] @ wk).reshape(-1), (emb[flat] @ wv).reshape(-1)]))
        r = np.arange(rows)
        q, k, v, o = up(c, o_q + r * H * D), up(c, o_kv + r * KV * D), up(c, o_kv + (rows + r) * KV * D), up(c, o_out + r * H * D)
        batch = c.batch(seqs, starts)
        with gpu.batch():
            gpu.map_qk_norm_rope_kv_dev(ACT, ACT, c.id, 0, q, k, v, *norm, q, *batch, len(seqs), rows, H, 1e4, 1e-6)
            gpu.map_attn_kv_dev(ACT, c.id, 0, q, o, *batch, len(seqs), rows, H, window, n_sink, D ** -0.5)
        last = (o_out + (starts[1:] - 1)[:, None] * H * D + np.arange(H * D)).astype(np.uint32)
        return gpu.gather(ACT, last.reshape(-1)).view(np.float32).reshape(len(seqs), -1) @ wo

    forward([0], [prompt[:17]])
    logits = np.repeat(forward([0], [prompt[17:]]), branches, 0)
    gpu.kv_fork(c.id, 0, [1, 2, 3])
    got, alive = [[] for _ in range(branches)], list(range(branches))
    for t in range(steps):
        if t == 5:
            gpu.kv_truncate(c.id, [1])
            alive.remove(1)
            logits = logits[[0, 2, 3]]
            live = gpu.kv_compact(c.id)
            assert live == 24 - gpu.kv_free_pages(c.id)
        n = len(alive)
        gpu.scatter_contiguous(ACT, o_log, logits.reshape(-1))
        gpu.scatter_contiguous(ACT, o_u, u[t, alive])
        rules = gpu.upload_dev(np.array([rule[b] for b in alive], A.SAMPLE_RULE))[0]
        c.handles.append(rules)
        gpu.map_sample_dev(ACT, up(c, o_log + np.arange(n) * V), rules, up(c, o_u + np.arange(n)), up(c, o_tok + np.arange(n)), n, V)
        toks = gpu.gather(ACT, (o_tok + np.arange(n)).astype(np.uint32)).view(np.float32).astype(int)
        for b, x in zip(alive, toks):
            got[b].append(int(x))
        logits = forward(alive, [[x] for x in toks])
    assert gpu.device_error() == 0
    # logits agree to some 1e-6 of the largest (16-bit keys rounded another way: 2^-11 of one key's value in a score); the draws
    # are this far from any other outcome
    assert margin > 1e-5
    assert got == want
    # the prompt's whole pages were never copied
    table = gpu.kv_table(c.id)
    assert len({tuple(table[b, :29 // page]) for b in alive}) == 1
    c.close()
