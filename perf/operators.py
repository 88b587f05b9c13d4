"""Timed cases of the paged-cache operators and of the sampling operator, plain and through the package.

A server that issues the backend's operators itself keeps the keys and values of its sequences in the pages of a cache:

* ``append``: the queries and keys of new tokens are normed per head and rotated, keys and values go into the pages
  (``map_qk_norm_rope_kv_dev``);
* ``attend``: the new tokens attend to their sequences' pages (``map_attn_kv_dev``), one token per sequence or a chunk of
  a prompt, with and without a sliding window and first tokens that stay visible;
* ``fork`` and ``compact``: several continuations of one prompt share its pages until they write; live pages move to the
  front of the pool (``kv_fork``, ``kv_extend``, ``kv_truncate``, ``kv_compact``);
* ``sample``: the next tokens from the logits, by each row's own rule and random number (``map_sample_dev``).

Shapes are the Gemma-3-1B one (4 query heads, 1 key head, head size 256, window 512), the Gemma-3-27B one (32, 16, 128,
window 1024) and smaller ones between them.
"""
import math
import weakref

import numpy as np
import torch

own = False

# ---- the cases ---------------------------------------------------------------------------------------------------


def listed():
    return [
        # one user's next token at the 1B shape, a short context: the smallest attention call
        {"name": "attend_1b_token", "kind": "attend", "heads": 4, "kv_heads": 1, "head_dim": 256, "type": "f16", "page": 64,
         "seqs": 1, "new": 1, "context": 130, "window": 0, "sinks": 0, "cap": 50.0},
        # a decode batch of 64 users at the 27B shape, contexts of different lengths
        {"name": "attend_27b_tokens", "kind": "attend", "heads": 32, "kv_heads": 16, "head_dim": 128, "type": "f16", "page": 64,
         "seqs": 64, "new": 1, "context": 2047, "window": 0, "sinks": 0, "cap": 50.0},
        # one user far into a long document: few rows, a long axis
        {"name": "attend_long_token", "kind": "attend", "heads": 32, "kv_heads": 8, "head_dim": 128, "type": "f16", "page": 16,
         "seqs": 1, "new": 1, "context": 65001, "window": 0, "sinks": 0, "cap": 0.0},
        # prompts of different lengths together, 32-bit cache
        {"name": "attend_ragged_f32", "kind": "attend", "heads": 4, "kv_heads": 1, "head_dim": 256, "type": "f32", "page": 64,
         "seqs": 7, "new": 259, "context": 300, "window": 0, "sinks": 0, "cap": 50.0},
        # a prompt's chunk behind a long context, windowed layer with sinks
        {"name": "attend_window_sinks", "kind": "attend", "heads": 32, "kv_heads": 16, "head_dim": 128, "type": "f16", "page": 64,
         "seqs": 2, "new": 1001, "context": 9000, "window": 1024, "sinks": 4, "cap": 0.0},
        # the largest: a chunk of 2048 tokens of a document behind 14000 others, global layer
        {"name": "attend_chunk", "kind": "attend", "heads": 32, "kv_heads": 16, "head_dim": 128, "type": "f16", "page": 64,
         "seqs": 1, "new": 2048, "context": 14000, "window": 0, "sinks": 0, "cap": 0.0},
        # a decode batch's queries, keys and values
        {"name": "append_1b_tokens", "kind": "append", "heads": 4, "kv_heads": 1, "head_dim": 256, "type": "f16", "page": 64,
         "seqs": 32, "new": 1, "context": 700},
        # a prompt's chunk at the 27B shape, far positions
        {"name": "append_27b_chunk", "kind": "append", "heads": 32, "kv_heads": 16, "head_dim": 128, "type": "f32", "page": 64,
         "seqs": 3, "new": 1365, "context": 30000},
        # 32 continuations of one prompt, each with room for its next token
        {"name": "fork_1b", "kind": "fork", "layers": 26, "kv_heads": 1, "head_dim": 256, "type": "f16", "page": 64, "seqs": 32, "tokens": 500},
        # half of the sequences ended: the others' pages move to the front
        {"name": "compact_1b", "kind": "compact", "layers": 26, "kv_heads": 1, "head_dim": 256, "type": "f16", "page": 64, "seqs": 14, "tokens": 509},
        # one user's next token out of a small vocabulary
        {"name": "sample_small", "kind": "sample", "rows": 1, "vocab": 32003, "rule": "default"},
        # a full batch over the full vocabulary, every row its own rule
        {"name": "sample_batch", "kind": "sample", "rows": 64, "vocab": 262144, "rule": "mixed"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


SHAPES = [(4, 1, 256), (32, 16, 128), (32, 8, 128), (14, 2, 64), (9, 3, 32), (8, 8, 64), (16, 1, 128), (10, 2, 256)]


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "append", "fork", "compact", "sample", "sample"])
    if kind == "sample":
        return {"kind": kind, "rows": _log(rng, 1, 64), "vocab": _log(rng, 100, 262144),
                "rule": rng.choice(["default", "mixed", "nucleus", "top_k", "min_p", "plain"])}
    heads, kv_heads, head_dim = rng.choice(SHAPES)
    kv_type, page = rng.choice(["f16", "f16", "f32"]), rng.choice([16, 64, 64, 48, 7])
    if kind in ("fork", "compact"):
        layers, seqs = rng.choice([1, 8, 26]), _log(rng, 2, 32)
        position = 2 * layers * kv_heads * head_dim * (2 if kv_type == "f16" else 4)
        most = min(700, int(2e9 / (position * seqs)))            # 2 GB of pages at most
        return {"kind": kind, "layers": layers, "kv_heads": kv_heads, "head_dim": head_dim, "type": kv_type, "page": page,
                "seqs": seqs, "tokens": _log(rng, 2, max(3, most))}
    seqs = _log(rng, 1, 64)
    new = 1 if rng.random() < 0.4 else _log(rng, 2, max(2, 2048 // seqs))
    c = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "type": kv_type, "page": page, "seqs": seqs, "new": new}
    if kind == "append":
        return dict(c, context=_log(rng, 1, 100000 // seqs))
    windowed = rng.random() < 0.4
    # scores of all heads times head size: those of the largest listed case at most
    most = int(2048 * 16048 * 32 * 128 / (seqs * new * heads * head_dim))
    return dict(c, context=_log(rng, 1, max(1, min(60000 // seqs, most) - new)), window=_log(rng, 16, 4096) if windowed else 0,
                sinks=rng.choice([0, 1, 4]) if windowed else 0, cap=rng.choice([0.0, 50.0]))


# ---- inputs ----------------------------------------------------------------------------------------------------------

LAYERS, LAYER = 2, 1                      # append and attend: a cache of two layers, the second one in use
BASE, EPS = 1e6, 1e-6
HALF = {"f16": torch.float16, "f32": torch.float32}


def _spread(most, n, low):
    """n lengths between most * low and most, evenly spread, in a mixed order; the first is the longest."""
    v = np.linspace(most, max(1, round(most * low)), n).round().astype(int)
    return [int(v[(3 * i) % n]) for i in range(n)] if n % 3 else [int(x) for x in v]


def _lengths(case):
    """New tokens and lengths (with them) of a batch's sequences."""
    new = _spread(case["new"], case["seqs"], 0.3)
    return new, [c + n for c, n in zip(_spread(case["context"], case["seqs"], 0.25), new)]


def _table(lens, page):
    """Pages of sequences that grew in turns, a page each at a time: [seqs][most pages], -1 where there is none."""
    need = [-(-n // page) for n in lens]
    table, at = np.full((len(lens), max(need)), -1, np.int32), 0
    for j in range(max(need)):
        for s, n in enumerate(need):
            if j < n:
                table[s, j], at = at, at + 1
    return table, at


def _inputs(case, seed):
    """What a program has in hand, as tensors on the GPU and numbers."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=gen)

    s = {"case": case, "kind": case["kind"]}
    if case["kind"] == "sample":
        R, V = case["rows"], case["vocab"]
        rng = np.random.default_rng(seed)
        # most logits around zero, some dozens far above: between a sure next word and an open one
        s["logits"] = randn(R, V) * 2.5 + 14.0 * torch.rand((R, V), device="cuda", generator=gen) ** (V / 40)
        s["u"] = torch.rand(R, device="cuda", generator=gen)
        rules = np.zeros(R, [("temperature", "f4"), ("top_k", "u4"), ("top_p", "f4"), ("min_p", "f4")])
        kinds = {"default": [(0.8, 40, 0.95, 0.0)], "nucleus": [(1.0, 0, 0.9, 0.0)], "top_k": [(0.7, 200, 1.0, 0.0)],
                 "min_p": [(1.3, 0, 1.0, 0.05)], "plain": [(1.0, 0, 1.0, 0.0)]}
        some = kinds[case["rule"]] if case["rule"] in kinds else sum(kinds.values(), []) + [(0.0, 0, 1.0, 0.0), (1.1, 5000, 0.99, 0.01)]
        for r in range(R):
            rules[r] = some[r % len(some)]
        s["rules_np"] = rules[rng.permutation(R)]
        s["rules"] = {k: torch.from_numpy(s["rules_np"][k].astype(np.float64)).cuda() for k in rules.dtype.names}
        return s
    KV, D, page, dtype = case["kv_heads"], case["head_dim"], case["page"], HALF[case["type"]]
    if case["kind"] in ("fork", "compact"):
        pages = -(-case["tokens"] // page)
        n_pages = pages + case["seqs"] + 3 if case["kind"] == "fork" else pages * case["seqs"] + 3
        s["shape"] = (n_pages, case["layers"], 2, KV, page, D)
        s["max_seqs"], s["max_pages"] = case["seqs"] + 1, pages + 1
        s["pool"] = torch.empty(s["shape"], dtype=dtype, device="cuda")
        for p in s["pool"].split(max(1, (1 << 26) // s["pool"][0].numel())):
            p.copy_(randn(*p.shape))
        return s
    H = case["heads"]
    new, lens = _lengths(case)
    table, n_pages = _table(lens, page)
    s.update(new=new, lens=lens, rows=sum(new), starts=np.cumsum([0] + new), shape=(n_pages, LAYERS, 2, KV, page, D),
             max_seqs=case["seqs"], max_pages=table.shape[1])
    s["pool"] = randn(*s["shape"]).to(dtype)
    s["table"] = torch.from_numpy(table).cuda()
    s["lens_dev"], s["new_dev"] = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (lens, new))
    s["starts_dev"] = torch.from_numpy(s["starts"].astype(np.int32)).cuda()
    if case["kind"] == "attend":
        s["q"] = randn(s["rows"], H, D) * 2.5                   # scores of a few units: some tokens matter more than others
    else:
        s["q"], s["k"], s["v"] = randn(s["rows"], H, D) * 3.0, randn(s["rows"], KV, D) * 0.7, randn(s["rows"], KV, D)
        s["q_norm"], s["k_norm"] = 1.0 + 0.1 * randn(D), 1.0 + 0.1 * randn(D)
    return s


# ---- the package's side: maps, handles and caches that a program keeps -------------------------------------------------

_kept = {}
_free_maps = list(range(255, -1, -1))


def _gpu():
    """The backend, on torch's stream (1 is the default stream's handle), in an open batch: calls do not wait for the GPU."""
    stream = torch.cuda.current_stream().cuda_stream or 1
    if "gpu" not in _kept:
        import adam_b200
        _kept["gpu"], _kept["stream"] = adam_b200.init(), None
        _kept["gpu"].batch_begin()
    if _kept["stream"] != stream:
        _kept["gpu"].set_stream(stream)
        _kept["stream"] = stream
    return _kept["gpu"]


class _Held:
    """Maps, loc handles and a cache of one program, given back with it."""

    def __init__(self):
        self.gpu, self.maps, self.handles, self.kvs = _gpu(), [], [], []
        self._end = weakref.finalize(self, _Held._release, self.gpu, self.maps, self.handles, self.kvs)

    def map(self, *tensors, extra=0):
        """A float32 map with the tensors one behind the other and room behind them: its id, their offsets, a view of it."""
        import adam_b200
        m = _free_maps.pop()
        self.maps.append(m)
        offs = np.cumsum([0] + [t.numel() for t in tensors]).tolist()
        self.gpu.map_create_typed(m, adam_b200.DTYPE_F32, 1, offs[-1] + extra)
        view = self.view(self.gpu.map_array(m))
        for o, t in zip(offs, tensors):
            view[o:o + t.numel()] = t.reshape(-1)
        return m, offs, view

    def view(self, array):
        """A tensor over the library's memory; what it lies in lives as long as the tensor does."""
        array.owner = self
        return torch.as_tensor(array, device="cuda")

    def up(self, values):
        h, _ = self.gpu.upload_dev(np.ascontiguousarray(values))
        self.handles.append(h)
        return h

    def cache(self, s, case, layers):
        n_pages, _, _, KV, page, D = s["shape"]
        kv = self.gpu.kv_create(n_layer=layers, n_head_kv=KV, head_dim=D, n_pages=n_pages, page_size=page, max_seqs=s["max_seqs"],
                                max_pages=s["max_pages"], kv_dtype=case["type"])
        self.kvs.append(kv)
        return kv

    @staticmethod
    def _release(gpu, maps, handles, kvs):
        for k in kvs:
            gpu.kv_destroy(k)
        for h in handles:
            gpu.free_handle(h)
        for m in maps:
            gpu.map_destroy(m)
            _free_maps.append(m)


def _hold(s):
    """The same inputs in the package's maps and cache, with the loc handles of the calls."""
    case = s["case"]
    held = s["held"] = _Held()
    g = s["gpu"] = held.gpu
    if s["kind"] == "sample":
        R, V = case["rows"], case["vocab"]
        s["map"], offs, view = held.map(s.pop("logits"), s["u"], extra=R)
        s["out"] = view[offs[2]:]
        s["handles"] = held.up((V * np.arange(R)).astype(np.uint32)), held.up(s["rules_np"]), held.up((offs[1] + np.arange(R)).astype(np.uint32)), \
            held.up((offs[2] + np.arange(R)).astype(np.uint32))
        return
    kv = s["kv"] = held.cache(s, case, case.get("layers", LAYERS))
    pool = held.view(g.kv_array(kv, "pool"))
    pool.copy_(s["pool"])
    s["pool"] = pool
    s["views"] = [held.view(g.kv_array(kv, k)) for k in ("table", "lens")]
    if s["kind"] == "fork":
        g.kv_extend(kv, [0], [case["tokens"]])
        s["others"] = np.arange(1, case["seqs"] + 1, dtype=np.uint32)
        return
    if s["kind"] == "compact":
        everyone = np.arange(case["seqs"], dtype=np.uint32)
        s["ended"], s["going"] = everyone[::2].copy(), everyone[1::2].copy()
        return
    left, H, D, rows = np.array(s["lens"]), case["heads"], case["head_dim"], s["rows"]
    while left.any():                                            # in turns, a page each at a time
        who = np.flatnonzero(left).astype(np.uint32)
        n = np.minimum(left[who], case["page"]).astype(np.uint32)
        g.kv_extend(kv, who, n)
        left[who] -= n
    s["batch"] = held.up(np.arange(case["seqs"], dtype=np.uint32)), held.up(s["starts"].astype(np.uint32))
    each = np.arange(rows)
    if s["kind"] == "attend":
        s["map"], offs, view = held.map(s["q"], extra=rows * H * D)
        s["handles"] = [held.up((o + each * H * D).astype(np.uint32)) for o in offs]
    else:
        s["map"], offs, view = held.map(s["q"], s["k"], s["v"], s["q_norm"], s["k_norm"], extra=rows * H * D)
        width = (H * D, case["kv_heads"] * D, case["kv_heads"] * D)
        s["handles"] = [held.up((o + each * w).astype(np.uint32)) for o, w in zip(offs, width)] + \
            [held.up(np.array([o], np.uint32)) for o in offs[3:5]] + [held.up((offs[5] + each * H * D).astype(np.uint32))]
    s["out"] = view[offs[-1]:].view(rows, H * D)


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        _hold(s)
    return s


# ---- run ---------------------------------------------------------------------------------------------------------------


def run(s):
    if own:
        return _own(s)
    return {"sample": _sample, "append": _append, "attend": _attend, "fork": _fork, "compact": _compact}[s["kind"]](s)


def _own(s):
    g, case = _gpu(), s["case"]
    if s["kind"] == "sample":
        g.map_sample_dev(s["map"], *s["handles"], case["rows"], case["vocab"])
        return s["out"]
    kv = s["kv"]
    if s["kind"] == "fork":
        g.kv_truncate(kv, s["others"], 0)
        g.kv_fork(kv, 0, s["others"])
        g.kv_extend(kv, s["others"], 1)
        return [s["pool"], *s["views"]]
    if s["kind"] == "compact":
        g.kv_truncate(kv, np.concatenate([s["ended"], s["going"]]), 0)
        g.kv_extend(kv, s["ended"], case["tokens"])
        g.kv_extend(kv, s["going"], case["tokens"])
        g.kv_truncate(kv, s["ended"], 0)
        return [s["pool"], *s["views"], g.kv_compact(kv)]
    seqs, starts = s["batch"]
    if s["kind"] == "attend":
        q, out = s["handles"]
        g.map_attn_kv_dev(s["map"], kv, LAYER, q, out, seqs, starts, case["seqs"], s["rows"], case["heads"], window=case["window"],
                          n_sink=case["sinks"], scale=case["head_dim"] ** -0.5, cap=case["cap"])
        return s["out"]
    q, k, v, q_norm, k_norm, out = s["handles"]
    g.map_qk_norm_rope_kv_dev(s["map"], s["map"], kv, LAYER, q, k, v, q_norm, k_norm, out, seqs, starts, case["seqs"], s["rows"],
                              case["heads"], freq_base=BASE, eps=EPS)
    return [s["out"], s["pool"]]


def _sample(s):
    x = s["logits"].double()
    x = torch.where(x.isnan(), -math.inf, x)
    T, top_k, top_p, min_p = (s["rules"][k][:, None] for k in ("temperature", "top_k", "top_p", "min_p"))
    best = x.amax(1, keepdim=True)
    greedy = T <= 0
    w = torch.exp((x - best) / torch.where(greedy, 1.0, T))
    _, order = torch.sort(x, dim=1, descending=True, stable=True)            # ties: the lower index first
    ws = w.gather(1, order)
    place = torch.arange(x.shape[1], device=x.device)
    ws = torch.where((top_k > 0) & (place >= top_k), 0.0, ws)
    before = ws.cumsum(1) - ws
    kept = (ws > 0) & ((top_p >= 1) | (place == 0) | (before < top_p * ws.sum(1, keepdim=True))) & (ws >= min_p)
    kept = torch.where(greedy, place == 0, kept)
    cdf = torch.where(torch.zeros_like(kept).scatter(1, order, kept), w, 0.0).cumsum(1)
    return (cdf <= s["u"].double()[:, None] * cdf[:, -1:]).sum(1).float()


def _places(s):
    """Of every row: its entry in the batch and its position."""
    row = torch.arange(s["rows"], device="cuda")
    entry = torch.searchsorted(s["starts_dev"][1:].long(), row, right=True)
    return entry, row - s["starts_dev"][entry] + s["lens_dev"][entry] - s["new_dev"][entry]


def _append(s):
    case, D = s["case"], s["case"]["head_dim"]
    entry, pos = _places(s)
    turn = BASE ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
    angle = pos.double()[:, None, None] * turn
    c, sn = angle.cos().float(), angle.sin().float()

    def rotated(x, w):
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        a, b = y[..., :D // 2], y[..., D // 2:]
        return torch.cat([a * c - b * sn, a * sn + b * c], -1)

    page = s["table"][entry, pos // case["page"]].long()
    slot = pos % case["page"]
    kv_head = torch.arange(case["kv_heads"], device="cuda")
    at = page[:, None], LAYER, 0, kv_head[None, :], slot[:, None]
    s["pool"][at] = rotated(s["k"], s["k_norm"]).to(s["pool"].dtype)
    s["pool"][at[0], LAYER, 1, at[3], at[4]] = s["v"].to(s["pool"].dtype)
    return [rotated(s["q"], s["q_norm"]).reshape(s["rows"], -1), s["pool"]]


def _attend(s):
    case = s["case"]
    S, KV, D, page = case["seqs"], case["kv_heads"], case["head_dim"], case["page"]
    H, T, L = case["heads"], max(s["new"]), s["max_pages"] * page
    tok = torch.arange(T, device="cuda")
    live = tok[None, :] < s["new_dev"][:, None]                                # [S, T]
    row = torch.where(live, s["starts_dev"][:-1, None] + tok, 0).long()
    pos = s["lens_dev"][:, None] - s["new_dev"][:, None] + tok
    kv = s["pool"][:, LAYER][s["table"].clamp(min=0).long()].float()            # [S, pages, 2, KV, page, D]
    k, v = (kv[:, :, i].permute(0, 2, 1, 3, 4).reshape(S, KV, L, D) for i in (0, 1))
    q = s["q"][row].reshape(S, T, KV, H // KV, D).permute(0, 2, 3, 1, 4).reshape(S, KV, -1, D)
    score = torch.matmul(q, k.transpose(2, 3)).mul_(D ** -0.5)
    if case["cap"]:
        score = score.div_(case["cap"]).tanh_().mul_(case["cap"])
    at = torch.arange(L, device="cuda")
    seen = at <= pos[..., None]                                                # [S, T, L]
    if case["window"]:
        seen = seen & ((at > pos[..., None] - case["window"]) | (at < case["sinks"]))
    score = score.view(S, KV, H // KV, T, L).masked_fill_(~seen[:, None, None], -math.inf).view(S, KV, -1, L)
    p = score.sub_(score.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    o = o.view(S, KV, H // KV, T, D).permute(0, 3, 1, 2, 4).reshape(S, T, H * D)
    return o[live]


def _pages(tokens, page):
    return -(-tokens // page)


def _fork(s):
    case, pool = s["case"], s["pool"]
    n, page, others = case["tokens"], case["page"], case["seqs"]
    have, need, rest = _pages(n, page), _pages(n + 1, page), n % page
    table = torch.full((s["max_seqs"], s["max_pages"]), -1, dtype=torch.int32, device="cuda")
    table[:, :have] = torch.arange(have, device="cuda", dtype=torch.int32)
    # a page of its own for every continuation's next token: a copy of the prompt's last page, or a new one
    mine = have + torch.arange(others, device="cuda")
    if rest:
        pool[mine, :, :, :, :rest] = pool[have - 1, :, :, :, :rest]
    table[1:, need - 1] = mine.int()
    lens = torch.full((s["max_seqs"],), n + 1, dtype=torch.int32, device="cuda")
    lens[0] = n
    return [pool, table, lens]


def _compact(s):
    case, pool = s["case"], s["pool"]
    each, seqs = _pages(case["tokens"], case["page"]), case["seqs"]
    ended, going = (seqs + 1) // 2, seqs // 2
    live = going * each
    old = ended * each + torch.arange(live, device="cuda")
    # the live pages from `live` on move down, in their order; those that lie below stay
    moved = old[old >= live]
    free = torch.arange(min(live, ended * each), device="cuda")[:len(moved)]
    pool[free] = pool[moved]
    now = old.clone()
    now[len(old) - len(moved):] = free
    table = torch.full((s["max_seqs"], s["max_pages"]), -1, dtype=torch.int32, device="cuda")
    table[1:2 * going:2, :each] = now.view(going, each).int()
    lens = torch.zeros(s["max_seqs"], dtype=torch.int32, device="cuda")
    lens[1:2 * going:2] = case["tokens"]
    return [pool, table, lens, live]


# ---- the same from the definitions, in 64 bits ------------------------------------------------------------------------


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "sample":
        return _exact_sample(s)
    if case["kind"] == "fork":
        return _exact_fork(s)
    if case["kind"] == "compact":
        return _exact_compact(s)
    table, D, page, rows = s["table"].cpu().numpy(), case["head_dim"], case["page"], s["rows"]
    out = torch.empty((rows, case["heads"] * D), dtype=torch.float64, device="cuda")
    if case["kind"] == "append":
        pool = s["pool"].double()
        freq = torch.tensor([BASE ** (-2.0 * i / D) for i in range(D // 2)], dtype=torch.float64, device="cuda")
        for i, (n, length) in enumerate(zip(s["new"], s["lens"])):
            r = slice(int(s["starts"][i]), int(s["starts"][i + 1]))
            pos = torch.arange(length - n, length, device="cuda")
            turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), pos.double()[:, None] * freq)[:, None]
            res = []
            for x, w in ((s["q"], s["q_norm"]), (s["k"], s["k_norm"])):
                y = x[r].double()
                y = y * ((y ** 2).sum(-1, keepdim=True) / D + EPS) ** -0.5 * w.double()
                z = torch.complex(y[..., :D // 2].contiguous(), y[..., D // 2:].contiguous()) * turn
                res.append(torch.cat([z.real, z.imag], -1))
            out[r] = res[0].flatten(1)
            pages = torch.from_numpy(table[i]).cuda().long()[pos // page]
            pool[pages, LAYER, 0, :, pos % page] = res[1]
            pool[pages, LAYER, 1, :, pos % page] = s["v"][r].double()
        return [out, pool]
    KV, H = case["kv_heads"], case["heads"]
    for i, (n, length) in enumerate(zip(s["new"], s["lens"])):
        pages = torch.from_numpy(table[i][:_pages(length, page)]).cuda().long()
        pos = torch.arange(length - n, length, device="cuda")[:, None]
        at = torch.arange(length, device="cuda")[None]
        hidden = at > pos
        if case["window"]:
            hidden |= (at + case["window"] <= pos) & (at >= case["sinks"])
        for h in range(KV):
            k, v = (s["pool"][pages, LAYER, j, h].reshape(-1, D)[:length].double() for j in (0, 1))
            for a in range(h * (H // KV), (h + 1) * (H // KV)):
                r = slice(int(s["starts"][i]), int(s["starts"][i + 1]))
                z = s["q"][r, a].double() @ k.T / math.sqrt(D)
                z = case["cap"] * torch.tanh(z / case["cap"]) if case["cap"] else z
                z[hidden] = -math.inf
                out[r, a * D:(a + 1) * D] = torch.exp(z - torch.logsumexp(z, 1, keepdim=True)) @ v
    return out


def _exact_sample(s):
    logits, u, res = s["logits"].cpu().numpy().astype(np.float64), s["u"].cpu().numpy().astype(np.float64), []
    for x, draw_at, (T, top_k, top_p, min_p) in zip(logits, u, s["rules_np"].tolist()):
        first = int(np.argmax(x))
        if T <= 0:
            res.append(first)
            continue
        w = np.exp((x - x[first]) / T)
        # the candidates: by weight, the lower index first among equal ones
        cand = np.argsort(-x, kind="stable")[:top_k or None]
        if top_p < 1:
            total = np.cumsum(w[cand])
            cand = cand[:int(np.searchsorted(total, top_p * total[-1], side="left")) + 1]
        cand = np.sort(cand[w[cand] >= min_p])
        total = np.cumsum(w[cand])
        res.append(int(cand[np.searchsorted(total, draw_at * total[-1], side="right")]))
    return torch.tensor(res, dtype=torch.float64)


def _exact_fork(s):
    """Page by page, as a table of owners would tell it."""
    case, pool = s["case"], s["pool"]
    n, page = case["tokens"], case["page"]
    table, lens = np.full((s["max_seqs"], s["max_pages"]), -1, np.int32), np.full(s["max_seqs"], n + 1, np.int32)
    lens[0], unused = n, _pages(n, page)
    for c in range(s["max_seqs"]):
        for j in range(_pages(n, page)):
            table[c, j] = j
        if c and n % page:
            pool[unused][..., :n % page, :] = pool[n // page][..., :n % page, :]
        if c:
            table[c, n // page], unused = unused, unused + 1
    return [pool.double(), torch.from_numpy(table), torch.from_numpy(lens)]


def _exact_compact(s):
    case, pool, page = s["case"], s["pool"], s["case"]["page"]
    each, seqs = _pages(case["tokens"], page), case["seqs"]
    first = {c: i * each for i, c in enumerate(list(range(0, seqs, 2)) + list(range(1, seqs, 2)))}
    going = list(range(1, seqs, 2))
    live = {first[c] + j: (c, j) for c in going for j in range(each)}
    table, lens = np.full((s["max_seqs"], s["max_pages"]), -1, np.int32), np.zeros(s["max_seqs"], np.int32)
    holes = [p for p in range(len(live)) if p not in live]
    for p in sorted(live):
        c, j = live[p]
        to = p if p < len(live) else holes.pop(0)
        if to != p:
            pool[to] = pool[p]
        table[c, j], lens[c] = to, case["tokens"]
    return [pool.double(), torch.from_numpy(table), torch.from_numpy(lens), len(live)]


# ---- what a pass cannot do without -----------------------------------------------------------------------------------


def work(case):
    if case["kind"] == "sample":
        return {"bytes": case["rows"] * (4 * case["vocab"] + 24), "flops": 8 * case["rows"] * case["vocab"]}
    size = 2 if case["type"] == "f16" else 4
    row = 2 * case["kv_heads"] * case["head_dim"] * size                     # a position's key and value, one layer
    if case["kind"] == "fork":
        rest, seqs = case["tokens"] % case["page"], case["seqs"]
        return {"bytes": (seqs + 1) * rest * row * case["layers"] + 4 * seqs * (_pages(case["tokens"] + 1, case["page"]) + 1), "flops": 0}
    if case["kind"] == "compact":
        each = _pages(case["tokens"], case["page"])
        moved = min(case["seqs"] // 2, (case["seqs"] + 1) // 2) * each
        return {"bytes": 2 * moved * case["page"] * row * case["layers"] + 4 * moved, "flops": 0}
    new, lens = _lengths(case)
    D, H, rows = case["head_dim"], case["heads"], sum(new)
    if case["kind"] == "append":
        KV = case["kv_heads"]
        return {"bytes": rows * (8 * H * D + 8 * KV * D + row) + 8 * D, "flops": rows * (10 * H + 10 * KV) * D}
    seen = read = 0
    for n, length in zip(new, lens):
        first = length - n
        w, k = case["window"] or length, case["sinks"]
        pos = np.arange(first, length)
        seen += int((np.minimum(pos + 1, w) + np.minimum(k, np.maximum(0, pos + 1 - w))).sum())
        read += min(length, n + w - 1) + min(k, max(0, first + 1 - w))
    return {"bytes": 8 * rows * H * D + read * row, "flops": 4 * seen * H * D}
