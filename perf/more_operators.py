"""The calls that a server of many chats makes around the paged 8-bit K/V cache, as cases to be timed and compared.

A case is a call at one size.  Its kinds:

  fork     sequences become the beginnings of others: their block tables; what the copied last pages stand for is read back
  attend   attention of a step's rows over a cache whose sequences share long prefixes
  rope     rotary positions of the q|k columns of fused q|k|v rows
  logits   penalties, biases and masks on a step's logits, and each row's best token

What the operators compute:

  fork     sequence b becomes the first keep[b] positions of sequence from[b], all at once.  Pages of 32 positions that are whole are
           shared.  A last page that is not whole stays with the first sequence that it is the last page of, if no sequence has it as
           a whole one; the others get copies, in the order of the sequences, in the free pages of the lowest numbers
  attend   softmax(q . K * head_dim^-1/2) V over the positions up to the row's own; head h reads kv head h / (heads / kv_heads)
  rope     (x, y) becomes amplitude * (x cos a - y sin a, y cos a + x sin a), a = position * frequency, for `rot` columns of a head, the
           others as they are; x and y lie rot / 2 columns apart ("halves") or side by side ("pairs")
  logits   of a token that occurs c > 0 times in the row's history x becomes x / r or, where x <= 0, x * r, then x - (f c + p); then
           the token's bias is added (of several the last one's); where its bit of the mask is 0 it is -inf.  The best token is the
           first of the largest values, before they are rounded to the outputs' type

The cache holds K and V in int8 with one fp32 scale for each page and kv head, for K and for V.  A run of rows goes into a page
from offset f on with t = max|x| / 127: at f = 0 the scale is t, else the old one times the smallest power of two that reaches
t, and the codes before f are halved (to the nearest even) as often.  Codes are x / scale, rounded to the nearest even.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

BLOCK = 32
REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# (query heads, kv heads, head_dim): the library's two models, then groups of 4, none and all heads in one group
LAYOUTS = [(14, 2, 64), (12, 2, 128), (32, 8, 128), (20, 20, 64), (8, 1, 128)]
VOCAB = 151936


def _cache_case(kind, layout, dtype, groups, members, prefix, hold=(0, 0), add=(0, 0), layers=1, name=None):
    """`groups` prefixes of prefix[0]..prefix[1] positions with `members` sequences each, which then hold hold[0]..hold[1]
    positions of their own and add add[0]..add[1] rows."""
    H, KVH, hd = layout
    case = {"kind": kind, "heads": H, "kv_heads": KVH, "head_dim": hd, "dtype": dtype, "groups": groups, "members": members,
            "prefix_lo": prefix[0], "prefix_hi": prefix[1], "hold_lo": hold[0], "hold_hi": hold[1], "add_lo": add[0], "add_hi": add[1],
            "layers": layers}
    if name:
        case["name"] = name
    return case


def _rope_case(layout, dtype, rows, positions, rot, order, scaling, name=None):
    H, KVH, hd = layout
    case = {"kind": "rope", "heads": H, "kv_heads": KVH, "head_dim": hd, "dtype": dtype, "rows": rows, "positions": positions, "rot": rot,
            "order": order, "scaling": scaling}
    if name:
        case["name"] = name
    return case


def _logits_case(rows, vocab, dtype, history, biases, masked, name=None):
    case = {"kind": "logits", "rows": rows, "vocab": vocab, "dtype": dtype, "history_lo": history[0], "history_hi": history[1],
            "biases": biases, "masked": masked}
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # four answers to one question are tried: the chat's cache for each of them
        _cache_case("fork", LAYOUTS[0], "f32", 1, 4, (301, 301), layers=2, name="fork_answers_05b"),
        # a server starts 256 chats from 4 system prompts
        _cache_case("fork", LAYOUTS[2], "bf16", 4, 64, (1000, 5000), layers=4, name="fork_server"),
        # the next token of the four answers
        _cache_case("attend", LAYOUTS[0], "f32", 1, 4, (301, 301), (1, 40), (1, 1), name="attend_answers_05b"),
        # 32 chats behind one long system prompt, two tokens each (the last one and a guess)
        _cache_case("attend", LAYOUTS[1], "f16", 1, 32, (4100, 4100), (100, 900), (1, 2), name="attend_chats_15b"),
        # questions about one very long text
        _cache_case("attend", LAYOUTS[4], "bf16", 1, 8, (131072, 131072), (1, 200), (1, 1), name="attend_long_text"),
        # a full server: 128 chats behind two system prompts with many examples
        _cache_case("attend", LAYOUTS[2], "bf16", 2, 64, (12000, 17000), (200, 2000), (1, 1), name="attend_server"),
        # the next token of one chat
        _rope_case(LAYOUTS[0], "f32", 1, 400, 64, "halves", "plain", name="rope_token_05b"),
        # 64 chats of very different lengths, a model whose context was stretched, half of each head turned
        _rope_case(LAYOUTS[2], "bf16", 64, 131072, 64, "pairs", "yarn", name="rope_batch"),
        # a long document as the prompt
        _rope_case(LAYOUTS[2], "bf16", 8192, 32768, 128, "halves", "bands", name="rope_prompt"),
        # the next token of one chat
        _logits_case(1, VOCAB, "f32", (300, 300), 8, 0, name="logits_chat"),
        # a server's 64 chats, a quarter of them answering in a grammar
        _logits_case(64, VOCAB, "bf16", (0, 4000), 40, 16, name="logits_server"),
        # 256 long chats in fp32
        _logits_case(256, VOCAB, "f32", (2000, 16000), 300, 40, name="logits_long"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm, odd half of the time."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, v | 1 if rng.random() < 0.5 else v))


def draw(rng):
    kind = rng.choice(["fork", "attend", "attend", "rope", "logits"])
    layout, dtype = rng.choice(LAYOUTS), rng.choice(sorted(TYPES))
    H, KVH, hd = layout
    if kind == "rope":
        return _rope_case(layout, dtype, _log(rng, 1, 8192 * 2560 // ((H + KVH) * hd) // 2), _log(rng, 64, 1000000),
                          hd // rng.choice([1, 1, 2, 4]), rng.choice(["halves", "pairs"]), rng.choice(["plain", "linear", "bands", "yarn"]))
    if kind == "logits":
        vocab = rng.choice([VOCAB, _log(rng, 1000, 200000)])
        rows = _log(rng, 1, min(512, 256 * VOCAB // vocab))
        hi = _log(rng, 4, 16000)
        return _logits_case(rows, vocab, dtype, (rng.choice([0, hi // 2]), hi), rng.choice([0, _log(rng, 1, 300)]),
                            rng.choice([0, rng.randint(0, rows)]))
    groups = rng.choice([1, 1, 2, 4])
    if kind == "fork":
        hi = _log(rng, 40, 5000)
        return _cache_case(kind, layout, dtype, groups, _log(rng, 2, 64), (hi * 3 // 4, hi), layers=rng.randint(1, 4))
    members = _log(rng, 2, 64 if groups < 4 else 16)
    hi = min(_log(rng, 40, 131072), 131072 // KVH, 262144 // members, 32768 // groups)
    own_hi = _log(rng, 2, 2000)
    return _cache_case(kind, layout, dtype, groups, members, (hi * 3 // 4, hi), (own_hi // 4, own_hi), (1, rng.choice([1, 1, 1, 3])))


# ---------------------------------------------------------------------------- inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _int(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def _pages(n):
    return -(-n // BLOCK)


_stream = None


def _program_stream():
    """The stream of the program: one for all of its calls."""
    global _stream
    if _stream is None:
        _stream = torch.cuda.Stream()
    return _stream.cuda_stream


def _lengths(case, seed):
    """Per sequence: its leader (the first of its group), the prefix it takes from it, positions of its own, rows it adds.  The
    lengths are the case's, which sequence has which the seed's."""
    n, m = case["groups"], case["members"]
    r = np.random.RandomState((n * 31 + m * 7 + case["prefix_hi"]) % (1 << 32))
    prefix = r.randint(case["prefix_lo"], case["prefix_hi"] + 1, n) | 1      # the last page is not whole
    hold = r.randint(case["hold_lo"], case["hold_hi"] + 1, n * m)
    add = r.randint(case["add_lo"], case["add_hi"] + 1, n * m)
    order = np.random.RandomState((seed * 7919 + 11) % (1 << 32)).permutation(n * m)
    return np.repeat(np.arange(n) * m, m), np.repeat(prefix, m), hold[order], add[order]


def _rounds(case, seed):
    """(have, add) of the history's two rounds and of the step: the leaders' prefixes, everybody's own positions, the step."""
    leader, prefix, hold, add = _lengths(case, seed)
    first = np.where(np.arange(len(leader)) == leader, prefix, 0)
    return [(first * 0, first), (prefix, hold), (prefix + hold, add)]


def _rows(case, seed, which, n):
    """The q|k|v rows of one round, [n][(heads + 2 kv_heads) * head_dim]: q only in the step (`which` 2)."""
    H, KVH, hd = case["heads"], case["kv_heads"], case["head_dim"]
    width = (H if which == 2 else 0) * hd
    x = torch.randn(n, width + 2 * KVH * hd, generator=_generator(seed * 3 + which + 1), device="cuda").to(TYPES[case["dtype"]])
    # columns of different size, as K and V have them
    column = torch.exp(0.5 * torch.randn(2 * KVH * hd, generator=_generator(seed * 3), device="cuda")).to(x.dtype)
    x[:, width:] *= column
    return x


def _parts(case, x):
    """K and V of rows of q|k|v, [n][kv_heads][head_dim] views."""
    KVH, hd = case["kv_heads"], case["head_dim"]
    return (x[:, -2 * KVH * hd:-KVH * hd].view(-1, KVH, hd), x[:, -KVH * hd:].view(-1, KVH, hd))


def _prepare_cache(s, case, seed):
    leader, prefix, hold, add = _lengths(case, seed)
    rounds = _rounds(case, seed)
    B = len(leader)
    ends = prefix + hold + add
    s.update(B=B, W=_pages(int(ends.max()) + 1), n=int(add.sum()), layers=case["layers"], leader=_int(leader), keep=_int(prefix),
             have=_int(rounds[2][0]), add=_int(add))
    pages = int(_pages(prefix[:: case["members"]]).sum() + (_pages(ends) - prefix // BLOCK).sum()) + 8
    if case["kind"] == "fork":
        # the last page's positions, in every sequence
        first, tail = prefix // BLOCK * BLOCK, prefix % BLOCK
        s["seq"] = _int(np.repeat(np.arange(B), tail))
        s["pos"] = _int(np.concatenate([np.arange(f, f + t) for f, t in zip(first, tail)]))
    # the history's first two rounds; a fork's case has the first one alone
    history = [(_int(h), _int(a), [_rows(case, seed + 1000 * layer, i, int(a.sum())) for layer in range(case["layers"])])
               for i, (h, a) in enumerate(rounds[:1 if case["kind"] == "fork" else 2])]
    if case["kind"] == "attend":
        s["x"] = _rows(case, seed, 2, s["n"])
    (_own_cache if own else _plain_cache)(s, case, history, pages)


def _scaling(case):
    """What stretches a model's context: by how much, the context it was trained for, the two bounds of what is left as it is."""
    return {"plain": {}, "linear": {"factor": 4.0}, "bands": {"factor": 8.0, "original": 8192, "low": 1.0, "high": 4.0},
            "yarn": {"factor": 16.0, "original": 8192, "low": 1.0, "high": 32.0}}[case["scaling"]]


def _frequencies(case):
    """Radians a position for each pair of columns, in 64 bits, and the amplitude."""
    rot, theta = case["rot"], 1000000.0
    f = theta ** (-2.0 * np.arange(rot // 2) / rot)
    p = _scaling(case)
    amplitude = 1.0
    if case["scaling"] == "linear":
        f = f / p["factor"]
    elif case["scaling"] == "bands":
        # by the turns over the trained context: below `low` stretched, above `high` not, between them in part
        share = np.clip((p["original"] * f / (2 * math.pi) - p["low"]) / (p["high"] - p["low"]), 0, 1)
        f = f / p["factor"] * (1 - share) + f * share
    elif case["scaling"] == "yarn":
        # the same between the columns at which the turns pass the bounds
        at = [rot * math.log(p["original"] / (2 * math.pi * t)) / (2 * math.log(theta)) for t in (p["high"], p["low"])]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
        share = 1 - np.clip((np.arange(rot // 2) - lo) / max(hi - lo, 0.001), 0, 1)
        f = f / p["factor"] * (1 - share) + f * share
        amplitude = 0.1 * math.log(p["factor"]) + 1
    return f, amplitude


def _prepare_rope(s, case, seed):
    H, KVH, hd, n = case["heads"], case["kv_heads"], case["head_dim"], case["rows"]
    s["x"] = torch.randn(n, (H + 2 * KVH) * hd, generator=_generator(seed), device="cuda").to(TYPES[case["dtype"]])
    s["pos"] = torch.randint(0, case["positions"], (n,), generator=_generator(seed + 1), device="cuda", dtype=torch.int32)
    f, s["amplitude"] = _frequencies(case)
    if own:
        q4hip = _library()
        freq, amplitude = q4hip.rope_frequencies(case["rot"], 1000000.0, case["scaling"], **_scaling(case))
        s["rope"] = q4hip.Rope(hd, case["rot"], case["order"], freq, amplitude)
        s["y"] = torch.empty(n, (H + KVH) * hd, dtype=s["x"].dtype, device="cuda")
        s["type"], s["stream"] = _type(case), _program_stream()
    else:
        s["freq"] = torch.from_numpy(f).cuda()


def _prepare_logits(s, case, seed):
    n, V = case["rows"], case["vocab"]
    g = _generator(seed)
    s["x"] = (3 * torch.randn(n, V, generator=g, device="cuda")).to(TYPES[case["dtype"]])
    lengths = np.random.RandomState((n * 31 + case["history_hi"]) % (1 << 32)).randint(case["history_lo"], case["history_hi"] + 1, n)
    r = np.random.RandomState((seed * 7919 + 11) % (1 << 32))
    lengths = lengths[r.permutation(n)]
    ends = np.cumsum(lengths)
    # some tokens much more often than others
    s["history"] = _int(V * np.minimum(r.random_sample(int(ends[-1])) ** 4, 0.999999)).contiguous()
    biases = case["biases"]
    tokens = r.randint(0, V, (n, biases))
    values = (2 * r.standard_normal((n, biases))).astype(np.float32)
    s["biases"] = torch.stack([_int(tokens.ravel()), _int(values.ravel().view(np.int32))], 1).contiguous()
    # a grammar's states: which tokens may come next
    states = 8 if case["masked"] else 0
    words = -(-V // 32)
    share = 0.002 * 400 ** torch.rand(states, 1, 1, generator=g, device="cuda")
    bits = torch.rand(states, words, 32, generator=g, device="cuda") < share
    s["mask"] = (bits.long() << torch.arange(32, device="cuda")).sum(2).to(torch.int32).contiguous()
    s["allowed"] = None if own else bits.view(states, words * 32)[:, :V]
    state = np.full(n, -1)
    state[r.permutation(n)[:case["masked"]]] = r.randint(0, 8, case["masked"])
    rows = np.zeros((n, 8), np.int32)
    rows[:, 0] = (1 + 0.3 * r.random_sample(n)).astype(np.float32).view(np.int32)      # repetition
    rows[:, 1] = (r.random_sample(n) * (r.random_sample(n) < 0.5)).astype(np.float32).view(np.int32)
    rows[:, 2] = (0.5 * r.random_sample(n) * (r.random_sample(n) < 0.5)).astype(np.float32).view(np.int32)
    rows[:, 3], rows[:, 4] = ends - lengths, ends
    rows[:, 5], rows[:, 6] = np.arange(n) * biases, (np.arange(n) + 1) * biases
    rows[:, 7] = state
    s["rows"] = _int(rows)
    if own:
        s["logits"] = _library().Logits(V, n)
        s["y"], s["best"] = torch.empty_like(s["x"]), torch.empty(n, dtype=torch.int32, device="cuda")
        s["type"], s["stream"] = _type(case), _program_stream()


def prepare(case, seed):
    s = {"case": case, "kind": case["kind"]}
    {"rope": _prepare_rope, "logits": _prepare_logits}.get(case["kind"], _prepare_cache)(s, case, seed)
    return s


# ---------------------------------------------------------------------------- the library's operators

def _library():
    at = os.path.join(REPO, "e2e-browser-voice-agent_amd", "py")
    if at not in sys.path:
        sys.path.insert(0, at)
    import q4hip
    return q4hip


def _type(case):
    q4hip = _library()
    return {"f32": q4hip.F32, "f16": q4hip.F16, "bf16": q4hip.BF16}[case["dtype"]]


def _own_cache(s, case, history, pages):
    H, KVH, hd, B, W = case["heads"], case["kv_heads"], case["head_dim"], s["B"], s["W"]
    rows = max([s["n"]] + [x[0].shape[0] for _, _, x in history] + [1])
    kv = _library().Kv8(layers=s["layers"], heads=H, kv_heads=KVH, head_dim=hd, seqs=B, max_len=W * BLOCK, pages=pages, max_rows=rows)
    s["kv"], s["type"], s["stream"] = kv, _type(case), _program_stream()
    torch.cuda.synchronize()         # calls without a stream run on the handle's own
    for i, (have, add, x) in enumerate(history):
        if i == 1:
            kv.fork(s["leader"].data_ptr(), s["keep"].data_ptr())
        kv.plan(have.data_ptr(), add.data_ptr(), x[0].shape[0])
        for layer, y in enumerate(x):
            if y.shape[0]:
                k, v = _parts(case, y)
                kv.append(layer, k.data_ptr(), v.data_ptr(), s["type"], y.shape[1], y.shape[1])
    if s["kind"] == "fork":
        s["tables"] = torch.empty(B, W, dtype=torch.int32, device="cuda")
        s["k"], s["v"] = (torch.empty(s["layers"], s["seq"].shape[0], KVH, hd, device="cuda") for _ in range(2))
    else:
        s["out"] = torch.empty(s["n"], H * hd, dtype=TYPES[case["dtype"]], device="cuda")
        kv.plan(s["have"].data_ptr(), s["add"].data_ptr(), s["n"])
        k, v = _parts(case, s["x"])
        kv.append(0, k.data_ptr(), v.data_ptr(), s["type"], s["x"].shape[1], s["x"].shape[1])


def _run_own(s):
    case, kind, stream = s["case"], s["kind"], s["stream"]
    if kind == "fork":
        kv, n = s["kv"], s["seq"].shape[0]
        kv.fork(s["leader"].data_ptr(), s["keep"].data_ptr(), s["tables"].data_ptr(), stream)
        for layer in range(s["layers"]):
            kv.read(layer, s["seq"].data_ptr(), s["pos"].data_ptr(), n, s["k"][layer].data_ptr(), s["v"][layer].data_ptr(), stream)
        return {"tables": s["tables"], "k": s["k"], "v": s["v"]}
    if kind == "attend":
        s["kv"].attend(0, s["x"].data_ptr(), s["out"].data_ptr(), s["type"], s["x"].shape[1], s["out"].shape[1], stream)
        return {"out": s["out"]}
    if kind == "rope":
        s["rope"].run(s["x"].data_ptr(), s["y"].data_ptr(), case["heads"] + case["kv_heads"], s["type"], s["x"].shape[1], s["y"].shape[1],
                      s["pos"].data_ptr(), case["rows"], stream=stream)
        return {"y": s["y"]}
    V = case["vocab"]
    s["logits"].run(s["x"].data_ptr(), s["y"].data_ptr(), s["type"], V, V, case["rows"], s["rows"].data_ptr(),
                    history=s["history"].data_ptr(), history_n=s["history"].shape[0], biases=s["biases"].data_ptr(),
                    biases_n=s["biases"].shape[0], mask=s["mask"].data_ptr(), mask_rows=s["mask"].shape[0], best=s["best"].data_ptr(),
                    stream=stream)
    return {"y": s["y"], "best": s["best"]}


# ---------------------------------------------------------------------------- the plain forms

def _plain_cache(s, case, history, pages):
    B, W, KVH, hd = s["B"], s["W"], case["kv_heads"], case["head_dim"]
    pool = {"tables": torch.full((B, W), -1, dtype=torch.int32, device="cuda"),
            "stack": torch.arange(pages - 1, -1, -1, dtype=torch.int32, device="cuda")}
    s["codes"] = [torch.zeros(s["layers"], pages, KVH, BLOCK, hd, dtype=torch.int8, device="cuda") for _ in range(2)]
    s["scales"] = [torch.zeros(s["layers"], pages, KVH, device="cuda") for _ in range(2)]
    for i, (have, add, x) in enumerate(history):
        if i == 1:
            pool = _plain_fork(s, pool)
        pool, slots = _plain_plan(pool, have, add)
        for layer, y in enumerate(x):
            if y.shape[0]:
                for c, sc, z in zip(s["codes"], s["scales"], _parts(case, y)):
                    _plain_append(c[layer], sc[layer], z, slots)
    if s["kind"] == "attend":
        pool, slots = _plain_plan(pool, s["have"], s["add"])
        for c, sc, z in zip(s["codes"], s["scales"], _parts(case, s["x"])):
            _plain_append(c[0], sc[0], z, slots)
        s["shape"] = [int(v) for v in (s["add"].max(), (s["keep"] // BLOCK).max(),
                                       ((s["have"] + s["add"] + BLOCK - 1) // BLOCK - s["keep"] // BLOCK).max())]
    s["pool"] = pool


def _plain_plan(pool, have, add):
    """The pool with the pages that a step takes, and its rows' slots.  (No sequence gives any back.)"""
    tables = pool["tables"].clone()
    need = ((have + add + BLOCK - 1) // BLOCK)[:, None]
    take = (tables < 0) & (torch.arange(tables.shape[1], device="cuda")[None, :] < need)
    n = int(take.sum())
    tables[take] = pool["stack"].flip(0)[:n]
    start = torch.cumsum(add, 0) - add
    seq = torch.repeat_interleave(torch.arange(add.shape[0], device="cuda"), add.long())
    pos = torch.arange(seq.shape[0], device="cuda") - start[seq] + have[seq]
    return {"tables": tables, "stack": pool["stack"][:pool["stack"].shape[0] - n]}, tables[seq, pos // BLOCK].long() * BLOCK + pos % BLOCK


def _plain_fork(s, pool):
    keep, B = s["keep"].long(), s["B"]
    pages = s["codes"][0].shape[1]
    column = torch.arange(pool["tables"].shape[1], device="cuda")[None, :]
    tables = torch.where(column * BLOCK < keep[:, None], pool["tables"][s["leader"].long()], -1)
    whole = column < (keep // BLOCK)[:, None]
    held = torch.zeros(pages, dtype=torch.bool, device="cuda")
    held[tables[tables >= 0].long()] = True
    # who keeps a last page that is not whole: its first holder, or nobody where it is another one's whole page
    seqs = torch.arange(B, device="cuda")
    last = tables.gather(1, (keep // BLOCK).clamp(max=tables.shape[1] - 1)[:, None])[:, 0].long()
    part = keep % BLOCK > 0
    keeper = torch.full((pages,), B, device="cuda").scatter_reduce(0, last[part], seqs[part], "amin")
    keeper[tables[whole].long()] = -1
    copies = part & (keeper[last.clamp(min=0)] != seqs)
    free = torch.nonzero(~held)[:, 0]
    n = int(copies.sum())
    to, source = free[:n], last[copies]
    for c in s["codes"] + s["scales"]:
        c[:, to] = c[:, source]
    tables[copies, keep[copies] // BLOCK] = to.to(torch.int32)
    return {"tables": tables, "stack": free[n:].flip(0).to(torch.int32)}


def _pow2(k):
    """2^k in fp32 for whole k, exactly."""
    return ((k.clamp(-126, 127) + 127) << 23).to(torch.int32).view(torch.float32)


def _plain_append(codes, scales, x, slots):
    """Rows x [n][kv_heads][head_dim] into codes [page][head][32][head_dim] and scales [page][head], in place."""
    x = x.float()
    page, off = slots // BLOCK, slots % BLOCK
    block, at = torch.unique(page, return_inverse=True)
    U, KVH = block.shape[0], x.shape[1]
    first = torch.full((U,), BLOCK, dtype=torch.int64, device="cuda").scatter_reduce(0, at, off, "amin")
    most = torch.zeros(U, KVH, device="cuda").scatter_reduce(0, at[:, None].expand(-1, KVH), x.abs().amax(2), "amax")
    t = most / torch.full_like(most, 127)      # a quotient, where a number on the right would be a product
    old = torch.where(first[:, None] > 0, scales[block], torch.zeros_like(t))
    # the smallest power of two with old * 2^k >= t
    (mt, et), (mo, eo) = torch.frexp(t), torch.frexp(old)
    k = torch.where((old > 0) & (t > old), et - eo + (mt > mo).int(), torch.zeros_like(et))
    s = torch.where(old > 0, old * _pow2(k), t)
    kept = codes[block].float()
    halved = torch.round(kept * _pow2(-k)[:, :, None, None])
    before = torch.arange(BLOCK, device="cuda")[None, None, :, None] < first[:, None, None, None]
    codes[block] = torch.where(before, halved, kept).to(torch.int8)
    sx = s[at][:, :, None]
    q = torch.where(sx > 0, torch.round(x / sx), torch.zeros_like(x)).clamp(-127, 127)
    codes[page, :, off] = q.to(torch.int8)
    scales[block] = s


def _values(s, which, pages):
    """[n][kv_heads][positions][head_dim] in fp32 of pages [n][pages]."""
    page = pages.clamp(min=0).long()
    x = s["codes"][which][0][page].float() * s["scales"][which][0][page][:, :, :, None, None]
    return x.transpose(1, 2).flatten(2, 3).contiguous()


def _plain_attend(s):
    """Scores of the prefix for all members of a group at once, of the rest sequence by sequence, in one softmax."""
    case, tables = s["case"], s["pool"]["tables"]
    H, KVH, hd, n, m = case["heads"], case["kv_heads"], case["head_dim"], case["groups"], case["members"]
    B, G, (A, C, S) = s["B"], H // KVH, s["shape"]
    common = s["keep"] // BLOCK                                             # pages of a prefix
    seq = torch.repeat_interleave(torch.arange(B, device="cuda"), s["add"].long(), output_size=s["n"])
    start = torch.cumsum(s["add"], 0) - s["add"]
    row = torch.arange(s["n"], device="cuda") - start[seq]
    q = torch.zeros(B, A, H * hd, device="cuda")
    q[seq, row] = s["x"][:, :H * hd].float()
    q = q.view(B, A, KVH, G, hd).permute(0, 2, 3, 1, 4).reshape(B, KVH, G * A, hd) / math.sqrt(hd)
    q_group = q.view(n, m, KVH, G * A, hd).transpose(1, 2).reshape(n, KVH, m * G * A, hd)
    keys, vals = (_values(s, w, tables[::m, :C]) for w in range(2))
    first = torch.matmul(q_group, keys.transpose(2, 3))
    first.masked_fill_(torch.arange(C * BLOCK, device="cuda") >= common[::m, None, None, None] * BLOCK, -math.inf)
    column = common[:, None] + torch.arange(S, device="cuda")
    rest = tables.gather(1, column.clamp(max=s["W"] - 1))
    own_keys, own_vals = (_values(s, w, rest) for w in range(2))
    second = torch.matmul(q, own_keys.transpose(2, 3)).view(B, KVH, G, A, S * BLOCK)
    last = s["have"][:, None] + torch.arange(A, device="cuda") - common[:, None] * BLOCK       # the row's own position
    second.masked_fill_(torch.arange(S * BLOCK, device="cuda") > last[:, None, None, :, None], -math.inf)
    second = second.view(B, KVH, G * A, S * BLOCK)

    def by_group(x):
        return x.view(n, m, KVH, G * A, -1).transpose(1, 2).reshape(n, KVH, m * G * A, -1)

    def by_seq(x):
        return x.view(n, KVH, m, G * A, -1).transpose(1, 2).reshape(B, KVH, G * A, -1)

    top = torch.maximum(by_seq(first.amax(3)), second.amax(3, keepdim=True))
    first = torch.exp(first - by_group(top))
    second = torch.exp(second - top)
    total = by_seq(first.sum(3)) + second.sum(3, keepdim=True)
    out = (by_seq(torch.matmul(first, vals)) + torch.matmul(second, own_vals)) / total
    out = out.view(B, KVH, G, A, hd).permute(0, 3, 1, 2, 4).reshape(B, A, H * hd)
    return out[seq, row].to(TYPES[case["dtype"]])


def _plain_rope(s):
    case = s["case"]
    hd, rot, n, heads = case["head_dim"], case["rot"], case["rows"], case["heads"] + case["kv_heads"]
    x = s["x"][:, :heads * hd].view(n, heads, hd).float()
    angle = s["pos"].double()[:, None, None] * s["freq"]
    cos, sin = (s["amplitude"] * torch.cos(angle)).float(), (s["amplitude"] * torch.sin(angle)).float()
    if case["order"] == "halves":
        a, b = x[:, :, :rot // 2], x[:, :, rot // 2:rot]
    else:
        a, b = x[:, :, :rot:2], x[:, :, 1:rot:2]
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat([u, v], 2) if case["order"] == "halves" else torch.stack([u, v], 3).flatten(2)
    return torch.cat([turned, x[:, :, rot:]], 2).view(n, heads * hd).to(s["x"].dtype)


def _plain_logits(s):
    n, V = s["case"]["rows"], s["case"]["vocab"]
    rows, history, biases = s["rows"], s["history"], s["biases"]
    repetition, presence, frequency = (rows[:, i:i + 1].contiguous().view(torch.float32) for i in range(3))
    of = torch.repeat_interleave(torch.arange(n, device="cuda"), (rows[:, 4] - rows[:, 3]).long(), output_size=history.shape[0])
    count = torch.zeros(n * V, device="cuda").index_add_(0, of * V + history, torch.ones(history.shape[0], device="cuda")).view(n, V)
    x = s["x"].float()
    x = torch.where(count > 0, torch.where(x > 0, x / repetition, x * repetition) - (frequency * count + presence), x)
    of = torch.repeat_interleave(torch.arange(n, device="cuda"), (rows[:, 6] - rows[:, 5]).long(), output_size=biases.shape[0])
    at = of * V + biases[:, 0]
    entry = torch.arange(biases.shape[0], device="cuda")
    last = torch.full((n * V,), -1, device="cuda").scatter_reduce(0, at, entry, "amax")[at] == entry
    bias = torch.zeros(n * V, device="cuda")
    bias[at[last]] = biases[:, 1].contiguous().view(torch.float32)[last]
    x = x + bias.view(n, V)
    if s["allowed"].shape[0]:
        state = rows[:, 7].long()
        x = torch.where(s["allowed"][state.clamp(min=0)] | (state < 0)[:, None], x, -math.inf)
    best = torch.where(x == x.amax(1, keepdim=True), torch.arange(V, device="cuda"), V).amin(1).to(torch.int32)
    return {"y": x.to(s["x"].dtype), "best": best}


def _run_plain(s):
    if s["kind"] == "fork":
        tables = _plain_fork(s, s["pool"])["tables"]
        page = tables[s["seq"].long(), (s["pos"] // BLOCK).long()].long()
        k, v = (c[:, page, :, (s["pos"] % BLOCK).long()].transpose(0, 1).float() * sc[:, page][..., None]
                for c, sc in zip(s["codes"], s["scales"]))
        return {"tables": tables, "k": k, "v": v}
    if s["kind"] == "attend":
        return {"out": _plain_attend(s)}
    return {"y": _plain_rope(s)} if s["kind"] == "rope" else _plain_logits(s)


def run(state):
    return (_run_own if own else _run_plain)(state)


# ---------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    """Means over the lengths that a case's seeds give."""
    es = 4 if case["dtype"] == "f32" else 2
    kind = case["kind"]
    if kind == "logits":
        n, V = case["rows"], case["vocab"]
        history = n * (case["history_lo"] + case["history_hi"]) / 2
        mask = (min(8, case["masked"]) * V / 8)
        return {"bytes": 2 * n * V * es + 4 * history + 8 * n * case["biases"] + mask + 36 * n, "flops": n * V + 4 * history}
    H, KVH, hd = case["heads"], case["kv_heads"], case["head_dim"]
    if kind == "rope":
        n = case["rows"]
        return {"bytes": n * (2 * (H + KVH) * hd * es + 4), "flops": 3 * n * (H + KVH) * case["rot"]}
    n, B = case["groups"], case["groups"] * case["members"]
    row = KVH * hd
    prefix = (case["prefix_lo"] + case["prefix_hi"]) / 2
    if kind == "fork":
        read = B * BLOCK / 2 * case["layers"] * 2 * row
        copied = (B - n) * case["layers"] * 2 * (BLOCK * row + 4 * KVH)
        tables = 4 * B * prefix / BLOCK
        return {"bytes": 2 * copied + 2 * tables + 8 * B + 5 * read, "flops": read}
    hold, add = (case["hold_lo"] + case["hold_hi"]) / 2, (case["add_lo"] + case["add_hi"]) / 2
    cached = n * prefix + B * (hold + add)
    return {"bytes": 2 * cached * row + 8 * cached / BLOCK * KVH + 2 * B * add * H * hd * es,
            "flops": 4 * H * hd * B * add * (prefix + hold + (add + 1) / 2)}


# ---------------------------------------------------------------------------- the same in 64 bits

def _exact_blocks(chunks):
    """The values that one sequence's cache stands for in 64 bits, [positions][heads][dims]: chunks (position, values)
    in the order of the appends.  Scales are fp32 numbers, codes the roundings of fp32 quotients."""
    codes = scales = None
    for p0, x in chunks:
        x = x.double()
        n, KVH, hd = x.shape
        if codes is None:
            codes, scales = torch.zeros(0, BLOCK, KVH, hd, dtype=torch.float64, device="cuda"), torch.zeros(0, KVH, dtype=torch.float64, device="cuda")
        if n == 0:
            continue
        b0, f, b1 = p0 // BLOCK, p0 % BLOCK, _pages(p0 + n)
        part = torch.zeros((b1 - b0) * BLOCK, KVH, hd, dtype=torch.float64, device="cuda")
        part[f:f + n] = x
        part = part.view(b1 - b0, BLOCK, KVH, hd)
        s = part.abs().amax((1, 3))
        s = (s / torch.full_like(s, 127)).float().double()
        head = None
        if f:
            old = scales[b0]
            ratio = torch.where(old > 0, s[0] / old.clamp(min=1e-300), torch.zeros_like(old))
            twice = torch.ones_like(ratio)             # 2^k
            while bool((twice < ratio).any()):
                twice = torch.where(twice < ratio, 2 * twice, twice)
            s[0] = torch.where(old > 0, old * twice, s[0])
            head = torch.round(codes[b0, :f] / twice[None, :, None])
        d = s[:, None, :, None]
        q = torch.where(d > 0, torch.round((part / d).float().double()), part * 0).clamp(-127, 127)
        if f:
            q[0, :f] = head
        codes, scales = torch.cat([codes[:b0], q]), torch.cat([scales[:b0], s])
    return (codes * scales[:, None, :, None]).view(-1, codes.shape[2], codes.shape[3])


def _exact_fork(case, seed):
    leader, prefix, _, _ = _lengths(case, seed)
    _, first = _rounds(case, seed)[0]
    at = np.concatenate([[0], np.cumsum(first)])
    found = [[], []]
    for layer in range(case["layers"]):
        rows = _rows(case, seed + 1000 * layer, 0, int(first.sum()))
        for w in range(2):
            tails = {b: _exact_blocks([(0, _parts(case, rows[at[b]:at[b + 1]])[w])])[prefix[b] // BLOCK * BLOCK:prefix[b]]
                     for b in sorted(set(leader.tolist()))}
            found[w].append(torch.cat([tails[b] for b in leader.tolist()]))
    return {"tables": None, "k": torch.stack(found[0]), "v": torch.stack(found[1])}


def _exact_attend(case, seed):
    H, KVH, hd = case["heads"], case["kv_heads"], case["head_dim"]
    G = H // KVH
    leader, prefix, _, _ = _lengths(case, seed)
    rounds = _rounds(case, seed)
    rows = [_rows(case, seed, i, int(a.sum())) for i, (_, a) in enumerate(rounds)]
    at = [np.concatenate([[0], np.cumsum(a)]) for _, a in rounds]
    outs, common = [], {}
    for b in range(len(leader)):
        g, P = int(leader[b]), int(prefix[b])
        h0, n = int(rounds[2][0][b]), int(rounds[2][1][b])
        whole, values = P // BLOCK * BLOCK, []
        for w in range(2):
            if (g, w) not in common:
                common[g, w] = _exact_blocks([(0, _parts(case, rows[0][at[0][g]:at[0][g] + whole])[w])])
            # the last page as the leader left it, then the sequence's own rows
            chunks = [(0, rows[0][at[0][g] + whole:at[0][g] + P]), (P - whole, rows[1][at[1][b]:at[1][b + 1]]),
                      (h0 - whole, rows[2][at[2][b]:at[2][b + 1]])]
            values.append(torch.cat([common[g, w], _exact_blocks([(p, _parts(case, x)[w]) for p, x in chunks])])[:h0 + n].transpose(0, 1))
        q = rows[2][at[2][b]:at[2][b + 1], :H * hd].double().view(n, KVH, G, hd).permute(1, 0, 2, 3).reshape(KVH, n * G, hd)
        score = torch.bmm(q, values[0].transpose(1, 2).contiguous()) * hd ** -0.5
        pos = torch.arange(h0, h0 + n, device="cuda").repeat_interleave(G)
        score = torch.where(torch.arange(h0 + n, device="cuda")[None, :] <= pos[:, None], score, score.new_full((), -math.inf))
        out = torch.bmm(torch.softmax(score, 2), values[1].contiguous())
        outs.append(out.view(KVH, n, G, hd).permute(1, 0, 2, 3).reshape(n, H * hd))
    return {"out": torch.cat(outs)}


def _exact_rope(case, seed):
    s = {}
    _prepare_rope(s, case, seed)
    hd, rot, n, heads = case["head_dim"], case["rot"], case["rows"], case["heads"] + case["kv_heads"]
    freq, amplitude = _frequencies(case)
    y = s["x"][:, :heads * hd].double().view(n, heads, hd).clone()
    angle = torch.outer(s["pos"].double(), torch.from_numpy(freq).cuda())[:, None, :]
    turn = torch.polar(torch.full_like(angle, amplitude), angle)
    first, second = (slice(0, rot // 2), slice(rot // 2, rot)) if case["order"] == "halves" else (slice(0, rot, 2), slice(1, rot, 2))
    z = torch.complex(y[:, :, first].contiguous(), y[:, :, second].contiguous()) * turn
    y[:, :, first], y[:, :, second] = z.real, z.imag
    return {"y": y.view(n, heads * hd)}


def _exact_logits(case, seed):
    s = {}
    _prepare_logits(s, case, seed)
    y = s["x"].double()
    params = s["rows"].cpu().numpy()
    history, biases = s["history"].cpu().numpy(), s["biases"].cpu().numpy()
    words = s["mask"].cpu().numpy().view(np.uint32)
    for r in range(case["rows"]):
        repetition, presence, frequency = (float(v) for v in params[r, :3].view(np.float32))
        tokens, counts = np.unique(history[params[r, 3]:params[r, 4]], return_counts=True)
        at, c = torch.from_numpy(tokens).long().cuda(), torch.from_numpy(counts).double().cuda()
        x = y[r, at]
        y[r, at] = torch.where(x > 0, x / repetition, x * repetition) - (frequency * c + presence)
        own_biases = dict(zip(biases[params[r, 5]:params[r, 6], 0].tolist(), biases[params[r, 5]:params[r, 6], 1].view(np.float32).tolist()))
        if own_biases:
            at = torch.tensor(list(own_biases), device="cuda")
            y[r, at] += torch.tensor(list(own_biases.values()), dtype=torch.float64, device="cuda")
        if params[r, 7] >= 0:
            bits = np.unpackbits(words[params[r, 7]].view(np.uint8), bitorder="little")[:case["vocab"]]
            y[r, torch.from_numpy(bits == 0).cuda()] = -math.inf
    return {"y": y, "best": None}


def exact(case, seed):
    return {"fork": _exact_fork, "attend": _exact_attend, "rope": _exact_rope, "logits": _exact_logits}[case["kind"]](case, seed)
