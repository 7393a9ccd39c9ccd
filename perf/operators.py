"""The calls that a program makes on the paged 8-bit K/V cache, as cases to be timed and compared.

The cache holds K and V in int8, in pages of 32 positions.  Each page has one fp32 scale per kv head for K
and one for V.  A case is a call at one size.  Its kinds:

  plan     the step's rows from request lengths: block tables, starts, positions, slots
  append   K and V rows of the step into the cache; what its blocks then stand for is read back
  attend   attention of the step's rows over the cache
  step     the three as one step of a layer

A state has a history: every sequence was appended to in two rounds (half of its positions each), so that its
pages lie between those of the others.  Then comes the step: sequence b holds have[b] positions and adds add[b].

What the operators compute:

  plan     sequence b needs ceil((have + add) / 32) pages.  Pages beyond that go back to the pool's stack, sequence by
           sequence; then the sequences take what they lack from the top of the stack, in the same order.  Row t of the
           step is position have[b] + t - starts[b] of its sequence, its slot 32 * page + position % 32.
  append   a run of rows in one block, the first at offset f; t = max|x| / 127 of a head's values.  At f = 0 the
           scale is t, else the old scale times the smallest power of two that reaches t, and the codes
           before f are halved (to the nearest even) as often.  The codes are x / scale, rounded to nearest even.
  attend   softmax(q . K * head_dim^-1/2) V over the positions up to the row's own
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


def _case(kind, layout, dtype, seqs, hold, prompts=0, add=(1, 1), done=0, name=None):
    """`seqs` sequences that hold hold[0]..hold[1] positions: the first `done` have ended, the next `prompts` add
    add[0]..add[1] rows each, the others add one row."""
    H, KVH, hd = layout
    case = {"kind": kind, "heads": H, "kv_heads": KVH, "head_dim": hd, "dtype": dtype, "seqs": seqs, "hold_lo": hold[0],
            "hold_hi": hold[1], "prompts": prompts, "add_lo": add[0], "add_hi": add[1], "done": done}
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # the next token of 32 chats: the smallest plan, once for all layers of a step
        _case("plan", LAYOUTS[0], "f32", 32, (90, 420), name="plan_chats"),
        # a busy server: 1024 sequences, some of them ended, some with a prompt to run
        _case("plan", LAYOUTS[2], "bf16", 1024, (0, 4000), 24, (200, 1000), 40, name="plan_server"),
        # one token of each of 7 chats, as the 0.5B shape's q|k|v rows hold them
        _case("append", LAYOUTS[0], "f32", 7, (90, 420), name="append_tokens_05b"),
        # 8 documents at once
        _case("append", LAYOUTS[2], "bf16", 8, (0, 100), 8, (1000, 3000), name="append_prompts"),
        # the next token of one chat: the smallest attention
        _case("attend", LAYOUTS[0], "f32", 1, (300, 300), name="token_05b"),
        # the next token after a very long text
        _case("attend", LAYOUTS[0], "f16", 1, (131072, 131072), name="token_long_05b"),
        # a full server of the larger model
        _case("attend", LAYOUTS[1], "f32", 32, (1024, 1024), name="batch_15b"),
        # 64 long chats of very different lengths: a gigabyte of cache
        _case("attend", LAYOUTS[2], "bf16", 64, (2000, 16000), name="batch_long"),
        # a spoken sentence appended to a running chat
        _case("attend", LAYOUTS[0], "f32", 1, (220, 220), 1, (23, 23), name="turn_05b"),
        # a whole document as the prompt: the engine's largest pass
        _case("attend", LAYOUTS[0], "f32", 1, (0, 0), 1, (1024, 1024), name="prompt_05b_1024"),
        # a long document
        _case("attend", LAYOUTS[2], "bf16", 1, (0, 0), 1, (8192, 8192), name="prompt_long"),
        # a step of a server: 4 prompts beside 44 chats, a kv head for each query head
        _case("step", LAYOUTS[3], "f16", 48, (0, 2000), 4, (100, 900), name="step_mixed"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm, odd half of the time."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, v | 1 if rng.random() < 0.5 else v))


def draw(rng):
    kind = rng.choice(["plan", "append", "attend", "attend", "attend", "step"])
    layout, dtype = rng.choice(LAYOUTS), rng.choice(sorted(TYPES))
    row = layout[1] * layout[2]
    if kind == "plan":
        seqs = _log(rng, 1, 1024)
        hi = _log(rng, 8, 4000)
        return _case(kind, layout, dtype, seqs, (0, hi), min(seqs, rng.randint(0, 24)), (1, _log(rng, 8, 1000)),
                     rng.randint(0, seqs // 8))
    if kind == "append":
        if rng.random() < 0.5:           # tokens
            return _case(kind, layout, dtype, _log(rng, 1, 256), (0, _log(rng, 8, 1000)))
        seqs = _log(rng, 1, 8)
        hi = _log(rng, 40, 3000)
        return _case(kind, layout, dtype, seqs, (0, 100), seqs, (max(2, hi // 3), hi))
    if kind == "attend" and rng.random() < 0.4:
        n = _log(rng, 2, 4096)           # a prompt, or a part of one
        return _case(kind, layout, dtype, 1, (0, _log(rng, 8, 4000)) if rng.random() < 0.5 else (0, 0), 1, (n, n))
    seqs = _log(rng, 1, 64 if kind == "attend" else 256)
    hi = min(_log(rng, 16, 131072), 400000000 // (row * seqs), 4000 if kind == "step" else 131072)
    lo = 0 if rng.random() < 0.3 else hi // 2
    prompts = min(seqs, rng.randint(1, 4)) if kind == "step" or rng.random() < 0.3 else 0
    if prompts:
        lo, hi = min(lo, 2000), min(hi, 4000)
    return _case(kind, layout, dtype, seqs, (lo, max(hi, 1)), prompts, (2, _log(rng, 4, 900)))


# ---------------------------------------------------------------------------- inputs

def _lengths(case, seed):
    """(held, have, add): positions of every sequence's history, positions it holds before the step, rows it adds.  The
    lengths are the case's, which sequence has which the seed's."""
    B, done, prompts = case["seqs"], case["done"], case["prompts"]
    r = np.random.RandomState((B * 31 + case["hold_hi"] * 7 + case["add_hi"]) % (1 << 32))
    held = r.randint(case["hold_lo"], case["hold_hi"] + 1, B)
    have, add = held.copy(), np.ones(B, dtype=np.int64)
    have[:done], add[:done] = 0, 0
    n = min(prompts, B - done)
    add[done:done + n] = r.randint(case["add_lo"], case["add_hi"] + 1, n)
    order = np.random.RandomState((seed * 7919 + 11) % (1 << 32)).permutation(B)
    return held[order], have[order], add[order]


def _rounds(case, seed):
    """(have, add) of the two rounds of the history and of the step."""
    held, have, add = _lengths(case, seed)
    half = held // 2
    return [(held * 0, half), (half, held - half), (have, add)]


def _rows(case, seed, which, n):
    """The q|k|v rows of one round, [n][(heads + 2 kv_heads) * head_dim]: q only in the step (`which` 2)."""
    H, KVH, hd = case["heads"], case["kv_heads"], case["head_dim"]
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 3 + which + 1)
    width = (H if which == 2 else 0) * hd
    x = torch.randn(n, width + 2 * KVH * hd, generator=g, device="cuda", dtype=torch.float32).to(TYPES[case["dtype"]])
    c = torch.Generator(device="cuda")
    c.manual_seed(seed * 3)
    # columns of different size, as K and V have them
    column = torch.exp(0.5 * torch.randn(2 * KVH * hd, generator=c, device="cuda")).to(x.dtype)
    x[:, width:] *= column
    return x


def _parts(case, x):
    """K and V of rows of q|k|v, [n][kv_heads][head_dim] views."""
    KVH, hd = case["kv_heads"], case["head_dim"]
    n = x.shape[0]
    return x[:, -2 * KVH * hd:-KVH * hd].view(n, KVH, hd), x[:, -KVH * hd:].view(n, KVH, hd)


def _width(case):
    """Pages of the longest sequence that the case can have."""
    return max(1, _pages(case["hold_hi"] + max(case["add_hi"], 1)))


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


def prepare(case, seed):
    H, KVH, hd = case["heads"], case["kv_heads"], case["head_dim"]
    B, rounds = case["seqs"], _rounds(case, seed)
    W = _width(case)
    pages = int(sum(_pages(np.maximum(rounds[1][0] + rounds[1][1], rounds[2][0] + rounds[2][1])))) + 8
    have, add = rounds[2]
    n = int(add.sum())
    # the rows whose values an append changes: those of the blocks that it writes to, up to the last one
    seq, pos = [], []
    for b in range(B):
        if add[b]:
            p = np.arange(have[b] // BLOCK * BLOCK, have[b] + add[b])
            seq.append(np.full(len(p), b))
            pos.append(p)
    seq, pos = np.concatenate(seq), np.concatenate(pos)
    s = {"case": case, "kind": case["kind"], "B": B, "W": W, "n": n, "have": _int(have), "add": _int(add),
         "have_list": have.tolist(), "add_list": add.tolist(), "seq": _int(seq), "pos": _int(pos), "x": _rows(case, seed, 2, n)}
    (_own_state if own else _plain_state)(s, seed, rounds, pages)
    return s


def _history(case, seed, rounds):
    if case["kind"] == "plan":
        return [(h, a, None) for h, a in rounds[:2]]
    return [(h, a, _rows(case, seed, i, int(a.sum()))) for i, (h, a) in enumerate(rounds[:2])]


# ---------------------------------------------------------------------------- the library's operators

def _own_state(s, seed, rounds, pages):
    sys.path.insert(0, os.path.join(REPO, "e2e-browser-voice-agent_amd", "py"))
    import q4hip
    case, B, W, n = s["case"], s["B"], s["W"], s["n"]
    H, KVH, hd = case["heads"], case["kv_heads"], case["head_dim"]
    most = max(int(a.sum()) for _, a in rounds)
    kv = q4hip.Kv8(layers=1, heads=H, kv_heads=KVH, head_dim=hd, seqs=B, max_len=W * BLOCK, pages=pages, max_rows=max(most, 1))
    s["kv"], s["type"] = kv, {"f32": q4hip.F32, "f16": q4hip.F16, "bf16": q4hip.BF16}[case["dtype"]]
    s["stream"] = _program_stream()
    history = _history(case, seed, rounds)
    torch.cuda.synchronize()         # calls without a stream run on the handle's own
    for h, a, x in history:
        before, more = _int(h), _int(a)
        kv.plan(before.data_ptr(), more.data_ptr(), int(a.sum()))
        if x is not None and x.shape[0]:
            k, v = _parts(case, x)
            kv.append(0, k.data_ptr(), v.data_ptr(), s["type"], x.shape[1], x.shape[1])
    for name, shape in (("starts", (B + 1,)), ("positions", (n,)), ("slots", (n,)), ("tables", (B, W))):
        s[name] = torch.empty(shape, dtype=torch.int32, device="cuda")
    m = s["seq"].shape[0]
    if s["kind"] == "append":
        s["k"], s["v"] = (torch.empty(m, KVH, hd, device="cuda") for _ in range(2))
    s["out"] = torch.empty(n, H * hd, dtype=TYPES[case["dtype"]], device="cuda")
    if s["kind"] in ("append", "attend"):
        kv.plan(s["have"].data_ptr(), s["add"].data_ptr(), n)
    if s["kind"] == "attend":
        _own_append(s, 0)


def _own_append(s, stream):
    k, v = _parts(s["case"], s["x"])
    width = s["x"].shape[1]
    s["kv"].append(0, k.data_ptr(), v.data_ptr(), s["type"], width, width, stream)


def _run_own(s):
    kv, kind, stream, n = s["kv"], s["kind"], s["stream"], s["n"]
    got = {}
    if kind in ("plan", "step"):
        kv.plan(s["have"].data_ptr(), s["add"].data_ptr(), n, s["starts"].data_ptr(), s["positions"].data_ptr(),
                s["slots"].data_ptr(), s["tables"].data_ptr(), stream)
        got = {name: s[name] for name in ("starts", "positions", "slots", "tables")}
    if kind in ("append", "step"):
        _own_append(s, stream)
    if kind == "append":
        kv.read(0, s["seq"].data_ptr(), s["pos"].data_ptr(), s["seq"].shape[0], s["k"].data_ptr(), s["v"].data_ptr(), stream)
        got = {"k": s["k"], "v": s["v"]}
    if kind in ("attend", "step"):
        kv.attend(0, s["x"].data_ptr(), s["out"].data_ptr(), s["type"], s["x"].shape[1], s["out"].shape[1], stream)
        got["out"] = s["out"]
    return got


# ---------------------------------------------------------------------------- the plain forms

def _plain_state(s, seed, rounds, pages):
    case, B, W = s["case"], s["B"], s["W"]
    KVH, hd = case["kv_heads"], case["head_dim"]
    pool = {"tables": torch.full((B, W), -1, dtype=torch.int32, device="cuda"),
            "held": torch.zeros(B, dtype=torch.int64, device="cuda"),
            "stack": torch.arange(pages - 1, -1, -1, dtype=torch.int32, device="cuda")}
    size = 0 if case["kind"] == "plan" else pages
    s["codes"] = [torch.zeros(size, KVH, BLOCK, hd, dtype=torch.int8, device="cuda") for _ in range(2)]
    s["scales"] = [torch.zeros(size, KVH, device="cuda") for _ in range(2)]
    for h, a, x in _history(case, seed, rounds):
        step, pool = _plain_plan(pool, _int(h), _int(a))
        if x is not None and x.shape[0]:
            for c, sc, y in zip(s["codes"], s["scales"], _parts(case, x)):
                _plain_append(c, sc, y, step["slots"])
    s["pool"] = pool
    if case["kind"] in ("append", "attend"):
        s["step"], _ = _plain_plan(pool, s["have"], s["add"])
    if case["kind"] == "attend":
        for c, sc, y in zip(s["codes"], s["scales"], _parts(case, s["x"])):
            _plain_append(c, sc, y, s["step"]["slots"])


def _plain_plan(pool, have, add):
    tables, held = pool["tables"].clone(), pool["held"]
    need = (have + add + BLOCK - 1) // BLOCK
    j = torch.arange(tables.shape[1], device="cuda")[None, :]
    back = (j >= need[:, None]) & (j < held[:, None])
    take = (j >= held[:, None]) & (j < need[:, None])
    stack = torch.cat([pool["stack"], tables[back]])
    n = int(take.sum())
    tables[back] = -1
    tables[take] = stack.flip(0)[:n]
    starts = torch.zeros(add.shape[0] + 1, dtype=torch.int32, device="cuda")
    starts[1:] = torch.cumsum(add, 0)
    seq = torch.repeat_interleave(torch.arange(add.shape[0], device="cuda"), add.long())
    positions = torch.arange(seq.shape[0], device="cuda", dtype=torch.int32) - starts[seq] + have[seq]
    slots = tables[seq, (positions // BLOCK).long()] * BLOCK + positions % BLOCK
    return ({"starts": starts, "positions": positions, "slots": slots, "tables": tables},
            {"tables": tables, "held": need, "stack": stack[:stack.shape[0] - n]})


def _pow2(k):
    """2^k in fp32 for whole k, exactly."""
    return ((k.clamp(-126, 127) + 127) << 23).to(torch.int32).view(torch.float32)


def _plain_append(codes, scales, x, slots):
    """Rows x [n][kv_heads][head_dim] into codes [page][head][32][head_dim] and scales [page][head], in place."""
    x = x.float()
    page, off = (slots // BLOCK).long(), (slots % BLOCK).long()
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


def _plain_read(s, which):
    table, pos = s["step"]["tables"], s["pos"].long()
    page = table[s["seq"].long(), pos // BLOCK].long()
    return s["codes"][which][page, :, pos % BLOCK].float() * s["scales"][which][page][:, :, None]


def _plain_attend(s, tables):
    case = s["case"]
    H, KVH, hd = case["heads"], case["kv_heads"], case["head_dim"]
    G = H // KVH
    q = s["x"][:, :H * hd].view(-1, H, hd)
    out = torch.empty(s["n"], H * hd, dtype=s["x"].dtype, device="cuda")
    t = 0
    for b, (have, add) in enumerate(zip(s["have_list"], s["add_list"])):
        if not add:
            continue
        L = have + add
        page = tables[b, :_pages(L)].long()
        k, v = (((c[page].float() * sc[page][:, :, None, None]).transpose(0, 1).reshape(KVH, -1, hd)[:, :L])
                for c, sc in zip(s["codes"], s["scales"]))
        step = max(1, min(add, (1 << 28) // (L * H)))
        for r in range(0, add, step):
            m = min(step, add - r)
            y = q[t + r:t + r + m].float().view(m, KVH, G, hd).permute(1, 2, 0, 3).reshape(KVH, G * m, hd)
            score = torch.matmul(y, k.transpose(1, 2)) / math.sqrt(hd)
            if add > 1:
                last = torch.arange(have + r, have + r + m, device="cuda").repeat(G)
                score.masked_fill_(torch.arange(L, device="cuda")[None, :] > last[:, None], -math.inf)
            p = torch.exp(score - score.amax(2, keepdim=True))
            o = torch.matmul(p, v) / p.sum(2, keepdim=True)
            out[t + r:t + r + m] = o.view(KVH, G, m, hd).permute(2, 0, 1, 3).reshape(m, H * hd).to(out.dtype)
        t += add
    return out


def _run_plain(s):
    kind = s["kind"]
    if kind == "plan":
        return _plain_plan(s["pool"], s["have"], s["add"])[0]
    step = s["step"] if kind != "step" else _plain_plan(s["pool"], s["have"], s["add"])[0]
    if kind != "attend":
        for c, sc, y in zip(s["codes"], s["scales"], _parts(s["case"], s["x"])):
            _plain_append(c, sc, y, step["slots"])
    if kind == "append":
        return {"k": _plain_read(s, 0), "v": _plain_read(s, 1)}
    out = _plain_attend(s, step["tables"])
    return {"out": out} if kind == "attend" else {**step, "out": out}


def run(state):
    return (_run_own if own else _run_plain)(state)


# ---------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    """Means over the lengths that a case's seeds give."""
    H, KVH, hd = case["heads"], case["kv_heads"], case["head_dim"]
    es = 4 if case["dtype"] == "f32" else 2
    B, kind = case["seqs"], case["kind"]
    hold, add = (case["hold_lo"] + case["hold_hi"]) / 2, (case["add_lo"] + case["add_hi"]) / 2
    prompts = min(case["prompts"], B - case["done"])
    singles = B - case["done"] - prompts
    n = prompts * add + singles
    W = _width(case)
    row = KVH * hd
    total = {"bytes": 0, "flops": 0}
    if kind in ("plan", "step"):
        total["bytes"] += 4 * (2 * B + B + 1 + 2 * n + 2 * B * W)
    if kind in ("append", "step"):
        blocks = prompts * (add / BLOCK + 1) + singles
        total["bytes"] += 2 * n * row * (es + 1) + 2 * blocks * KVH * 4
        total["flops"] += 6 * n * row
    if kind == "append":
        total["bytes"] += 2 * 4 * row * (n + BLOCK / 2 * (prompts + singles if hold else 0))
    if kind in ("attend", "step"):
        seen = prompts * (hold + add) + singles * (hold + 1)
        total["bytes"] += 2 * seen * row + 2 * seen / BLOCK * KVH * 4 + 2 * n * H * hd * es
        total["flops"] += 4 * H * hd * (prompts * add * (hold + (add + 1) / 2) + singles * (hold + 1))
    return total


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


def exact(case, seed):
    kind = case["kind"]
    rounds = _rounds(case, seed)
    have, add = rounds[2]
    whole = {name: None for name in ("starts", "positions", "slots", "tables")}
    if kind == "plan":
        return None                       # whole numbers
    H, KVH, hd = case["heads"], case["kv_heads"], case["head_dim"]
    G = H // KVH
    rows = [_rows(case, seed, i, int(a.sum())) for i, (_, a) in enumerate(rounds)]
    at = [np.concatenate([[0], np.cumsum(a)]) for _, a in rounds]
    keys, vals, outs = [], [], []
    for b in range(case["seqs"]):
        if not add[b]:
            continue
        k, v = (_exact_blocks([(int(h[b]), _parts(case, x[at[i][b]:at[i][b + 1]])[w]) for i, ((h, a), x) in enumerate(zip(rounds, rows))])
                for w in range(2))
        L, h0, n = int(have[b] + add[b]), int(have[b]), int(add[b])
        if kind == "append":
            keys.append(k[h0 // BLOCK * BLOCK:L])
            vals.append(v[h0 // BLOCK * BLOCK:L])
            continue
        q = rows[2][at[2][b]:at[2][b + 1], :H * hd].view(n, H, hd)
        out = torch.empty(n, H, hd, dtype=torch.float64, device="cuda")
        step = max(1, (1 << 26) // L)
        for h in range(H):
            kk, vv = k[:L, h // G], v[:L, h // G]
            for r in range(0, n, step):
                score = (q[r:r + step, h].double() @ kk.T) * hd ** -0.5
                seen = torch.arange(L, device="cuda")[None, :] <= torch.arange(h0 + r, h0 + min(n, r + step), device="cuda")[:, None]
                out[r:r + step, h] = torch.softmax(torch.where(seen, score, score.new_full((), -math.inf)), 1) @ vv
        outs.append(out.view(n, H * hd))
    if kind == "append":
        return {"k": torch.cat(keys), "v": torch.cat(vals)}
    out = {"out": torch.cat(outs)}
    return out if kind == "attend" else {**whole, **out}
