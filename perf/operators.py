"""Keys and values held in 4 bits: the operators on such a cache, as cases that can be timed and checked.

Microscaled 4-bit floating point: 32 neighbouring elements of a row share a scale 2^(s - 127), one byte s, and each of
them is a code of 4 bits (sign, 2 bits of exponent, 1 of fraction: 0, 0.5, 1, 1.5, 2, 3, 4, 6).  A row's block is held with
s - 127 = floor(log2(largest magnitude)) - 2, at least -124; its elements are rounded to the nearest value, ties to the
even code, beyond 6 to 6.  A block with an infinity or a NaN has s = 255 and reads as NaN.

A cache unit is uint8 [pages, kv_heads, 68 * head_dim].  A page's part of one kv head, for its 64 tokens and a head size
of 32 m: keys' codes [64 tokens][16 m bytes], keys' scales [16][m][4], values' codes [8][4 m][8 tokens][4 bytes], values'
scales [8][m][8 tokens].  Codes lie low half byte first.  The key scale of token t and block b stands at
[4 ((t % 32) / 8) + t % 4][b][2 (t / 32) + (t / 4) % 2]; token t is number t % 8 of group t / 8 of the values.

Tasks:
* `write`: the new tokens of a step (keys and values side by side in rows [q heads | k heads | v heads]) go into the pages
  and are read back: what the cache now holds for them.
* `read`: the keys and values of whole sequences, out of the pages.
* `decode`: attention of one new token per sequence over the pages.
* `prefill`: attention of the new tokens of every sequence, which stand in the pages already, over all tokens up to
  each (of the last `window`).
"""
import math

import torch

own = False

PAGE = 64
MIN_EXP, MAX_EXP = -124, 125
_VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _case(name, task, lens, nq=32, nkv=8, hd=128, new=0, window=0, pad=0, dtype="bfloat16"):
    """`lens`: the sequences' lengths as text, "1088" or "9*100..8000" (so many, spread evenly); `new`: how many of each
    sequence's tokens are new, 0: all of them; `pad`: sequences of one token without a slot behind the others."""
    return {"name": name, "task": task, "lens": lens, "nq": nq, "nkv": nkv, "hd": hd, "new": new, "window": window,
            "pad": pad, "dtype": dtype}


def listed():
    return [
        # the new rows of a single-token step of eight users: the smallest call
        _case("write step of 8", "write", "8*128..2048", new=1),
        # several requests of unequal length taken in together, small heads, behind tokens that are there already
        _case("write ragged", "write", "6*401..1357", nq=28, nkv=4, hd=64, new=333),
        # four long prompts
        _case("write prompts", "write", "4*4096..4096"),
        # one chat's cache, taken out in 16 bits
        _case("read one", "read", "777", hd=128),
        # documents' caches, handed to a program that holds 16 bits
        _case("read documents", "read", "4*8192..8192"),
        # one user in a chat, the answer being written
        _case("decode 1", "decode", "1088", new=1),
        # a small batch of unequal contexts through window attention, padded to eight
        _case("decode window", "decode", "7*128..9001", new=1, window=4096, pad=1),
        # a server's full batch
        _case("decode 64", "decode", "64*128..8192", new=1),
        # agents over long documents
        _case("decode long", "decode", "16*32768..32768", new=1),
        # a question of 67 tokens behind a document
        _case("prefill question", "prefill", "16411", new=67),
        # prompts of unequal length, small heads
        _case("prefill ragged", "prefill", "5*93..1357", nq=32, nkv=4, hd=64),
        # a document
        _case("prefill document", "prefill", "8192"),
    ]


def _lengths(case):
    text = str(case["lens"])
    if "*" not in text:
        return [int(text)]
    n, span = text.split("*")
    lo, hi = (int(x) for x in span.split(".."))
    n = int(n)
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    task = rng.choice(["write", "read", "decode", "decode", "prefill", "prefill"])
    hd = rng.choice([32, 64, 64, 96, 128, 128, 128, 160, 256])
    nkv = rng.choice([1, 2, 3, 4, 8, 8])
    group = rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16])
    n = _spread(rng, 1, 64 if task == "decode" else 8)
    # tokens of all sequences: up to the largest listed case's work
    most = {"write": 16384, "read": 32768, "decode": 524288, "prefill": 8192}[task] * 1024 / (nkv * hd)
    hi = max(1, _spread(rng, 1, max(2, min(32768, most / n))))
    if task == "prefill":
        hi = min(hi, max(1, int(math.sqrt(8192.0 * 8192 * 4096 / (n * nkv * group * hd)))))
    lo = max(1, _spread(rng, 1, hi + 1) if rng.random() < 0.7 else hi)
    lo = min(lo, hi)
    new = 0
    if task == "decode":
        new = 1
    elif task in ("write", "prefill") and rng.random() < 0.5:
        new = _spread(rng, 1, 300)
    window = rng.choice([0, 0, 0, 1, _spread(rng, 2, 5000)]) if task in ("decode", "prefill") else 0
    lens = str(hi) if n == 1 else "%d*%d..%d" % (n, lo, hi)
    return {"task": task, "lens": lens, "nq": nkv * group, "nkv": nkv, "hd": hd, "new": new, "window": window,
            "pad": rng.choice([0, 0, 1, 2]) if task in ("decode", "write") else 0,
            "dtype": rng.choice(["bfloat16", "bfloat16", "float32"]) if task in ("write", "read") else "bfloat16"}


def _new_of(case, lens):
    return [n if not case["new"] else min(n, int(case["new"])) for n in lens]


def work(case):
    lens = _lengths(case)
    new = _new_of(case, lens)
    nq, nkv, hd, w = case["nq"], case["nkv"], case["hd"], case["window"]
    size = 4 if case["dtype"] == "float32" else 2
    held = hd / 2 + hd / 32                                     # bytes of a row of one head in the cache
    if case["task"] == "write":                                 # rows in, rows held, and read back
        rows = 2 * nkv * sum(new)
        return {"bytes": rows * (2 * hd * size + 2 * held), "flops": 4 * rows * hd}
    if case["task"] == "read":
        rows = 2 * nkv * sum(lens)
        return {"bytes": rows * (hd * size + held), "flops": rows * hd}
    tokens = pairs = 0
    for n, k in zip(lens, new):
        first = n - k
        tokens += n - max(0, first - w + 1) if w else n
        seen = sum(range(first + 1, n + 1)) if not w else sum(min(w, i) for i in range(first + 1, n + 1))
        pairs += seen
    return {"bytes": 2 * nkv * tokens * held + 2 * 2 * nq * hd * (sum(new) + case["pad"]), "flops": 4 * nq * hd * pairs}


# ---------------------------------------------------------------- the cache's layout ----
def _addresses(state, pos, slot):
    """Byte places in the flat cache of what tokens `pos` of slots `slot` hold ([n] each): key codes [n, nkv, 16 m], key
    scales [n, nkv, m], value codes [n, nkv, 16 m], value scales [n, nkv, m]."""
    nkv, hd, dev = state["nkv"], state["hd"], pos.device
    m = hd // 32
    page = state["table"].long()[slot, pos // PAGE]
    t = pos % PAGE
    heads = torch.arange(nkv, device=dev)
    base = (page[:, None] * nkv + heads[None, :])[:, :, None] * (68 * hd)
    t = t[:, None, None]
    byte = torch.arange(16 * m, device=dev)[None, None, :]
    block = torch.arange(m, device=dev)[None, None, :]
    kc = base + t * (16 * m) + byte
    r, j = 4 * ((t % 32) // 8) + t % 4, 2 * (t // 32) + (t // 4) % 2
    ks = base + 1024 * m + (r * m + block) * 4 + j
    vc = base + 1088 * m + ((t // 8) * (4 * m) + byte // 4) * 32 + (t % 8) * 4 + byte % 4
    vs = base + 2112 * m + ((t // 8) * m + block) * 8 + t % 8
    return kc, ks, vc, vs


def _pack(x):
    """Rows [..., hd] -> (codes as bytes [..., hd / 2], scale bytes [..., hd / 32])."""
    shape = x.shape
    y = x.float().reshape(shape[:-1] + (shape[-1] // 32, 32))
    big = y.abs().amax(-1)
    bad = ~torch.isfinite(big)
    e = torch.frexp(torch.where(bad | (big == 0), torch.full_like(big, 2.0 ** -126), big)).exponent - 3
    e = e.clamp(MIN_EXP, MAX_EXP)
    y = torch.where(bad[..., None], torch.zeros_like(y), y) * torch.pow(2.0, -e.float())[..., None]
    a = y.abs()
    r = torch.where(a < 2, torch.round(a * 2) / 2, torch.where(a < 4, torch.round(a), torch.round(a / 2) * 2)).clamp(max=6)
    code = torch.where(r < 2, r * 2, torch.where(r < 4, r + 2, r / 2 + 4)).to(torch.uint8)
    code = code | (torch.signbit(y).to(torch.uint8) << 3)
    code = code.reshape(shape)
    codes = code[..., 0::2] | (code[..., 1::2] << 4)
    return codes, torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)


def _unpack(codes, scales):
    """The values that codes and scales stand for, float32 [..., hd]."""
    table = torch.tensor(_VALUES + [-v for v in _VALUES], device=codes.device)
    both = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    s = torch.pow(2.0, scales.float() - 127)
    s = torch.where(scales == 255, torch.full_like(s, float("nan")), s)
    return table[both] * s.repeat_interleave(32, -1)


def _store(state, k, v, pos, slot):
    flat = state["cache"].view(-1)
    kc, ks, vc, vs = _addresses(state, pos, slot)
    for at_c, at_s, x in ((kc, ks, k), (vc, vs, v)):
        codes, scales = _pack(x)
        flat[at_c] = codes
        flat[at_s] = scales


def _fetch(state, pos, slot):
    flat = state["cache"].view(-1)
    kc, ks, vc, vs = _addresses(state, pos, slot)
    return _unpack(flat[kc], flat[ks]), _unpack(flat[vc], flat[vs])


# ------------------------------------------------------------------------- the cases ----
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed) * 7919 + 17)
    host = torch.Generator().manual_seed(int(seed))
    lens = _lengths(case)
    new = _new_of(case, lens)
    nq, nkv, hd, pad = case["nq"], case["nkv"], case["hd"], case["pad"]
    n_seqs = len(lens)
    pages = [-(-n // PAGE) for n in lens]
    n_pages = sum(pages) + 3
    order = torch.randperm(n_pages, generator=host)
    table = torch.full((n_seqs + 1, max(pages)), -1, dtype=torch.int32)
    at = 0
    slots = torch.randperm(n_seqs + 1, generator=host)[:n_seqs]
    for s, n in zip(slots.tolist(), pages):
        table[s, :n] = order[at:at + n].int()
        at += n
    state = {"task": case["task"], "nq": nq, "nkv": nkv, "hd": hd, "window": case["window"], "scale": 1.0 / math.sqrt(hd),
             "lens": lens, "new": new, "pad": pad, "host_slots": slots.tolist(), "table": table.to(dev)}
    # pages that held other sequences before: every byte is there already
    state["cache"] = torch.randint(0, 256, (n_pages, nkv, 68 * hd), dtype=torch.uint8, device=dev, generator=g)
    dt = torch.float32 if case["dtype"] == "float32" else torch.bfloat16
    # some channels of the keys are large, as those of trained models are
    loud = torch.exp(0.7 * torch.randn((nkv, hd), device=dev, generator=g))

    def rows(n):
        k = torch.randn((n, nkv, hd), device=dev, generator=g) * loud
        v = torch.randn((n, nkv, hd), device=dev, generator=g)
        return k.to(dt), v.to(dt)

    for i, (n, s) in enumerate(zip(lens, slots.tolist())):
        old = n - new[i] if case["task"] == "write" else n
        for a in range(0, old, 8192):
            pos = torch.arange(a, min(old, a + 8192), device=dev)
            k, v = rows(pos.numel())
            _store(state, k, v, pos, torch.full_like(pos, s))
    # the step's arrays
    T = sum(new) + pad
    counts = new + [1] * pad
    pos = torch.cat([torch.arange(n - k, n) for n, k in zip(lens, new)] + [torch.zeros(pad, dtype=torch.long)])
    seq = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts))
    cu = torch.zeros(len(counts) + 1, dtype=torch.long)
    cu[1:] = torch.cumsum(torch.tensor(counts), 0)
    arrays = {"positions": pos, "seq_of_token": seq, "cu": cu, "slots": torch.tensor(slots.tolist() + [-1] * pad),
              "ctx": torch.tensor(lens + [0] * pad)}
    state.update({name: t.int().to(dev) for name, t in arrays.items()})
    state["B"], state["T"] = len(counts), T
    if case["task"] != "read":
        qkv = torch.randn((T, (nq + 2 * nkv) * hd), device=dev, generator=g)
        qkv.view(T, nq + 2 * nkv, hd)[:, nq:nq + nkv] *= loud
        state["qkv"] = qkv.to(dt)
    if case["task"] in ("write", "read"):
        if case["task"] == "read":
            pos = torch.cat([torch.arange(n) for n in lens])
            seq = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))
            state["positions"], state["seq_of_token"] = pos.int().to(dev), seq.int().to(dev)
        n_rows = state["positions"].numel()
        state["k_out"] = torch.zeros((n_rows, nkv * hd), dtype=dt, device=dev)
        state["v_out"] = torch.zeros((n_rows, nkv * hd), dtype=dt, device=dev)
    else:
        state["out"] = torch.zeros((T, nq * hd), dtype=dt, device=dev)
        if own:
            from braidinfer_amd import kernels as K
            state["nsplit"] = K.attention_kv4_splits(state["B"], max(counts), nq, nkv, hd, max(lens), case["window"] or None,
                                                     case["task"] == "decode")
            n = state["nsplit"]
            state["part_o"] = torch.empty(T * nq * n * hd, device=dev) if n > 1 else None
            state["part_ml"] = torch.empty(T * nq * n * 2, device=dev) if n > 1 else None
    return state


def _rows_of(state):
    """Keys and values of the step's rows, [T, nkv, hd]."""
    nq, nkv, hd = state["nq"], state["nkv"], state["hd"]
    heads = state["qkv"].view(state["T"], nq + 2 * nkv, hd)
    return heads[:, nq:nq + nkv], heads[:, nq + nkv:]


def _attend(state, i):
    """Attention of the new tokens of sequence i in 32 bits, [n, nq, hd]."""
    nq, nkv, hd, w = state["nq"], state["nkv"], state["hd"], state["window"]
    n, k = state["lens"][i], state["new"][i]
    first = n - k
    lo = max(0, first - w + 1) if w else 0
    dev = state["qkv"].device
    pos = torch.arange(lo, n, device=dev)
    keys, values = _fetch(state, pos, torch.full_like(pos, state["host_slots"][i]))
    at, G = sum(state["new"][:i]), nq // nkv
    # heads first: [nkv, hd, n] and [nkv, n, hd], queries [nkv, new, G, hd]
    keys, values = keys.permute(1, 2, 0).contiguous(), values.transpose(0, 1).contiguous()
    q = state["qkv"][at:at + k, :nq * hd].float().view(k, nkv, G, hd).transpose(0, 1) * state["scale"]
    out = torch.empty((nkv, k, G, hd), device=dev)
    step = max(1, (1 << 28) // max(1, nq * (n - lo)))                       # rows whose scores are held at a time
    for a in range(0, k, step):
        b = min(k, a + step)
        s = torch.matmul(q[:, a:b].reshape(nkv, -1, hd), keys).view(nkv, b - a, G, n - lo)
        if k > 1:
            place = torch.arange(first + a, first + b, device=dev)[:, None, None]
            gone = pos > place
            if w:
                gone = gone | (pos <= place - w)
            s = s.masked_fill(gone, float("-inf"))
        e = torch.exp(s - s.amax(-1, keepdim=True)).view(nkv, -1, n - lo)
        out[:, a:b] = (torch.matmul(e, values) / e.sum(-1, keepdim=True)).view(nkv, b - a, G, hd)
    return out.transpose(0, 1).reshape(k, nq, hd)


def run(state):
    task = state["task"]
    if own:
        from braidinfer_amd import kernels as K
        if task in ("write", "read"):
            if task == "write":
                K.rope_kv4_write(state["qkv"], None, None, state["positions"], state["seq_of_token"], state["slots"],
                                 state["table"], state["cache"], state["nq"], state["nkv"], state["hd"], 0, False, PAGE, True)
            K.kv4_read(state["k_out"], state["v_out"], state["positions"], state["seq_of_token"], state["slots"],
                       state["table"], state["cache"], state["nkv"], state["hd"], PAGE)
            return state["k_out"], state["v_out"]
        sizes = (state["nq"], state["nkv"], state["hd"], PAGE, state["window"] or None, state["scale"], state["nsplit"],
                 state["part_o"], state["part_ml"])
        if task == "decode":
            K.attention_decode_kv4(state["qkv"], state["qkv"].stride(0), state["out"], state["slots"], state["ctx"],
                                   state["table"], state["cache"], state["B"], *sizes)
        else:
            K.attention_prefill_kv4(state["qkv"], state["qkv"].stride(0), state["out"], state["cu"], state["slots"],
                                    state["ctx"], state["table"], state["cache"], state["B"], max(state["new"]), *sizes)
        return state["out"]
    if task in ("write", "read"):
        live = state["positions"].numel() - (state["pad"] if task == "write" else 0)
        pos = state["positions"][:live].long()
        slot = state["slots"].long()[state["seq_of_token"][:live].long()]
        if task == "write":
            k, v = _rows_of(state)
            _store(state, k[:live], v[:live], pos, slot)
        k, v = _fetch(state, pos, slot)
        state["k_out"][:live] = k.reshape(live, -1).to(state["k_out"].dtype)
        state["v_out"][:live] = v.reshape(live, -1).to(state["v_out"].dtype)
        return state["k_out"], state["v_out"]
    at = 0
    for i in range(len(state["lens"])):
        k = state["new"][i]
        state["out"][at:at + k] = _attend(state, i).reshape(k, -1).to(state["out"].dtype)
        at += k
    if state["pad"]:
        state["out"][at:] = 0
    return state["out"]


# ----------------------------------------------------- from the definition, in 64 bits ----
def _held_pages(state, i):
    """Keys and values of sequence i as its pages hold them, float64 [tokens of its pages, nkv, hd] each."""
    nkv, hd = state["nkv"], state["hd"]
    m = hd // 32
    n = -(-state["lens"][i] // PAGE)
    pages = state["cache"][state["table"][state["host_slots"][i], :n].long()]
    kc, ks, vc, vs = pages.split([1024 * m, 64 * m, 1024 * m, 64 * m], -1)
    kc = kc.reshape(n, nkv, 64, 16 * m)
    # scales [4 (octet of a half) + t % 4][block][2 half + (t / 4) % 2] -> [half, octet, t / 4 % 2, t % 4, block]
    ks = ks.reshape(n, nkv, 4, 4, m, 2, 2).permute(0, 1, 5, 2, 6, 3, 4).reshape(n, nkv, 64, m)
    vc = vc.reshape(n, nkv, 8, 4 * m, 8, 4).permute(0, 1, 2, 4, 3, 5).reshape(n, nkv, 64, 16 * m)
    vs = vs.reshape(n, nkv, 8, m, 8).transpose(-1, -2).reshape(n, nkv, 64, m)
    out = []
    for codes, scales in ((kc, ks), (vc, vs)):
        code = torch.empty(codes.shape[:-1] + (hd,), dtype=torch.int32, device=codes.device)
        code[..., 0::2] = (codes & 15).int()
        code[..., 1::2] = (codes >> 4).int()
        exp, frac = (code >> 1) & 3, (code & 1).double()
        mag = torch.where(exp == 0, frac * 0.5, (1 + frac * 0.5) * torch.exp2((exp - 1).double()))
        val = torch.where(code >= 8, -mag, mag).view(codes.shape[:-1] + (m, 32))
        val = val * torch.exp2(scales.double() - 127)[..., None]
        val = torch.where((scales == 255)[..., None], torch.full_like(val, float("nan")), val)
        out.append(val.reshape(n, nkv, 64, hd).transpose(1, 2).reshape(n * PAGE, nkv, hd))
    return out


def _nearest(x):
    """Rows [n, nkv, hd] as the cache holds them, float64."""
    y = x.double().unflatten(-1, (-1, 32))
    big = y.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(big.clamp(min=2.0 ** -130))) - 2
    # log2 of a number just below a power of two may come out as its exponent
    e = torch.where(torch.exp2(e + 2) > big, e - 1, e).clamp(MIN_EXP, MAX_EXP)
    u = y.abs() / torch.exp2(e)
    grid = torch.tensor(_VALUES, dtype=torch.float64, device=x.device)
    best, dist = torch.zeros_like(u), u.clone()
    for c in range(1, 8):
        d = (u - grid[c]).abs()
        nearer = (d < dist) | ((d == dist) & (c % 2 == 0))
        best, dist = torch.where(nearer, grid[c], best), torch.where(nearer, d, dist)
    val = torch.where(y < 0, -best, best) * torch.exp2(e)
    return torch.where(torch.isfinite(big), val, torch.full_like(val, float("nan"))).flatten(-2)


def exact(case, seed):
    state = prepare(case, seed)
    nq, nkv, hd, w = case["nq"], case["nkv"], case["hd"], case["window"]
    if case["task"] == "write":
        out = []
        for x in _rows_of(state):
            y = _nearest(x).reshape(state["T"], -1)
            if case["pad"]:
                y[state["T"] - case["pad"]:] = 0
            out.append(y)
        return tuple(out)
    if case["task"] == "read":
        ks, vs = [], []
        for i, n in enumerate(state["lens"]):
            k, v = _held_pages(state, i)
            ks.append(k[:n].reshape(n, -1))
            vs.append(v[:n].reshape(n, -1))
        return torch.cat(ks), torch.cat(vs)
    out = torch.zeros((state["T"], nq * hd), dtype=torch.float64, device=state["qkv"].device)
    G, at = nq // nkv, 0
    for i, (n, new) in enumerate(zip(state["lens"], state["new"])):
        k, v = _held_pages(state, i)
        q = state["qkv"][at:at + new, :nq * hd].double().view(new, nq, hd)
        step = max(1, (1 << 27) // n)
        for h in range(nq):
            kh, vh = k[:n, h // G], v[:n, h // G]
            for a in range(0, new, step):
                b = min(new, a + step)
                first, last = n - new + a, n - new + b - 1              # positions of these rows
                lo = max(0, first - w + 1) if w else 0
                s = (q[a:b, h] @ kh[lo:last + 1].T) / math.sqrt(hd)
                rows = torch.arange(first, last + 1, device=s.device).view(-1, 1)
                cols = torch.arange(lo, last + 1, device=s.device).view(1, -1)
                gone = (cols > rows) | ((cols <= rows - w) if w else torch.zeros_like(cols > rows))
                s[gone] = -math.inf
                out[at + a:at + b, h * hd:(h + 1) * hd] = torch.softmax(s, -1) @ vh[lo:last + 1]
        at += new
    return out
