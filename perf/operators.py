"""A KV cache in pages, of 16 or of 8 bits, as a server uses it: written, attended over and read back.

Three operators, each over a batch of sequences of their own lengths whose rows lie in pages of one pool:

* ``append``: the new tokens' q and k are rotated, k and v go into the pages, in 8 bits with a power of two to a row or
  as they are (an 8-bit cache is read back at once, so that what it holds is looked at);
* ``attend``: the new tokens attend over the pages, causally, over all keys or over a sliding window and a few first
  tokens that stay visible (sinks).  One new token to a sequence (decode), pieces of prompts, whole prompts, or all of
  these in one batch;
* ``read``: rows of the cache come back as dense tensors.

A page holds, for each kv head, ``page_size`` rows of 128; in 8 bits it ends with a byte to each of these rows, the
exponent of the row's scale plus 127.  Sequence b's tokens are rows ``q_starts[b]`` to ``q_starts[b + 1]`` of the dense
tensors and the last ones of its ``kv_lens[b]`` cached rows.

``own`` False: the plain form, elementary torch operations in 32 bits.  ``own`` True: the calls of the framework.
Head layouts are those of the benchmark's configurations.
"""
import functools
import math
import random

import torch

own = False

HEAD_DIM = 128

# name: (query heads, kv heads, dtype, neox pairs, rotary theta)
LAYOUTS = {
    "llama2-7b": (32, 32, "fp16", False, 1e4),
    "qwen2.5-1.5b": (12, 2, "bf16", True, 1e6),
    "qwen2.5-7b": (28, 4, "bf16", True, 1e6),
    "qwen2.5-32b": (40, 8, "bf16", True, 1e6),
}

# Bounds of the ranges that draw() covers: the longest prompt and cache of the benchmark's configurations
MAX_PROMPT, MAX_CACHE, MAX_BATCH = 8192, 32768, 64
MOST_ROWS = 16 * 32768 * 8  # cached rows of all kv heads, of the largest listed case
MOST_PAIRS = 28 * 1024 * 8192  # pairs of query row and visible key of the largest listed case, about


def _case(kind, layout, bits, page_size, batch, new, past, ragged=0, singles=0, window=0, sinks=0):
    """batch sequences of `past` cached and `new` tokens, `singles` of them with one new token; ragged: what the lengths
    are drawn with, up to these bounds (0: all have them)."""
    return {"kind": kind, "layout": layout, "bits": bits, "page_size": page_size, "batch": batch, "new": new, "past": past,
            "ragged": ragged, "singles": singles, "window": window, "sinks": sinks}


def listed():
    return [
        # a generated token of the smallest model in the middle of its answer: launches and latency only
        {"name": "decode 1.5b past 383", **_case("attend", "qwen2.5-1.5b", 16, 16, 1, 1, 383)},
        # a server's small batch at an ordinary length that fits no page, in 8 bits
        {"name": "decode 32b 5 x 2999, 8 bits", **_case("attend", "qwen2.5-32b", 8, 16, 5, 1, 2998)},
        # the largest batch of the longest contexts, in 8 bits
        {"name": "decode 32b 16 x 32768, 8 bits", **_case("attend", "qwen2.5-32b", 8, 64, 16, 1, 32767)},
        # many conversations of all lengths, of which a window and the first tokens are attended to
        {"name": "decode 7b 48 ragged, window", **_case("attend", "qwen2.5-7b", 16, 32, 48, 1, 16383, ragged=1, window=4096, sinks=4)},
        # the second turn of a long conversation
        {"name": "chunk 7b 200 past 16001", **_case("attend", "qwen2.5-7b", 16, 64, 1, 200, 16001)},
        # prompts of several users at once, fp16, as many kv heads as query heads
        {"name": "prompts llama 6 ragged to 1019", **_case("attend", "llama2-7b", 16, 16, 6, 1019, 0, ragged=2)},
        # a piece of a prompt among generated tokens of others, in 8 bits
        {"name": "mixed 7b 512 past 6000 and 31, 8 bits", **_case("attend", "qwen2.5-7b", 8, 16, 32, 512, 6000, ragged=3, singles=31)},
        # a long prompt with a sliding window and sinks
        {"name": "prompt 7b 8192, window", **_case("attend", "qwen2.5-7b", 16, 128, 1, 8192, 0, window=1024, sinks=4)},
        # the generated tokens of a batch enter an 8-bit cache
        {"name": "append 32b 24 ragged, 8 bits", **_case("append", "qwen2.5-32b", 8, 16, 24, 1, 8191, ragged=4)},
        # a prompt enters a 16-bit cache
        {"name": "append 7b 4096", **_case("append", "qwen2.5-7b", 16, 64, 1, 4096, 0)},
        # a short sequence leaves the cache for a dense one
        {"name": "read 1.5b 301", **_case("read", "qwen2.5-1.5b", 16, 16, 1, 301, 0)},
        # the longest one, out of 8 bits
        {"name": "read 32b 32768, 8 bits", **_case("read", "qwen2.5-32b", 8, 64, 1, 32768, 0)},
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    layout = rng.choice(sorted(LAYOUTS))
    heads, kv_heads = LAYOUTS[layout][:2]
    what = rng.choice(["decode", "decode", "chunk", "prompts", "mixed", "append", "append", "read"])
    bits, page_size = rng.choice([8, 16]), rng.choice([16, 16, 32, 48, 64, 128])
    ragged = rng.randint(1, 1 << 20) if rng.random() < 0.7 else 0
    most_keys = lambda batch: min(MAX_CACHE, MOST_ROWS // (batch * kv_heads))
    window = sinks = 0
    if what in ("decode", "chunk", "prompts", "mixed") and rng.random() < 0.4:
        window, sinks = _log_uniform(rng, 64, 8192), rng.choice([0, 1, 4, 16, 100])
    if what == "decode":
        batch = _log_uniform(rng, 1, MAX_BATCH)
        return _case("attend", layout, bits, page_size, batch, 1, _log_uniform(rng, 1, most_keys(batch)) - 1, ragged, 0, window, sinks)
    if what == "chunk":
        new = _log_uniform(rng, 2, 1024)
        past = min(_log_uniform(rng, 64, MAX_CACHE - 1024), MOST_PAIRS // (heads * new))
        return _case("attend", layout, bits, page_size, 1, new, past, ragged, 0, window, sinks)
    if what == "prompts":
        batch = _log_uniform(rng, 1, 16)
        new = _log_uniform(rng, 1, min(MAX_PROMPT, int(math.sqrt(2 * MOST_PAIRS / (heads * batch)))))
        return _case("attend", layout, bits, page_size, batch, new, 0, ragged, 0, window, sinks)
    if what == "mixed":
        batch = _log_uniform(rng, 2, MAX_BATCH)
        new = _log_uniform(rng, 2, 1024)
        past = min(_log_uniform(rng, 64, most_keys(batch)), MOST_PAIRS // (2 * heads * (new + batch)))
        singles = rng.randint(max(1, batch - 4), batch - 1)
        return _case("attend", layout, bits, page_size, batch, new, past, ragged, singles, window, sinks)
    if what == "append":
        batch = _log_uniform(rng, 1, MAX_BATCH)
        new = 1 if rng.random() < 0.5 else _log_uniform(rng, 1, MAX_PROMPT // batch)
        return _case("append", layout, bits, page_size, batch, new, _log_uniform(rng, 1, 4096) - 1, ragged)
    batch = _log_uniform(rng, 1, 16)
    return _case("read", layout, bits, page_size, batch, _log_uniform(rng, 1, MAX_CACHE * 8 // (batch * kv_heads)), 0, ragged)


def _lengths(case):
    """(cached, new) tokens of each sequence."""
    rng = random.Random(case["ragged"])
    lengths = []
    for i in range(case["batch"]):
        past, new = case["past"], case["new"]
        if case["ragged"] and i > 0:
            past, new = int(past * rng.random()), rng.randint(1, new)
        if i >= case["batch"] - case["singles"]:
            new = 1
        lengths.append((past, new))
    return lengths


def _dtype(case):
    return torch.float16 if LAYOUTS[case["layout"]][2] == "fp16" else torch.bfloat16


def _power(byte):
    """2^(byte - 127) as float32."""
    return (byte.to(torch.int32) << 23).view(torch.float32)


def _quantise(x, dtype):
    """Rows of 128 in `dtype` -> e4m3 values and the byte of each row's power of two: the least one that brings the row
    within 448, and at least 2^-63.  Magnitudes above 1.875 * 2^(the type's largest exponent) count as that, so that what
    the row stands for is in the type; infinities become NaN, and do not count in the row's largest magnitude."""
    most = 1.875 * 2.0 ** (15 if dtype == torch.float16 else 127)
    x = x.float()
    finite = torch.isfinite(x)
    clamped = torch.where(finite, x.clamp(-most, most), torch.zeros_like(x))
    bits = clamped.abs().amax(-1).view(torch.int32)
    byte = (((bits + 0x1FFFFF) >> 23) - 8).clamp(min=64)
    scaled = clamped * _power(254 - byte).unsqueeze(-1)
    scaled = torch.where(finite, scaled, torch.full_like(x, math.nan))
    return scaled.to(torch.float8_e4m3fn), byte.to(torch.uint8)


def _rotary_table(rows, theta, dtype):
    inv = theta ** (-torch.arange(0, HEAD_DIM, 2, dtype=torch.float64, device="cuda") / HEAD_DIM)
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * inv
    table = torch.stack([angle.cos(), angle.sin()], -1).float()
    return table.bfloat16().float() if dtype == torch.bfloat16 else table


class _Pool:
    """The pages of K, or of V: `raw` holds num_pages pages of bytes."""

    def __init__(self, num_pages, page_size, kv_heads, bits, dtype):
        self.shape = (num_pages, kv_heads, page_size)
        self.bits, self.dtype = bits, dtype
        self.values_bytes = kv_heads * page_size * HEAD_DIM * bits // 8
        self.page_bytes = self.values_bytes + (kv_heads * page_size if bits == 8 else 0)
        self.raw = torch.zeros(num_pages, self.page_bytes, dtype=torch.uint8, device="cuda")

    @property
    def values(self):  # [page][kv head][row][128]
        v = self.raw[:, :self.values_bytes]
        return v.view(torch.float8_e4m3fn if self.bits == 8 else self.dtype).unflatten(1, (*self.shape[1:], HEAD_DIM))

    @property
    def exponents(self):  # [page][kv head][row]
        return self.raw[:, self.values_bytes:].unflatten(1, self.shape[1:])

    def rows(self, page, row):
        """Rows `row` of pages `page` (tensors alike), in 32 bits: [...][kv head][128]."""
        x = self.values.view(torch.uint8)[page, :, row].view(self.values.dtype).float() if self.bits == 8 else self.values[page, :, row].float()
        return x * _power(self.exponents[page, :, row]).unsqueeze(-1) if self.bits == 8 else x

    def put(self, page, row, x):
        """x [tokens][kv head][128], in the type of the tensors."""
        if self.bits == 16:
            self.values[page, :, row] = x
            return
        values, byte = _quantise(x, self.dtype)
        self.values.view(torch.uint8)[page, :, row] = values.view(torch.uint8)
        self.exponents[page, :, row] = byte


def prepare(case, seed):
    heads, kv_heads, _, neox, theta = LAYOUTS[case["layout"]]
    dtype, page_size, bits = _dtype(case), case["page_size"], case["bits"]
    lengths = _lengths(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)

    # every sequence's pages, anywhere in a pool that has some more
    pages_of = [-(-(past + new) // page_size) for past, new in lengths]
    num_pages = sum(pages_of) + 3
    order = torch.randperm(num_pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    pages_per_seq = max(pages_of)
    table, at = torch.full((len(lengths), pages_per_seq), -1, dtype=torch.int32), 0
    for b, count in enumerate(pages_of):
        table[b, :count] = order[at:at + count]
        at += count
    tokens = sum(new for _, new in lengths)
    starts = [0]
    for _, new in lengths:
        starts.append(starts[-1] + new)
    s = {"kind": case["kind"], "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "neox": neox, "bits": bits, "batch": len(lengths),
         "page_size": page_size, "pages_per_seq": pages_per_seq, "num_pages": num_pages, "tokens": tokens, "lengths": lengths,
         "window": case["window"], "sinks": case["sinks"], "max_q_len": max(new for _, new in lengths),
         "max_kv_len": max(past + new for past, new in lengths), "page_table": table.cuda(),
         "q_starts": torch.tensor(starts, dtype=torch.int32, device="cuda"),
         "kv_lens": torch.tensor([past + new for past, new in lengths], dtype=torch.int32, device="cuda"),
         "k_pages": _Pool(num_pages, page_size, kv_heads, bits, dtype), "v_pages": _Pool(num_pages, page_size, kv_heads, bits, dtype)}
    # Cached rows of differing magnitude, e^(normal / 2): what a scale for each row is there for
    for name in ("k_pages", "v_pages"):
        pool = s[name]
        for first in range(0, num_pages, 4096):
            pages = torch.arange(first, min(num_pages, first + 4096), device="cuda")
            x = normal(len(pages), kv_heads, page_size, HEAD_DIM)
            x *= torch.exp(0.5 * normal(len(pages), kv_heads, page_size, 1))
            if bits == 16:
                pool.values[first:first + 4096] = x
            else:
                values, byte = _quantise(x, dtype)
                pool.values.view(torch.uint8)[first:first + 4096] = values.view(torch.uint8)
                pool.exponents[first:first + 4096] = byte
    if case["kind"] != "read":
        s["q"] = normal(tokens, heads, HEAD_DIM)
    if case["kind"] == "append":
        s["k"], s["v"] = normal(tokens, kv_heads, HEAD_DIM), normal(tokens, kv_heads, HEAD_DIM)
        s["table_rows"] = -(-s["max_kv_len"] // 256) * 256
        s["table"] = _rotary_table(s["table_rows"], theta, dtype)
    if own:
        from llm_simple_amd import ops

        s["ops"] = ops
        s["dt"] = ops.DT_FLOAT16 if dtype == torch.float16 else ops.DT_BFLOAT16
        s["cache_dt"] = ops.DT_FLOAT8_E4M3 if bits == 8 else s["dt"]
        for name, count in (("out", heads), ("out_k", kv_heads), ("out_v", kv_heads)):
            s[name] = torch.empty(tokens, count, HEAD_DIM, device="cuda", dtype=dtype)
        s["ws_bytes"] = ops.paged_flash_attn_workspace_bytes(tokens, len(lengths), s["max_q_len"], s["max_kv_len"], s["window"],
                                                             s["sinks"], heads // kv_heads, kv_heads, HEAD_DIM)
        s["ws"] = torch.empty(max(16, s["ws_bytes"]), device="cuda", dtype=torch.uint8)
    return s


# ---- the calls of the framework ----

def _own_append(s):
    s["ops"].hip_paged_rope_kv_append_layer(
        s["out"], s["k_pages"].raw, s["v_pages"].raw, s["page_table"], s["q_starts"], s["kv_lens"], s["table"], s["q"], s["k"], s["v"],
        s["tokens"], s["batch"], s["pages_per_seq"], s["num_pages"], s["page_size"], s["k_pages"].page_bytes, s["table_rows"],
        s["heads"], s["kv_heads"], HEAD_DIM, s["neox"], s["cache_dt"], s["dt"], torch.cuda.current_stream().cuda_stream)


def _own_read(s):
    s["ops"].hip_paged_kv_read_layer(
        s["out_k"], s["out_v"], s["k_pages"].raw, s["v_pages"].raw, s["page_table"], s["q_starts"], s["kv_lens"], s["tokens"], s["batch"],
        s["pages_per_seq"], s["num_pages"], s["page_size"], s["k_pages"].page_bytes, s["kv_heads"], HEAD_DIM, s["cache_dt"], s["dt"],
        torch.cuda.current_stream().cuda_stream)


def _own_attend(s):
    s["ops"].hip_paged_flash_attn_gqa_layer(
        s["out"], s["q"], s["k_pages"].raw, s["v_pages"].raw, s["page_table"], s["q_starts"], s["kv_lens"], s["ws"], s["ws_bytes"],
        s["tokens"], s["batch"], s["max_q_len"], s["max_kv_len"], s["pages_per_seq"], s["num_pages"], s["page_size"],
        s["k_pages"].page_bytes, s["window"], s["sinks"], s["heads"] // s["kv_heads"], s["kv_heads"], HEAD_DIM, s["cache_dt"], s["dt"],
        torch.cuda.current_stream().cuda_stream)


# ---- the plain form ----

def _places(s, everything=False):
    """Page and row of each new token, or of each cached row of sequence after sequence."""
    pages, rows = [], []
    for b, (past, new) in enumerate(s["lengths"]):
        at = torch.arange(0 if everything else past, past + new, device="cuda")
        pages.append(s["page_table"][b][at // s["page_size"]].long())
        rows.append(at % s["page_size"])
    return torch.cat(pages), torch.cat(rows)


def _rotate(x, table, positions, neox):
    """Every product and sum in 32 bits, rounded once at the end."""
    c, d = table[positions, None, :, 0], table[positions, None, :, 1]
    x32 = x.float()
    a, b = (x32[..., :64], x32[..., 64:]) if neox else (x32[..., 0::2], x32[..., 1::2])
    first, second = a * c - b * d, a * d + b * c
    return (torch.cat([first, second], -1) if neox else torch.stack([first, second], -1).flatten(-2)).to(x.dtype)


def _plain_append(s):
    positions = torch.cat([torch.arange(past, past + new, device="cuda") for past, new in s["lengths"]])
    page, row = _places(s)
    s["k_pages"].put(page, row, _rotate(s["k"], s["table"], positions, s["neox"]))
    s["v_pages"].put(page, row, s["v"])
    return _rotate(s["q"], s["table"], positions, s["neox"])


def _plain_attend(s):
    out = torch.empty_like(s["q"])
    group, at = s["heads"] // s["kv_heads"], 0
    for b, (past, new) in enumerate(s["lengths"]):
        n = past + new
        keys = torch.arange(n, device="cuda")
        pages, rows = s["page_table"][b][keys // s["page_size"]].long(), keys % s["page_size"]
        k, v = (s[name].rows(pages, rows).transpose(0, 1).contiguous() for name in ("k_pages", "v_pages"))
        last = torch.arange(past, n, device="cuda")[:, None]
        hidden = keys > last
        if s["window"]:
            hidden |= (keys <= last - s["window"]) & (keys >= s["sinks"])
        for h in range(s["kv_heads"]):
            q = s["q"][at:at + new, h * group:(h + 1) * group].float().transpose(0, 1).reshape(group * new, HEAD_DIM)
            scores = (q @ k[h].t()).view(group, new, n).mul_(HEAD_DIM ** -0.5)
            scores.masked_fill_(hidden, -math.inf)
            scores -= scores.amax(-1, keepdim=True)
            weights = scores.exp_()
            o = (weights.view(group * new, n) @ v[h]).view(group, new, HEAD_DIM) / weights.sum(-1, keepdim=True)
            out[at:at + new, h * group:(h + 1) * group] = o.transpose(0, 1).to(out.dtype)
        at += new
    return out


def run(s):
    if s["kind"] == "attend":
        if own:
            _own_attend(s)
            return s["out"]
        return _plain_attend(s)
    out = {}
    if s["kind"] == "append":
        if own:
            _own_append(s)
        out["q"] = s["out"] if own else _plain_append(s)
        if s["bits"] == 16:
            out["k_pages"], out["v_pages"] = s["k_pages"].values, s["v_pages"].values
            return out
    if own:
        _own_read(s)
        out["k"], out["v"] = s["out_k"], s["out_v"]
    else:
        page, row = _places(s)
        out["k"], out["v"] = (s[name].rows(page, row).to(s["dtype"]) for name in ("k_pages", "v_pages"))
    return out


# ---- the definition, in 64 bits ----

def _exact_rotate(x, s, positions):
    table = s["table"].double()[positions]
    turn = torch.complex(table[..., 0], table[..., 1])[:, None]
    x = x.double()
    pairs = torch.stack([x[..., :64], x[..., 64:]], -1) if s["neox"] else x.unflatten(-1, (64, 2))
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    return torch.cat([turned[..., 0], turned[..., 1]], -1) if s["neox"] else turned.flatten(-2)


def _exact_power(exponent):
    """2^exponent as float64 (by the bits: pow is not exact)."""
    return ((exponent.long() + 1023) << 52).view(torch.float64)


def _exact_eight_bits(x, dtype):
    """What a row stands for after 8 bits: four significant bits above 2^-6 of the row's power of two, steps of 2^-9 below."""
    x = x.to(dtype).double()
    fraction, power = torch.frexp(x.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100) / 448)  # fraction from 1/2 to 1
    power = torch.where(fraction > 0.5, power, power - 1).clamp(min=-63)
    scaled = x * _exact_power(-power)
    step = _exact_power(torch.frexp(scaled.abs().clamp(min=2.0 ** -6))[1] - 4)
    return torch.round(scaled / step) * step * _exact_power(power)


def _exact_rows(s, name, b, first, last):
    """Rows first to last of sequence b: [row][kv head][128]."""
    ps, pool, rows = s["page_size"], s[name], []
    for i in range(first // ps, -(-last // ps)):
        p = int(s["page_table_host"][b][i])
        x = pool.values[p].double()
        if pool.bits == 8:
            x = x * _exact_power(pool.exponents[p].int() - 127)[..., None]
        rows.append(x[:, max(0, first - i * ps):last - i * ps].transpose(0, 1))
    return torch.cat(rows)


def exact(case, seed):
    s = prepare(case, seed)
    s["page_table_host"] = s["page_table"].cpu()
    starts = [int(x) for x in s["q_starts"].cpu()]
    ends = [int(x) for x in s["kv_lens"].cpu()]
    if case["kind"] == "read":
        k, v = ([_exact_rows(s, name, b, n - (starts[b + 1] - starts[b]), n) for b, n in enumerate(ends)] for name in ("k_pages", "v_pages"))
        return {"k": torch.cat(k), "v": torch.cat(v)}
    if case["kind"] == "append":
        positions = torch.cat([torch.arange(n - (starts[b + 1] - starts[b]), n, device="cuda") for b, n in enumerate(ends)])
        out, k, v = {"q": _exact_rotate(s["q"], s, positions)}, _exact_rotate(s["k"], s, positions), s["v"].double()
        if s["bits"] == 8:
            return {**out, "k": _exact_eight_bits(k, s["dtype"]), "v": _exact_eight_bits(v, s["dtype"])}
        pools = [s[name].values.double() for name in ("k_pages", "v_pages")]
        for b, n in enumerate(ends):
            for t in range(starts[b], starts[b + 1]):
                place = n - starts[b + 1] + t
                for pool, x in zip(pools, (k, v)):
                    pool[int(s["page_table_host"][b][place // s["page_size"]]), :, place % s["page_size"]] = x[t]
        return {**out, "k_pages": pools[0], "v_pages": pools[1]}
    group = s["heads"] // s["kv_heads"]
    out = torch.empty(s["tokens"], s["heads"], HEAD_DIM, dtype=torch.float64, device="cuda")
    for b, n in enumerate(ends):
        k, v = (_exact_rows(s, name, b, 0, n) for name in ("k_pages", "v_pages"))
        at = torch.arange(n, device="cuda")
        for t0 in range(starts[b], starts[b + 1], 512):
            t1 = min(t0 + 512, starts[b + 1])
            p = n - starts[b + 1] + torch.arange(t0, t1, device="cuda")
            seen = at[None, :] <= p[:, None]
            if s["window"] > 0:
                seen &= (at[None, :] > p[:, None] - s["window"]) | (at[None, :] < s["sinks"])
            bias = torch.where(seen, 0.0, -math.inf).double()
            for h in range(s["heads"]):
                weights = torch.softmax(s["q"][t0:t1, h].double() @ k[:, h // group].t().contiguous() / math.sqrt(HEAD_DIM) + bias, -1)
                out[t0:t1, h] = weights @ v[:, h // group].contiguous()
    return out


@functools.lru_cache(maxsize=256)
def _visible(past, new, window, sinks):
    """(pairs of a new token and a key that it sees, keys that any of them sees)."""
    if not window:
        return new * past + new * (new + 1) // 2, past + new
    pairs = sum(min(p + 1, window) + min(sinks, max(0, p + 1 - window)) for p in range(past, past + new))
    first = max(0, past + 1 - window)
    return pairs, past + new - first + min(sinks, first)


def work(case):
    heads, kv_heads = LAYOUTS[case["layout"]][:2]
    lengths, row = _lengths(case), 2 * HEAD_DIM
    tokens = sum(new for _, new in lengths)
    cached = row if case["bits"] == 16 else HEAD_DIM + 1  # bytes of a cached row
    if case["kind"] == "read":
        return {"bytes": tokens * 2 * kv_heads * (cached + row), "flops": 0}
    if case["kind"] == "append":
        moved = tokens * (2 * heads * row + 4 * HEAD_DIM + 2 * kv_heads * (row + cached))
        if case["bits"] == 8:
            moved += tokens * 2 * kv_heads * (cached + row)  # read back
        return {"bytes": moved, "flops": 6 * HEAD_DIM // 2 * tokens * (heads + kv_heads)}
    visible = [_visible(past, new, case["window"], case["sinks"]) for past, new in lengths]
    pairs, keys = (sum(v[i] for v in visible) for i in (0, 1))
    return {"bytes": 2 * tokens * heads * row + keys * 2 * kv_heads * cached, "flops": 4 * HEAD_DIM * heads * pairs}
