"""Timed cases of the cached-attention operators: query and key norms with the position rotation, the 8-bit
cache written and read back, and attention over that cache.

The plain forms are elementary torch operations in 32 bits (angles in 64). The cache they work on is the one the
library keeps: pages of 32 tokens, one exponent byte e per page and head (scale 2^(e - 127)), e4m3 values, K of one
page and head as tiles [D/32][token][32], V as [D][slot] with token t = 8 g + 4 half + r at slot 16 half + 4 g + r.

Sizes: the DiT's heads (9 x 64 over 256 tokens, contexts of 1 to 128 tokens, packed q|k|v rows) in float32, and
the generic grouped-query shapes of token-by-token decoding and of prompts, in bfloat16 and float16.
"""

import itertools
import math
import os
import sys

import torch

own = False

TOKENS, DIT_HEADS, DIT_DIM = 256, 9, 64
BLOCK = 32  # tokens that share a page and a scale
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SLOT = [16 * (t // 4 % 2) + 4 * (t // 8) + t % 4 for t in range(BLOCK)]  # V: slot of token t
E4M3_MAX = 448.0


def listed():
    return [
        # one new token of one sequence: query and key norms and the rotation before it enters the cache
        dict(name="rope_token", kind="rope", T=1, H=32, Hkv=8, D=128, rot=128, pairs="half", far=4096, type="bf16"),
        # a batch of prompts, an odd number of tokens
        dict(name="rope_prompts", kind="rope", T=8191, H=32, Hkv=8, D=128, rot=128, pairs="half", far=8192, type="bf16"),
        # the packed q|k|v rows of a 64-image DiT batch, half of each head rotated, in neighbouring pairs
        dict(name="rope_dit", kind="rope", T=64 * TOKENS, H=DIT_HEADS, Hkv=DIT_HEADS, D=DIT_DIM, rot=32, pairs="near", far=TOKENS, type="f32"),
        # wide heads with one key head, far positions, a quarter of each head rotated
        dict(name="rope_wide", kind="rope", T=777, H=8, Hkv=1, D=256, rot=64, pairs="half", far=1 << 20, type="f16"),
        # a decoding step's append: one token for each of 64 sequences into their last pages, those pages read back
        dict(name="cache_append", kind="cache", B=64, new=1, most_new=1, lo=1, hi=2048, back=64, Hkv=8, D=128, type="bf16"),
        # ragged prompts behind prefixes that end inside a page, read back whole (a prefix taken up again)
        dict(name="cache_prompts", kind="cache", B=5, new=1, most_new=4095, lo=100, hi=4195, back=0, Hkv=8, D=128, type="bf16"),
        # the text contexts of a 64-image DiT batch, written once for a run of denoising steps
        dict(name="cache_dit", kind="cache", B=64, new=1, most_new=128, lo=1, hi=128, back=0, Hkv=DIT_HEADS, D=DIT_DIM, type="f32"),
        # the next token of one sequence
        dict(name="attn_token", kind="attn", B=1, n=1, most_n=1, lo=777, hi=777, H=32, Hkv=8, D=128, causal=True, type="bf16"),
        # a decoding step of 64 ragged sequences
        dict(name="attn_decode_b64", kind="attn", B=64, n=1, most_n=1, lo=333, hi=8191, H=32, Hkv=8, D=128, causal=True, type="bf16"),
        # two long sequences: split along the keys
        dict(name="attn_decode_long", kind="attn", B=2, n=1, most_n=1, lo=100001, hi=131089, H=32, Hkv=4, D=128, causal=True, type="f16"),
        # ragged prompts, the longest of 2048 new tokens behind as many cached ones
        dict(name="attn_prompts", kind="attn", B=3, n=5, most_n=2048, lo=1000, hi=4096, H=32, Hkv=8, D=128, causal=True, type="bf16"),
        # the DiT batch's image tokens over their text contexts, in float32
        dict(name="attn_dit_cross", kind="attn", B=64, n=TOKENS, most_n=TOKENS, lo=1, hi=128, H=DIT_HEADS, Hkv=DIT_HEADS, D=DIT_DIM, causal=False, type="f32"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    kind = rng.choice(["rope", "cache", "cache", "attn", "attn", "attn"])
    D, type_ = rng.choice([64, 128, 128, 256]), rng.choice(["f32", "f16", "bf16"])
    Hkv = rng.choice([1, 2, 4, 8, 9])
    H = Hkv * rng.choice([1, 2, 3, 4, 7, 8] if Hkv < 8 else [1, 2, 4])
    if kind == "rope":
        T = _log(rng, 1, max(1, min(8192, 80_000_000 // ((H + Hkv) * D * TYPES[type_].itemsize))))
        return dict(kind=kind, T=T, H=H, Hkv=Hkv, D=D, rot=rng.choice([D, D, D // 2, D // 4]), pairs=rng.choice(["half", "near"]),
                    far=_log(rng, 256, 1 << 20), type=type_)
    if kind == "cache":
        B = _log(rng, 1, 64)
        room = max(1, min(4096, 16_000_000 // (B * Hkv * D * TYPES[type_].itemsize)))  # tokens of each sequence
        most = _log(rng, 1, room)
        lo = rng.randint(most, room)
        return dict(kind=kind, B=B, new=rng.randint(1, most), most_new=most, lo=lo, hi=rng.randint(lo, room),
                    back=rng.choice([0, 0, 64]), Hkv=Hkv, D=D, type=type_)
    B, prompt = _log(rng, 1, 64), rng.random() < 0.5
    if not prompt:  # decoding, a few tokens at a time at most
        hi = _log(rng, 16, max(16, min(131072, 200_000_000 // (B * Hkv * D))))
        most = min(hi, rng.choice([1, 1, 1, 2, 4]))
        return dict(kind=kind, B=B, n=rng.randint(1, most), most_n=most, lo=rng.randint(most, hi), hi=hi, H=H, Hkv=Hkv, D=D, causal=True, type=type_)
    causal = rng.random() < 0.6
    budget = 3e10 / (B * H * D)  # rows x keys
    most = _log(rng, 2, max(2, min(2048, int(budget ** 0.5))))
    hi = _log(rng, most if causal else 1, max(most, 1, min(8192, int(budget / most))))
    return dict(kind=kind, B=B, n=rng.randint(1, most), most_n=most, lo=rng.randint(min(most, hi), hi) if causal else rng.randint(1, hi), hi=hi, H=H, Hkv=Hkv, D=D, causal=causal, type=type_)


# ---- sizes of a case, the same for every seed (their order among the sequences is the seed's)

def _spread(lo, hi, B):
    return [hi] if B == 1 else [lo + (hi - lo) * i // (B - 1) for i in range(B)]


def _sizes(case):
    """(new rows, tokens in the cache with them) of each sequence."""
    most, least = (case["most_new"], case["new"]) if case["kind"] == "cache" else (case["most_n"], case["n"])
    rows, lens = _spread(least, most, case["B"]), _spread(case["lo"], case["hi"], case["B"])
    if case["kind"] == "attn" and not case["causal"]:
        return rows, lens
    return rows, [max(a, b) for a, b in zip(rows, lens)]


# ---- inputs, made from the seed alone

def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _starts(rows):
    return list(itertools.accumulate(rows, initial=0))


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    D, Hkv, type_ = case["D"], case["Hkv"], TYPES[case["type"]]
    s = dict(case=case)
    if case["kind"] == "rope":
        T, H, R = case["T"], case["H"], case["rot"]
        # rows as a projection leaves them: q | k | v side by side, channels of unequal size
        s["qkv"] = (_normal(g, T, (H + 2 * Hkv) * D) * torch.exp(0.5 * _normal(g, (H + 2 * Hkv) * D))).to(type_)
        s["wq"], s["wk"] = 1 + 0.2 * _normal(g, D), 1 + 0.2 * _normal(g, D)
        s["inv_freq"] = 10000.0 ** (-torch.arange(0, R, 2, device="cuda", dtype=torch.float64) / R)
        s["positions"] = torch.randint(0, case["far"], (T,), generator=g, device="cuda", dtype=torch.int32)
        s["q_out"], s["k_out"] = torch.empty(T, H * D, device="cuda", dtype=type_), torch.empty(T, Hkv * D, device="cuda", dtype=type_)
        return s
    rows, lens = _sizes(case)
    order = torch.randperm(case["B"], generator=g, device="cuda").tolist()
    rows, lens = [rows[i] for i in order], [lens[i] for i in order]
    B, blocks = case["B"], [-(-n // BLOCK) for n in lens]
    pages = sum(blocks) + 3
    ids = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((B, max(blocks)), -1, dtype=torch.int32, device="cuda")  # behind a sequence's last page: no page
    at = _starts(blocks)
    table[torch.arange(max(blocks), device="cuda")[None] < _int32(blocks)[:, None]] = ids[:at[-1]]
    s.update(rows=rows, lens=lens, starts=_int32(_starts(rows)), seq_len=_int32(lens), table=table, T=sum(rows), pages=pages)
    channel = torch.exp(0.7 * _normal(g, 2, Hkv, 1, D))  # some channels are larger than others, in K above all
    s["k_cache"], s["k_scale"] = _pack(_normal(g, pages, Hkv, BLOCK, D) * channel[0], False)
    s["v_cache"], s["v_scale"] = _pack(_normal(g, pages, Hkv, BLOCK, D) * channel[1] ** 0.3, True)
    if case["kind"] == "cache":
        s["k"] = (_normal(g, s["T"], Hkv, D) * 1.3 * channel[0, :, 0]).to(type_)
        s["v"] = (_normal(g, s["T"], Hkv, D) * 1.3 * channel[1, :, 0] ** 0.3).to(type_)
        s["back"] = [min(n, case["back"] or n) for n in lens]
        s["back_starts"], s["back_T"] = _int32(_starts(s["back"])), sum(s["back"])
        s["k_out"], s["v_out"] = (torch.empty(s["back_T"], Hkv * D, device="cuda", dtype=type_) for _ in range(2))
    else:
        s["q"] = _normal(g, s["T"], case["H"] * D).to(type_)
        s["out"] = torch.empty_like(s["q"])
    return s


# ---- the cache's layout and numbers, in torch

def _exponent(amax):
    """The smallest exponent byte whose scale brings amax under e4m3's largest value; 0 for zeros."""
    m, x = torch.frexp(amax.double())  # amax = m 2^x, 1/2 <= m < 1; 448 = (7/8) 2^9
    e = x + (m > 0.875).to(x.dtype) - 9 + 127
    return torch.where(amax > 0, e.clamp(0, 254), torch.zeros_like(e))


def _scaled(x, e):
    """x 2^(127 - e), e a byte: in 32 bits by two factors, each a power of two."""
    h = (127 - e).div(2, rounding_mode="floor")
    return x * torch.exp2(h.float()) * torch.exp2((127 - e - h).float())


def _codes(x):
    return x.to(torch.float8_e4m3fn)


def _layout(c, is_v):
    """e4m3 values [pages, Hkv, token, D] as the bytes of the pages."""
    P, H, _, D = c.shape
    c = c.view(torch.uint8)
    if is_v:
        out = torch.empty(P, H, D, BLOCK, dtype=torch.uint8, device=c.device)
        out[..., torch.tensor(SLOT, device=c.device)] = c.transpose(2, 3)
        return out
    return c.view(P, H, BLOCK, D // 32, 32).transpose(2, 3).contiguous()


def _values(cache, scale, is_v):
    """The float32 values [..., Hkv, token, D] of pages' bytes and exponents."""
    if is_v:
        x = cache[..., torch.tensor(SLOT, device=cache.device)].transpose(-1, -2)
    else:
        x = cache.transpose(-2, -3).flatten(-2)
    return _scaled(x.contiguous().view(torch.float8_e4m3fn).float(), (254 - scale.int())[..., None, None])


def _pack(x, is_v):
    e = _exponent(x.abs().amax((2, 3)))
    return _layout(_codes(_scaled(x, e[..., None, None])), is_v), e.to(torch.uint8)


# ---- one pass

def run(state):
    kind = state["case"]["kind"]
    if own:
        return _own(state)
    return _rope(state) if kind == "rope" else _cache(state) if kind == "cache" else _attn(state)


def _rope(s):
    c = s["case"]
    T, H, Hkv, D, R = (c[k] for k in ("T", "H", "Hkv", "D", "rot"))
    angle = s["positions"].double()[:, None] * s["inv_freq"]
    cos, sin = (f(angle).float()[:, None] for f in (torch.cos, torch.sin))

    def one(x, w):
        x = x.float()
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
        turned, rest = y[..., :R], y[..., R:]
        if c["pairs"] == "half":
            a, b = turned[..., :R // 2], turned[..., R // 2:]
            turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        else:
            a, b = turned[..., 0::2], turned[..., 1::2]
            turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        return torch.cat((turned, rest), -1).to(TYPES[c["type"]]).flatten(1)

    q, k = s["qkv"][:, :H * D].view(T, H, D), s["qkv"][:, H * D:(H + Hkv) * D].view(T, Hkv, D)
    return [one(q, s["wq"]), one(k, s["wk"])]


def _places(s, rows, starts, T):
    """Sequence and position of each row."""
    rows_t = starts[1:] - starts[:-1]
    b = torch.repeat_interleave(torch.arange(len(rows), device="cuda"), rows_t.long(), output_size=T)
    return b, torch.arange(T, device="cuda") - starts[b] + s["seq_len"][b] - rows_t[b]


def _cache(s):
    Hkv, D, type_ = s["case"]["Hkv"], s["case"]["D"], TYPES[s["case"]["type"]]
    b, at = _places(s, s["rows"], s["starts"], s["T"])
    first = (s["seq_len"] - s["starts"].diff()).long()  # the first new token's position
    width = s["table"].shape[1]
    block = torch.arange(width, device="cuda")[None]
    touched = (block >= (first // BLOCK)[:, None]) & (block * BLOCK < s["seq_len"][:, None])
    seq, blk = touched.nonzero(as_tuple=True)
    page = s["table"][seq, blk].long()
    where = torch.full((len(s["rows"]), width), -1, device="cuda", dtype=torch.int64)
    where[seq, blk] = torch.arange(len(seq), device="cuda")
    mine, slot = where[b, at // BLOCK], at % BLOCK
    kept = (blk[:, None] * BLOCK + torch.arange(BLOCK, device="cuda") < first[seq][:, None])[:, None, :, None]
    new = torch.zeros(len(seq), BLOCK, dtype=torch.bool, device="cuda")
    new[mine, slot] = True
    new = new[:, None, :, None]
    outs = {}
    for name, is_v in (("k", False), ("v", True)):
        cache, scale = s[name + "_cache"], s[name + "_scale"]
        old = _values(cache[page], scale[page], is_v)
        x = torch.zeros(len(seq), BLOCK, Hkv, D, device="cuda")
        x[mine, slot] = s[name].float()
        x = x.transpose(1, 2)
        e = _exponent(x.abs().amax((2, 3)))
        e = torch.where(kept.any(2)[..., 0], torch.maximum(e, scale[page].to(e.dtype)), e)
        codes = _codes(_scaled(torch.where(kept, old, x), e[..., None, None]))
        codes = torch.where(kept | new, codes.view(torch.uint8), _codes(_scaled(old, scale[page].int()[..., None, None])).view(torch.uint8))
        cache[page], scale[page] = _layout(codes.view(torch.float8_e4m3fn), is_v), e.to(torch.uint8)
        rb, rat = _places(s, s["back"], s["back_starts"], s["back_T"])
        p = s["table"][rb, rat // BLOCK].long()
        bytes_ = cache[p, :, :, torch.tensor(SLOT, device="cuda")[rat % BLOCK]] if is_v else cache[p, :, :, rat % BLOCK].flatten(2)
        outs[name] = _scaled(bytes_.contiguous().view(torch.float8_e4m3fn).float(), 254 - scale[p].int()[..., None]).to(type_).flatten(1)
        outs[name + "_scale"] = scale
    return outs


def _attn(s):
    c = s["case"]
    H, Hkv, D = c["H"], c["Hkv"], c["D"]
    G, B, N, L = H // Hkv, c["B"], max(s["rows"]), s["table"].shape[1] * BLOCK
    pages = s["table"].clamp(min=0).long()
    k = _values(s["k_cache"][pages], s["k_scale"][pages], False).permute(0, 2, 4, 1, 3).reshape(B, Hkv, D, L)
    v = _values(s["v_cache"][pages], s["v_scale"][pages], True).permute(0, 2, 1, 3, 4).reshape(B, Hkv, L, D)
    b, at = _places(s, s["rows"], s["starts"], s["T"])
    n = at - s["seq_len"][b] + (s["starts"].diff())[b]  # a row's number in its sequence
    q = torch.zeros(B, N, H, D, device="cuda")
    q[b, n] = s["q"].view(-1, H, D).float()
    q = q.view(B, N, Hkv, G, D).transpose(1, 2).reshape(B, Hkv, N * G, D)
    key = torch.arange(L, device="cuda")
    seen = (key < s["seq_len"][:, None])[:, None].expand(B, N, L)
    if c["causal"]:
        seen = seen & (key <= (s["seq_len"] - s["starts"].diff())[:, None, None] + torch.arange(N, device="cuda")[:, None])
    seen = seen[:, None, :, None].expand(B, Hkv, N, G, L).reshape(B, Hkv, N * G, L)
    score = (q @ k).mul_(D ** -0.5).masked_fill_(~seen, -torch.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(torch.isfinite(top), top, 0)).exp_()
    o = (p @ v) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = o.view(B, Hkv, N, G, D).transpose(1, 2).reshape(B, N, H * D)
    return o[b, n].to(TYPES[c["type"]])


# ---- the framework's calls

def _own(s):
    if "calls" not in s:
        s["calls"], s["outs"] = _calls(s)
    stream = torch.cuda.current_stream().cuda_stream
    for f, args in s["calls"]:
        f(args, stream)
    return s["outs"]


def _calls(s):
    """The argument structs that a program keeps beside its buffers."""
    path = os.path.join(os.getcwd(), "supra2-img-web_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from supra_attn import _lib

    c, ptr = s["case"], torch.Tensor.data_ptr
    D, Hkv = c["D"], c["Hkv"]
    dtype = _lib.SA_DT[c["type"].upper()]
    if c["kind"] == "rope":
        H, ld = c["H"], (c["H"] + 2 * c["Hkv"]) * D
        args = _lib.QkRopeArgs(dtype=dtype, T=c["T"], H=H, Hkv=Hkv, D=D, rotary_dim=c["rot"], pairs=_lib.SA_ROPE_HALF if c["pairs"] == "half" else _lib.SA_ROPE_NEAR,
                               norm=_lib.SA_NORM_RMS, eps=1e-6, q=ptr(s["qkv"]), k=ptr(s["qkv"]), k_off=H * D, ldq=ld, ldk=ld, q_out=ptr(s["q_out"]), k_out=ptr(s["k_out"]),
                               q_weight=ptr(s["wq"]), k_weight=ptr(s["wk"]), inv_freq=ptr(s["inv_freq"]), positions=ptr(s["positions"]))
        return [(_lib.qk_norm_rope, args)], [s["q_out"], s["k_out"]]
    cache = _lib.KvCache(pages=s["pages"], Hkv=Hkv, D=D, k=ptr(s["k_cache"]), v=ptr(s["v_cache"]), k_scale=ptr(s["k_scale"]), v_scale=ptr(s["v_scale"]))
    common = dict(seq_len=ptr(s["seq_len"]), block_table=ptr(s["table"]), B=c["B"], max_blocks=s["table"].shape[1])
    seqs = _lib.KvSeqs(row_start=ptr(s["starts"]), T=s["T"], max_rows=max(s["rows"]), **common)
    if c["kind"] == "cache":
        back = _lib.KvSeqs(row_start=ptr(s["back_starts"]), T=s["back_T"], max_rows=max(s["back"]), **common)
        return ([(_lib.kv_write, _lib.KvRowsArgs(dtype=dtype, cache=cache, seqs=seqs, k=ptr(s["k"]), v=ptr(s["v"]))),
                 (_lib.kv_read, _lib.KvRowsArgs(dtype=dtype, cache=cache, seqs=back, k=ptr(s["k_out"]), v=ptr(s["v_out"])))],
                dict(k=s["k_out"], v=s["v_out"], k_scale=s["k_scale"], v_scale=s["v_scale"]))
    args = _lib.KvAttnArgs(dtype=dtype, cache=cache, seqs=seqs, H=c["H"], causal=int(c["causal"]), scale=D ** -0.5, max_len=max(s["lens"]), q=ptr(s["q"]), o=ptr(s["out"]))
    need = _lib.kv_attention_workspace_bytes(args)
    if need:
        s["workspace"] = torch.empty(need, dtype=torch.uint8, device="cuda")
        args.workspace, args.workspace_bytes = ptr(s["workspace"]), need
    return [(_lib.kv_attention, args)], s["out"]


# ---- the work a pass cannot do without

def work(case):
    size, D, Hkv = TYPES[case["type"]].itemsize, case["D"], case["Hkv"]
    if case["kind"] == "rope":
        T, heads = case["T"], case["H"] + Hkv
        return {"bytes": T * (2 * heads * D * size + 4) + 8 * D + 4 * case["rot"], "flops": T * heads * (4 * D + 3 * case["rot"])}
    rows, lens = _sizes(case)
    blocks = sum(-(-n // BLOCK) for n in lens)
    if case["kind"] == "cache":
        back = [min(n, case["back"] or n) for n in lens]
        # rows read and their bytes written; bytes read back and rows written; the exponents
        new, old = sum(rows), sum(back)
        return {"bytes": 2 * Hkv * D * (new + old) * (size + 1) + 4 * Hkv * (new + old) // BLOCK + 4 * blocks, "flops": 2 * Hkv * D * (2 * new + old)}
    if case["causal"]:  # row t of n sees len - n + t + 1 keys
        pairs = sum(n * l - n * (n - 1) // 2 for n, l in zip(rows, lens))
    else:
        pairs = sum(n * l for n, l in zip(rows, lens))
    H = case["H"]
    return {"bytes": 2 * sum(lens) * Hkv * D + 2 * blocks * Hkv + 4 * blocks + 2 * sum(rows) * H * D * size, "flops": 4 * D * H * pairs}


# ---- the definition, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    D, Hkv = case["D"], case["Hkv"]
    if case["kind"] == "rope":
        T, R = case["T"], case["rot"]
        i = torch.arange(R // 2, device="cuda")
        first, second = (i, i + R // 2) if case["pairs"] == "half" else (2 * i, 2 * i + 1)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["positions"].double()[:, None] * s["inv_freq"])[:, None]
        outs = []
        for at, heads, w in ((0, case["H"], s["wq"]), (case["H"] * D, Hkv, s["wk"])):
            x = s["qkv"][:, at:at + heads * D].double().reshape(T, heads, D)
            x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / D + 1e-6) * w.double()
            z = torch.complex(x[..., first], x[..., second]) * turn
            x[..., first], x[..., second] = z.real, z.imag
            outs.append(x.reshape(T, heads * D))
        return outs
    # e4m3: sign, four exponent bits of bias 7, three bits of fraction
    code = torch.arange(256, device="cuda")
    ex, fr = code // 8 % 16, (code % 8).double()
    table = torch.where(ex == 0, fr / 8 * 2.0 ** -6, (1 + fr / 8) * torch.exp2(ex.double() - 7)) * torch.where(code < 128, 1.0, -1.0)
    token, slot = torch.arange(BLOCK, device="cuda"), torch.tensor(SLOT, device="cuda")

    def stored(name, b, length):
        """[length, Hkv, D] values of sequence b."""
        ids = s["table"][b, :-(-length // BLOCK)].long()
        raw = s[name + "_cache"][ids].long()
        x = table[raw[..., slot]].permute(0, 3, 1, 2) if name == "v" else table[raw].permute(0, 3, 1, 2, 4).flatten(3)
        x = x * torch.exp2(s[name + "_scale"][ids].double() - 127)[:, None, :, None]
        return x.reshape(-1, Hkv, D)[:length]

    starts = s["starts"].tolist()
    if case["kind"] == "attn":
        G, outs = case["H"] // Hkv, []
        for b, (n, length) in enumerate(zip(s["rows"], s["lens"])):
            k, v = stored("k", b, length), stored("v", b, length)
            q = s["q"][starts[b]:starts[b] + n].double().view(n, Hkv, G, D)
            out = torch.zeros(n, Hkv, G, D, dtype=torch.float64, device="cuda")
            for h in range(Hkv):
                z = (q[:, h].reshape(n * G, D) @ k[:, h].T.contiguous()) * D ** -0.5
                if case["causal"]:
                    z += torch.where(torch.arange(length, device="cuda") > (length - n + torch.arange(n, device="cuda"))[:, None], -torch.inf, 0.0).repeat_interleave(G, 0)
                out[:, h] = (torch.softmax(z, -1) @ v[:, h]).view(n, G, D)
            outs.append(out.reshape(n, case["H"] * D))
        return torch.cat(outs)
    # the cache: old tokens of a page keep their steps unless a larger new one makes the page's scale grow
    grid = torch.cat((table[:127], -table[1:127])).sort().values
    limit, outs = (grid[1:] + grid[:-1]) / 2, {}

    def nearest(x):
        """The e4m3 value nearest to x; of two as near, the one whose last fraction bit is 0."""
        i = torch.bucketize(x, limit)
        up = (i + 1).clamp(max=len(grid) - 1)
        mantissa = torch.frexp(grid[up].abs()).mantissa * 16
        even = torch.where(grid[up].abs() < 2.0 ** -6, grid[up].abs() * 2.0 ** 9 % 2 == 0, mantissa % 2 == 0)
        tie = (i < len(limit)) & (x == limit[i.clamp(max=len(limit) - 1)])
        return torch.where(tie & even, grid[up], grid[i])

    for name in ("k", "v"):
        scale, back = s[name + "_scale"].long(), []
        for b, (n, length) in enumerate(zip(s["rows"], s["lens"])):
            begin = length - n
            blocks = -(-length // BLOCK)
            x = torch.zeros(blocks * BLOCK, Hkv, D, dtype=torch.float64, device="cuda")
            x[begin:length] = s[name][starts[b]:starts[b] + n].double()
            large = x.view(blocks, BLOCK, Hkv, D).abs().amax((1, 3))
            e = torch.ceil(torch.log2(large / E4M3_MAX)).clamp(min=-127)
            e += (large > E4M3_MAX * torch.exp2(e)).double() - (large <= E4M3_MAX * torch.exp2(e - 1)).double()
            e = e.clamp(min=-127)
            ids = s["table"][b, :blocks].long()
            was = (scale[ids] - 127).double()
            first = begin // BLOCK
            number = torch.arange(blocks, device="cuda")[:, None]
            e = torch.where((number == first) & (begin % BLOCK > 0), torch.maximum(e, was), e)
            e = torch.where(number < first, was, e)
            x[:begin] = stored(name, b, length)[:begin]
            step = torch.exp2(e).repeat_interleave(BLOCK, 0)[..., None]
            back.append((nearest(x / step) * step)[length - s["back"][b]:length].reshape(-1, Hkv * D))
            scale[ids] = (e + 127).long()
        outs[name], outs[name + "_scale"] = torch.cat(back), None
    return outs
