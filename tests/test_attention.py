"""Attention over prompts and over a paged key-value cache, and the calls that keep the cache, against plain implementations in 64 bits.

Tolerances.  With u the half step of the type (bf16 2^-8, fp16 2^-11, fp32 2^-24) and A = sum_j p_j |v_j| / sum_j p_j, an output o is off by at most
    u |o|              its own rounding
    u A                16 bits: the weights are rounded before they multiply the values
    2 delta A          weights from scores that are off by delta, in the sum above and in the one below the fraction
    (n 2^-23 + 2^-20) A    n additions that may cut off, exp2 (2^-22), products of split operands (2^-20)
with delta = scale B (d 2^-23 + 2^-20) for d additions of products of size B = max sum |q| |k| in all.
"""
import ctypes as C
import math

import numpy as np
import pytest

from aspen_b200 import api

HALF = {api.FP32: 2.0 ** -24, api.BF16: 2.0 ** -8, api.FP16: 2.0 ** -11}
NAMES = {api.FP32: "fp32", api.BF16: "bf16", api.FP16: "fp16"}
TYPES = [api.FP32, api.BF16, api.FP16]
ids = NAMES.get


def torch_type(kind):
    import torch
    return {api.FP32: torch.float32, api.BF16: torch.bfloat16, api.FP16: torch.float16}[kind]


def rounded(a, kind):
    """Values of the type, in 64 bits."""
    import torch
    return torch.from_numpy(np.asarray(a, dtype=np.float32)).to(torch_type(kind)).double().numpy()


def to_device(a, kind):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).to(torch_type(kind)).cuda()


def ints(a):
    import torch
    return torch.tensor(np.asarray(a, dtype=np.int32)).cuda()


def attend(q, k, v, scale, seen):
    """q [n][H][d], k, v [m][KV][d], seen [n][m]: outputs and their tolerance without the type's part, [n][H][d] each, and A."""
    n, H, d = q.shape
    group = H // k.shape[1]
    out, away, size = np.zeros((n, H, d)), np.zeros((n, H, d)), np.zeros((n, H, d))
    for h in range(H):
        kk, vv = k[:, h // group], v[:, h // group]
        s = q[:, h] @ kk.T * scale
        products = np.abs(q[:, h]) @ np.abs(kk.T) * abs(scale)
        with np.errstate(invalid="ignore"):
            s = np.where(seen, s, -np.inf)
            p = np.exp(s - np.max(s, axis=1, keepdims=True, initial=-1e300))
        total = p.sum(1, keepdims=True)
        w = np.divide(p, total, out=np.zeros_like(p), where=total > 0)
        out[:, h] = w @ vv
        size[:, h] = w @ np.abs(vv)
        B = np.max(np.where(seen, products, 0), axis=1, initial=0)
        delta = B * (d * 2.0 ** -23 + 2.0 ** -20)
        away[:, h] = size[:, h] * (2 * delta + k.shape[0] * 2.0 ** -23 + 2.0 ** -20)[:, None]
    return out, away, size


def check(got, want, away, size, kind):
    got = got.float().cpu().numpy().astype(np.float64)
    u = HALF[kind]
    bound = u * np.abs(want) + away + (u * size if kind != api.FP32 else 0) + 1e-30
    assert np.isfinite(got).all()
    worst = np.max(np.abs(got - want) / bound, initial=0)
    assert worst <= 1, f"off by {worst:.2f} of the tolerance, at {np.unravel_index(np.argmax(np.abs(got - want) / bound), got.shape)}"


# ---- a pool with its books ---------------------------------------------------------------------------------------------------

class Pool:
    """A cache on the device, with values that would show if they were used: everything outside live tokens is NaN."""

    def __init__(self, kind, kv_heads, dim, page, pages, sequences, max_pages, layers=1, strides=None):
        import torch
        self.kind, self.shape = kind, (layers, pages, kv_heads, page, dim)
        self.k, self.v = (torch.full(self.shape, math.nan, dtype=torch_type(kind), device="cuda") for _ in range(2))
        self.table, self.lengths, self.refs, self.status = ints(np.full((sequences, max_pages), -1)), ints(np.zeros(sequences)), ints(np.zeros(pages)), ints([0])
        self.cache = api.Cache(type=kind, layers=layers, pages=pages, page_size=page, kv_heads=kv_heads, head_dim=dim, sequences=sequences, max_pages=max_pages,
                               k=self.k.data_ptr(), v=self.v.data_ptr(), page_table=self.table.data_ptr(), lengths=self.lengths.data_ptr(),
                               refs=self.refs.data_ptr(), status=self.status.data_ptr())

    def space(self, entries):
        import torch
        need = self.cache.workspace(entries)
        self._space = torch.full((need,), 0x5a, dtype=torch.uint8, device="cuda")
        return self._space.data_ptr(), need

    def fill(self, lengths, rng, order=None):
        """Sequences of these lengths with random keys and values; the pages in a random order."""
        pages, page = self.shape[1], self.shape[3]
        order = rng.permutation(pages) if order is None else order
        table, refs, at = self.table.cpu().numpy(), np.zeros(pages, np.int32), 0
        k, v = (np.full(self.shape, np.nan) for _ in range(2))
        for s, n in enumerate(lengths):
            for i in range(-(-n // page)):
                p = order[at]
                at += 1
                table[s, i], refs[p] = p, 1
                used = min(page, n - i * page)
                for a in (k, v):
                    a[:, p, :, :used] = rounded(rng.standard_normal(a[:, p, :, :used].shape), self.kind)
        self.k.copy_(to_device(k, self.kind)); self.v.copy_(to_device(v, self.kind))
        self.table.copy_(ints(table)); self.refs.copy_(ints(refs))
        self.lengths.copy_(ints(list(lengths) + [0] * (self.lengths.numel() - len(lengths))))
        self.host_k, self.host_v, self.host_table = k, v, table

    def tokens(self, s, n, layer=0):
        page = self.shape[3]
        rows = [(self.host_table[s, t // page], t % page) for t in range(n)]
        shape = (n, self.shape[2], self.shape[4])
        k = np.array([self.host_k[layer, p, :, r] for p, r in rows]).reshape(shape)
        v = np.array([self.host_v[layer, p, :, r] for p, r in rows]).reshape(shape)
        return k, v

    def books(self):
        return [x.cpu().numpy().copy() for x in (self.table, self.lengths, self.refs, self.status)]


def decode(pool, q, heads, slots=None, scale=None, layer=0, stream=0, **strides):
    import torch
    n = q.shape[0] if slots is None else len(slots)
    out = torch.full_like(q, math.nan)
    need = pool.cache.decode_workspace(n, heads)
    space = torch.full((need,), 0x7f, dtype=torch.uint8, device="cuda")
    at = ints(slots) if slots is not None else None
    args = api.DecodeArgs(entries=n, heads=heads, scale=scale if scale is not None else q.shape[-1] ** -0.5, q=q.data_ptr(), out=out.data_ptr(),
                          slots=at.data_ptr() if at is not None else 0, workspace=space.data_ptr(), workspace_bytes=need, **strides)
    pool.cache.decode(layer, args, stream)
    torch.cuda.synchronize()
    return out


def decode_want(pool, q, slots, lengths, scale):
    parts = []
    for i, s in enumerate(slots):
        k, v = pool.tokens(s, lengths[s])
        parts.append(attend(q[i:i + 1], k, v, scale, np.ones((1, lengths[s]), bool)))
    return [np.concatenate(p) for p in zip(*parts)]


# ---- refusals: nothing of these reaches a GPU --------------------------------------------------------------------------------

def good_cache(**change):
    c = dict(type=api.BF16, layers=2, pages=8, page_size=16, kv_heads=2, head_dim=64, sequences=4, max_pages=3, k=4096, v=8192, page_table=64, lengths=128,
             refs=192, status=256)
    c.update(change)
    return api.Cache(**c)


BAD_CACHES = [(dict(type=3), -1), (dict(type=-1), -1), (dict(head_dim=0), -1), (dict(head_dim=12), -1), (dict(head_dim=264), -1), (dict(page_size=0), -1),
              (dict(pages=0), -1), (dict(layers=0), -1), (dict(kv_heads=0), -1), (dict(sequences=0), -1), (dict(max_pages=0), -1), (dict(k=0), -1), (dict(v=0), -1),
              (dict(k=4104), -1), (dict(page_table=0), -1), (dict(lengths=0), -1), (dict(status=0), -1), (dict(token_stride=65), -1), (dict(head_stride=4), -1),
              (dict(page_stride=1001), -1), (dict(layer_stride=4), -1), (dict(page_size=2**20, max_pages=2**12), -2), (dict(pages=2**31), -2), (dict(layers=1025), -2),
              (dict(token_stride=2**30), -2), (dict(page_stride=2**31), -2)]


@pytest.mark.parametrize("change,rc", BAD_CACHES, ids=lambda c: "-".join(c) if isinstance(c, dict) else str(c))
def test_a_cache_that_cannot_be_is_refused(change, rc):
    L, c = api.lib(), good_cache(**change)
    call = api.DecodeArgs(entries=1, heads=2, scale=1.0, q=4096, out=4096, workspace=4096, workspace_bytes=1 << 30)
    rows = api.AppendArgs(k=4096, v=4096, entries=1, rows=1)
    assert L.aspen_b200_attention_decode(C.byref(c), 0, C.byref(call), None) == rc
    assert L.aspen_b200_cache_append(C.byref(c), 0, C.byref(rows), None) == rc
    assert L.aspen_b200_cache_extend(C.byref(c), None, None, 1, 4096, 1 << 30, None) == rc
    assert L.aspen_b200_cache_fork(C.byref(c), 64, 64, 1, 4096, 1 << 30, None) == rc
    assert L.aspen_b200_cache_free(C.byref(c), 64, 1, None) == rc
    assert L.aspen_b200_cache_compact(C.byref(c), 4096, 1 << 30, None) == rc
    assert L.aspen_b200_cache_copy(C.byref(c), 64, 64, 1, None) == rc
    assert L.aspen_b200_cache_workspace(C.byref(c), 1) == 0
    assert L.aspen_b200_attention_decode_workspace(C.byref(c), 1, 2) == 0


def test_calls_on_the_cache_refuse_what_they_cannot_do():
    L, c = api.lib(), good_cache()
    need = L.aspen_b200_cache_workspace(C.byref(c), 5)
    assert need > 0 and need % 4 == 0 and L.aspen_b200_cache_workspace(C.byref(c), 0) <= need
    assert L.aspen_b200_cache_extend(C.byref(c), None, None, 5, None, need, None) == -1
    assert L.aspen_b200_cache_extend(C.byref(c), None, None, 5, 4096, need - 1, None) == -1
    assert str(need) in api.last_error()
    assert L.aspen_b200_cache_extend(C.byref(c), None, None, 5, 4097, need, None) == -1
    assert L.aspen_b200_cache_extend(C.byref(c), None, None, 2**31, 4096, 1 << 40, None) == -2
    assert L.aspen_b200_cache_extend(C.byref(c), None, None, 0, 4096, need, None) == 0
    assert L.aspen_b200_cache_fork(C.byref(c), None, 64, 1, 4096, need, None) == -1
    assert L.aspen_b200_cache_fork(C.byref(c), 64, None, 1, 4096, need, None) == -1
    assert L.aspen_b200_cache_free(C.byref(c), None, 1, None) == -1
    assert L.aspen_b200_cache_compact(C.byref(c), 4096, 8, None) == -1
    assert L.aspen_b200_cache_copy(C.byref(c), None, 64, 1, None) == -1
    assert L.aspen_b200_cache_extend(None, None, None, 5, 4096, need, None) == -1
    for change, rc in [(dict(k=0), -1), (dict(k=4098), -1), (dict(k_row_stride=129), -1), (dict(v_head_stride=2**29), -2), (dict(entries=2), -1), (dict(entries=0), -1)]:
        a = dict(k=4096, v=4096, entries=1, rows=1)
        a.update(change)
        assert L.aspen_b200_cache_append(C.byref(c), 0, C.byref(api.AppendArgs(**a)), None) == rc, change
    assert L.aspen_b200_cache_append(C.byref(c), 2, C.byref(api.AppendArgs(k=4096, v=4096, entries=1, rows=1)), None) == -1
    assert L.aspen_b200_cache_append(C.byref(c), 0, None, None) == -1
    for change, rc in [(dict(heads=3), -1), (dict(heads=0), -1), (dict(q=0), -1), (dict(out=8), -1), (dict(scale=math.inf), -1), (dict(scale=math.nan), -1), (dict(workspace=0), -1),
                       (dict(workspace=4100), -1), (dict(entries=5), -1), (dict(entries=2**30), -2), (dict(q_row_stride=12), -1)]:
        a = dict(entries=1, heads=4, scale=1.0, q=4096, out=4096, workspace=4096, workspace_bytes=1 << 30)
        a.update(change)
        assert L.aspen_b200_attention_decode(C.byref(c), 0, C.byref(api.DecodeArgs(**a)), None) == rc, change
    assert L.aspen_b200_attention_decode(C.byref(c), 2, C.byref(api.DecodeArgs(entries=1, heads=2, scale=1.0, q=4096, out=4096, workspace=4096, workspace_bytes=1 << 30)), None) == -1
    assert L.aspen_b200_attention_decode(C.byref(c), 0, None, None) == -1
    with pytest.raises(RuntimeError, match="layer 7"):
        c.append(7, api.AppendArgs(k=4096, v=4096, entries=1, rows=1))


def test_a_prompt_that_cannot_be_is_refused():
    L = api.lib()
    good = dict(type=api.FP16, heads=4, kv_heads=2, head_dim=64, scale=1.0, sequences=1, q_rows=3, kv_rows=3, q_starts=64, kv_starts=64, q=4096, k=4096, v=4096, out=8192)
    for change, rc in [(dict(type=7), -1), (dict(heads=5), -1), (dict(heads=0), -1), (dict(kv_heads=0), -1), (dict(head_dim=20), -1), (dict(head_dim=512), -1), (dict(scale=math.nan), -1),
                       (dict(q=0), -1), (dict(k=0), -1), (dict(v=0), -1), (dict(out=0), -1), (dict(q=4100), -1), (dict(q_starts=0), -1), (dict(kv_starts=0), -1),
                       (dict(out_row_stride=257), -1), (dict(k_head_stride=2**30), -2), (dict(q_rows=2**31), -2), (dict(sequences=2**24 + 1), -2), (dict(heads=2**16, kv_heads=2**16), -2)]:
        assert L.aspen_b200_attention_prompt(C.byref(api.PromptArgs(**{**good, **change})), None) == rc, change
    assert L.aspen_b200_attention_prompt(None, None) == -1
    for change in (dict(sequences=0), dict(q_rows=0)):
        assert L.aspen_b200_attention_prompt(C.byref(api.PromptArgs(**{**good, **change})), None) == 0


def test_calls_without_a_gpu_say_so():
    import torch
    if torch.cuda.is_available():
        pytest.skip("there is one")
    L, c = api.lib(), good_cache()
    assert L.aspen_b200_attention_decode_workspace(C.byref(c), 1, 2) == 0
    assert L.aspen_b200_cache_extend(C.byref(c), None, None, 1, 4096, 1 << 20, None) == -3
    assert L.aspen_b200_cache_compact(C.byref(c), 4096, 1 << 20, None) == -3
    good = dict(type=api.FP16, heads=4, kv_heads=2, head_dim=64, scale=1.0, sequences=1, q_rows=3, kv_rows=3, q_starts=64, kv_starts=64, q=4096, k=4096, v=4096, out=8192)
    assert L.aspen_b200_attention_prompt(C.byref(api.PromptArgs(**good)), None) == -3


# ---- one new token over the cache --------------------------------------------------------------------------------------------

@pytest.mark.gpu
def test_host_memory_is_refused():
    import torch
    host, dev = torch.zeros(1 << 16, dtype=torch.uint8), torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    p = (host.data_ptr() + 15) // 16 * 16
    L, d = api.lib(), dev.data_ptr()
    pinned = torch.zeros(1 << 12, dtype=torch.uint8, pin_memory=True)
    assert L.aspen_b200_attention_prompt(C.byref(api.PromptArgs(type=api.FP16, heads=1, kv_heads=1, head_dim=8, scale=1.0, sequences=1, q_rows=1, kv_rows=1, q_starts=d, kv_starts=d,
                                                               q=pinned.data_ptr(), k=d, v=d, out=d + 4096)), None) == -1
    good = dict(type=api.FP16, heads=1, kv_heads=1, head_dim=8, scale=1.0, sequences=1, q_rows=1, kv_rows=1, q_starts=d, kv_starts=d, q=d, k=d, v=d, out=d + 4096)
    for name in ("q", "k", "v", "out", "q_starts", "kv_starts"):
        assert L.aspen_b200_attention_prompt(C.byref(api.PromptArgs(**{**good, name: p})), None) == -1, name
    for name in ("k", "v", "page_table", "lengths", "refs", "status"):
        c = good_cache(**{"k": d, "v": d, "page_table": d, "lengths": d, "refs": d, "status": d, name: p})
        if name != "k" and name != "v":
            assert L.aspen_b200_cache_extend(C.byref(c), None, None, 1, d, 1 << 20, None) == -1, name
        if name != "refs":
            call = api.DecodeArgs(entries=1, heads=2, scale=1.0, q=d, out=d, workspace=d, workspace_bytes=1 << 30)
            assert L.aspen_b200_attention_decode(C.byref(c), 0, C.byref(call), None) == -1, name


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES, ids=ids)
@pytest.mark.parametrize("heads,kv_heads,dim,page,lengths", [
    (1, 1, 8, 1, [1]), (12, 12, 64, 16, [37, 0, 1, 16, 17, 300]), (8, 2, 80, 7, [100, 33, 1, 250]), (28, 4, 128, 32, [513, 64, 5]), (12, 1, 64, 16, [90, 400]),
    (20, 1, 128, 16, [77, 160]), (16, 2, 256, 64, [129, 1, 31]), (36, 2, 256, 3, [50]), (3, 3, 96, 256, [700, 2]), (16, 4, 32, 16, [1000] * 9), (4, 4, 64, 16, list(range(1, 60)))])
def test_a_token_attends_to_all_pages_of_its_sequence(heads, kv_heads, dim, page, lengths, kind):
    rng = np.random.default_rng(dim + page)
    most = -(-max(lengths) // page)
    pool = Pool(kind, kv_heads, dim, page, sum(-(-n // page) for n in lengths) + 3, len(lengths) + 1, most + 2)
    pool.fill(lengths, rng)
    q = rounded(rng.standard_normal((len(lengths), heads, dim)) * 1.5, kind)
    got = decode(pool, to_device(q, kind), heads)
    want, away, size = decode_want(pool, q, range(len(lengths)), lengths, dim ** -0.5)
    check(got, want, away, size, kind)
    assert pool.status.item() == 0
    again = decode(pool, to_device(q, kind), heads)
    assert got.equal(again)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES, ids=ids)
def test_a_long_sequence_is_split_and_joined_beside_short_ones(kind):
    rng = np.random.default_rng(5)
    lengths = [30011, 1, 0, 17, 4000]
    pool = Pool(kind, 2, 64, 16, 2200, 6, 1900)
    pool.fill(lengths, rng)
    q = rounded(rng.standard_normal((5, 8, 64)), kind)
    q[0] *= 6                       # a few keys take nearly all weight: the parts' maxima differ
    q = rounded(q, kind)
    want, away, size = decode_want(pool, q, range(5), lengths, 0.125)
    check(decode(pool, to_device(q, kind), 8), want, away, size, kind)


@pytest.mark.gpu
def test_sequences_may_be_named_in_any_order_twice_and_wrongly():
    rng = np.random.default_rng(6)
    lengths = [50, 3, 200]
    pool = Pool(api.FP32, 2, 64, 16, 20, 3, 13)
    pool.fill(lengths, rng)
    slots = [2, 0, 2, 1, -1, 3, 2**31 - 1, -2**31, 0]
    q = rounded(rng.standard_normal((len(slots), 4, 64)), api.FP32)
    got = decode(pool, to_device(q, api.FP32), 4, slots=slots)
    there = [0, 1, 2, 3, 8]
    want, away, size = decode_want(pool, q[there], [slots[i] for i in there], lengths, 0.125)
    check(got[there], want, away, size, api.FP32)
    assert (got[4:8] == 0).all() and pool.status.item() == api.CACHE_BAD_INDEX


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [api.FP32, api.BF16], ids=ids)
def test_tokens_whose_page_does_not_exist_are_left_out_and_lengths_end_with_the_table(kind):
    """Arithmetic of these indices on the CPU: tests/native/attention_index.cpp."""
    import torch
    rng = np.random.default_rng(7)
    lengths = [70, 40, 20]
    pool = Pool(kind, 1, 64, 16, 12, 3, 5)
    pool.fill(lengths, rng)
    table = pool.host_table.copy()
    table[0, 2], table[1, 0], table[1, 1], table[1, 2], table[2, 0], table[2, 1] = -1, 12, 2**31 - 1, -2**31, -7, 99
    pool.table.copy_(ints(table))
    pool.lengths.copy_(ints([70, 40, 2**31 - 1]))
    q = rounded(rng.standard_normal((3, 2, 64)), kind)
    got = decode(pool, to_device(q, kind), 2)
    k, v = pool.tokens(0, 70)
    seen = np.ones((1, 70), bool)
    seen[0, 32:48] = False
    want, away, size = attend(q[:1], k, v, 0.125, seen)
    check(got[:1], want, away, size, kind)
    assert (got[1:] == 0).all()
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [api.FP32, api.FP16], ids=ids)
def test_strides_and_layers_of_a_cache_and_of_queries(kind):
    """Pages of [token][head] order with all layers of a token side by side, queries inside a fused projection."""
    import torch
    rng = np.random.default_rng(8)
    layers, pages, page, kv, dim, heads, lengths = 3, 9, 5, 2, 24, 6, [13, 22, 1]
    k, v = (rounded(rng.standard_normal((pages, page, layers, kv, dim)), kind) for _ in range(2))
    dk, dv = to_device(k, kind), to_device(v, kind)
    pool = Pool(kind, kv, dim, page, pages, 3, 6)
    pool.fill(lengths, rng)
    c = pool.cache
    c.k, c.v, c.layers = dk.data_ptr(), dv.data_ptr(), layers
    c.layer_stride, c.head_stride, c.token_stride, c.page_stride = kv * dim, dim, layers * kv * dim, page * layers * kv * dim
    fused = rounded(rng.standard_normal((3, heads + 2 * kv, dim)), kind)
    q = to_device(fused, kind)
    out = torch.full((3, heads, 2, dim), math.nan, dtype=q.dtype, device="cuda")
    for layer in range(layers):
        pool.host_k, pool.host_v = (a[:, :, layer].transpose(0, 2, 1, 3)[None] for a in (k, v))
        need = c.decode_workspace(3, heads)
        space = torch.empty(need, dtype=torch.uint8, device="cuda")
        c.decode(layer, api.DecodeArgs(entries=3, heads=heads, scale=0.3, q=q.data_ptr(), out=out.data_ptr(), workspace=space.data_ptr(), workspace_bytes=need,
                                       q_row_stride=(heads + 2 * kv) * dim, q_head_stride=dim, out_row_stride=heads * 2 * dim, out_head_stride=2 * dim))
        torch.cuda.synchronize()
        want, away, size = decode_want(pool, fused[:, :heads], range(3), lengths, 0.3)
        check(out[:, :, 0], want, away, size, kind)
        assert out[:, :, 1].isnan().all()


@pytest.mark.gpu
def test_rows_past_32_bits_of_a_long_cache_are_read():
    """Pages of 2^28 elements apart: the last ones lie more than 2^32 bytes behind the first."""
    import torch
    rng = np.random.default_rng(9)
    pages, page, dim, apart = 21, 16, 64, 1 << 28
    flat = torch.zeros((pages - 1) * apart + page * dim, dtype=torch.bfloat16, device="cuda")
    n = pages * page - 5
    pool = Pool(api.BF16, 1, dim, page, pages, 1, pages)
    pool.fill([n], rng)
    for p in range(pages):
        flat[p * apart:p * apart + page * dim] = pool.k[0, p, 0].reshape(-1)
    pool.cache.k = pool.cache.v = flat.data_ptr()         # keys that are their own values
    pool.cache.page_stride = apart
    pool.host_v = pool.host_k
    q = rounded(rng.standard_normal((1, 4, dim)), api.BF16)
    want, away, size = decode_want(pool, q, [0], [n], 0.125)
    check(decode(pool, to_device(q, api.BF16), 4), want, away, size, api.BF16)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES, ids=ids)
def test_a_nan_key_makes_its_own_rows_nan_and_no_other(kind):
    rng = np.random.default_rng(10)
    lengths = [40, 40]
    pool = Pool(kind, 2, 64, 16, 8, 2, 4)
    pool.fill(lengths, rng)
    page = int(pool.host_table[0, 1])
    pool.k[0, page, 1, 3] = math.nan
    q = rounded(rng.standard_normal((2, 4, 64)), kind)
    got = decode(pool, to_device(q, kind), 4)
    want, away, size = decode_want(pool, q, [0, 1], lengths, 0.125)
    assert got[0, 2:].isnan().all()
    check(got[0, :2], want[0, :2], away[0, :2], size[0, :2], kind)
    check(got[1], want[1], away[1], size[1], kind)


# ---- whole prompts -----------------------------------------------------------------------------------------------------------

def prompt(q, k, v, q_starts, kv_starts, kind, masked, scale, out=None, stream=0, **strides):
    import torch
    out = torch.full_like(q, math.nan) if out is None else out
    qs, ks = ints(q_starts), ints(kv_starts)
    args = api.PromptArgs(type=kind, heads=q.shape[1], kv_heads=k.shape[1], head_dim=q.shape[2], masked=int(masked), scale=scale, sequences=len(q_starts) - 1,
                          q_rows=q.shape[0], kv_rows=k.shape[0], q_starts=qs.data_ptr(), kv_starts=ks.data_ptr(), q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(), **strides)
    api.attention_prompt(args, stream)
    torch.cuda.synchronize()
    return out


def seen_by(n, m, masked):
    return np.arange(m)[None] <= np.arange(n)[:, None] + (m - n) if masked else np.ones((n, m), bool)


PROMPTS = [  # heads, kv_heads, dim, lengths of queries, lengths of keys
    (1, 1, 8, [1], [1]), (12, 12, 64, [37], [37]), (4, 2, 64, [1, 64, 65, 0, 128, 200], [1, 64, 65, 0, 128, 200]), (8, 2, 128, [130, 3, 257], [130, 3, 257]),
    (7, 1, 80, [100, 1], [300, 129]), (4, 4, 96, [5, 70, 3], [0, 20, 64]), (2, 1, 256, [90, 33], [90, 33]), (3, 3, 32, [511], [511]), (6, 2, 128, [129, 1, 1], [1000, 127, 128]),
    (2, 2, 64, [300], [1100]), (24, 2, 64, [70, 9], [75, 200]), (128, 1, 64, [3, 1], [200, 5]), (130, 1, 64, [2], [70]), (48, 1, 128, [4, 130], [4, 130])]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES, ids=ids)
@pytest.mark.parametrize("masked", [True, False], ids=["masked", "full"])
@pytest.mark.parametrize("heads,kv_heads,dim,q_len,kv_len", PROMPTS)
def test_prompts_of_different_lengths(heads, kv_heads, dim, q_len, kv_len, masked, kind):
    """Rows of no sequence stand before, between and behind: NaN in them reaches no result, and theirs stay as they were."""
    rng = np.random.default_rng(dim + len(q_len))
    lead = 3
    q_starts, kv_starts = lead + np.concatenate([[0], np.cumsum(q_len)]), 2 + np.concatenate([[0], np.cumsum(kv_len)])
    q, k, v = (np.full((n, h, dim), np.nan) for n, h in ((q_starts[-1] + 5, heads), (kv_starts[-1] + 140, kv_heads), (kv_starts[-1] + 140, kv_heads)))
    q[lead:q_starts[-1]] = rng.standard_normal((sum(q_len), heads, dim)) * 1.5
    for a in (k, v):
        a[2:kv_starts[-1]] = rng.standard_normal((sum(kv_len), kv_heads, dim))
    q, k, v = (rounded(a, kind) for a in (q, k, v))
    scale = dim ** -0.5
    got = prompt(*(to_device(a, kind) for a in (q, k, v)), q_starts, kv_starts, kind, masked, scale)
    for s in range(len(q_len)):
        a, b, x, y = q_starts[s], q_starts[s + 1], kv_starts[s], kv_starts[s + 1]
        want, away, size = attend(q[a:b], k[x:y], v[x:y], scale, seen_by(b - a, y - x, masked))
        check(got[a:b], want, away, size, kind)
    assert got[:lead].isnan().all() and got[q_starts[-1]:].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES, ids=ids)
@pytest.mark.parametrize("dim", [64, 128])
def test_a_neighbours_nan_does_not_reach_a_sequence(kind, dim):
    """Sequences end inside a tile of keys, and the next one's keys and values behind them are NaN and infinities."""
    rng = np.random.default_rng(11)
    lengths = [70, 30, 150, 1]
    starts = np.concatenate([[0], np.cumsum(lengths)])
    q, k, v = (rounded(rng.standard_normal((sum(lengths), 2, dim)), kind) for _ in range(3))
    k[70:100], v[70:100], v[250:] = np.inf, np.nan, -np.inf
    got = prompt(*(to_device(a, kind) for a in (q, k, v)), starts, starts, kind, True, 0.2)
    for a, b in ((0, 70), (100, 250)):
        want, away, size = attend(q[a:b], k[a:b], v[a:b], 0.2, seen_by(b - a, b - a, True))
        check(got[a:b], want, away, size, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES, ids=ids)
@pytest.mark.parametrize("dim", [64, 128])
def test_many_more_pieces_of_work_than_multiprocessors(kind, dim):
    """Each takes several, most of them short and all with keys that end inside a tile; every third sequence's values are NaN, behind the others' last ones too."""
    rng = np.random.default_rng(dim)
    lengths = rng.integers(65, 260, 90)
    starts = np.concatenate([[0], np.cumsum(lengths)])
    q, k, v = (rounded(rng.standard_normal((starts[-1], h, dim)), kind) for h in (12, 6, 6))
    for s in range(2, 90, 3):
        v[starts[s]:starts[s + 1]] = np.nan
    got = prompt(*(to_device(a, kind) for a in (q, k, v)), starts, starts, kind, True, 0.2)
    for s in range(90):
        a, b = starts[s], starts[s + 1]
        if s % 3 == 2:
            assert got[a:b].isnan().all()
        else:
            want, away, size = attend(q[a:b], k[a:b], v[a:b], 0.2, seen_by(b - a, b - a, True))
            check(got[a:b], want, away, size, kind)


FEW_ROWS = [  # heads, kv_heads, dim, lengths of queries, lengths of keys: CTAs of a cluster share a block's keys, two to eight of them
    (2, 1, 8, [1], [4000]), (4, 4, 64, [1, 5], [1500, 900]), (3, 3, 96, [70, 3, 0], [20, 4000, 7]), (6, 2, 128, [100], [100 + 513]), (2, 2, 256, [65, 1], [70, 1200]), (2, 2, 128, [200], [300]),
    (1, 1, 256, [1], [257]), (8, 2, 80, [1, 1, 1], [0, 2049, 128]), (2, 2, 32, [1000], [1000]), (2, 1, 64, [300], [700])]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES, ids=ids)
@pytest.mark.parametrize("masked", [True, False], ids=["masked", "full"])
@pytest.mark.parametrize("heads,kv_heads,dim,q_len,kv_len", FEW_ROWS)
def test_few_rows_over_many_keys(heads, kv_heads, dim, q_len, kv_len, masked, kind):
    """Keys and values of nobody, NaN, stand between the sequences; out's rows of nobody stay."""
    rng = np.random.default_rng(dim + sum(kv_len))
    q_starts, kv_starts = np.concatenate([[0], np.cumsum(q_len)]), np.concatenate([[0], np.cumsum(kv_len)]) + 3
    q = rounded(rng.standard_normal((q_starts[-1] + 2, heads, dim)) * 1.5, kind)
    k, v = (rounded(rng.standard_normal((kv_starts[-1] + 9, kv_heads, dim)), kind) for _ in range(2))
    for a in (k, v):
        a[:3] = a[kv_starts[-1]:] = np.nan
    got = prompt(*(to_device(a, kind) for a in (q, k, v)), q_starts, kv_starts, kind, masked, dim ** -0.5)
    for s in range(len(q_len)):
        a, b, x, y = q_starts[s], q_starts[s + 1], kv_starts[s], kv_starts[s + 1]
        want, away, size = attend(q[a:b], k[x:y], v[x:y], dim ** -0.5, seen_by(b - a, y - x, masked))
        check(got[a:b], want, away, size, kind)
    assert got[q_starts[-1]:].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES, ids=ids)
@pytest.mark.parametrize("dim", [64, 256])
def test_few_rows_with_a_nan_an_infinity_and_nothing_to_see(kind, dim):
    """A NaN key makes its rows NaN whichever CTA has it; scores of -inf everywhere and rows before the first key give what one CTA gives: NaN and zeros."""
    rng = np.random.default_rng(4)
    q, k, v = (rounded(rng.standard_normal((n, 2, dim)), kind) for n in (12, 2000, 2000))
    k[1500, 1, 3] = np.nan
    got = prompt(*(to_device(a, kind) for a in (q, k, v)), [0, 12], [0, 2000], kind, False, 0.1)
    assert got[:, 1].isnan().all()
    want, away, size = attend(q[:, :1], k[:, :1], v[:, :1], 0.1, seen_by(12, 2000, False))
    check(got[:, :1], want, away, size, kind)
    # two sequences: one without keys, one whose first queries see none
    got = prompt(*(to_device(a, kind) for a in (q, k[:1024], v[:1024])), [0, 5, 12], [0, 0, 4], kind, True, 0.1)
    assert (got[:8] == 0).all() and got[8:, 0].isfinite().all() and (got[8:, 0] != 0).any()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES, ids=ids)
@pytest.mark.parametrize("masked", [True, False], ids=["masked", "full"])
@pytest.mark.parametrize("kv_heads,dim", [(4, 64), (16, 64), (4, 128), (16, 80)])
def test_long_prompts_of_many_heads(kv_heads, dim, masked, kind):
    rng = np.random.default_rng(kv_heads + dim)
    starts = np.array([0, 700, 1001])
    q, k, v = (rounded(rng.standard_normal((1001, h, dim)), kind) for h in (16, kv_heads, kv_heads))
    got = prompt(*(to_device(a, kind) for a in (q, k, v)), starts, starts, kind, masked, dim ** -0.5)
    for s in range(2):
        a, b = starts[s], starts[s + 1]
        want, away, size = attend(q[a:b], k[a:b], v[a:b], dim ** -0.5, seen_by(b - a, b - a, masked))
        check(got[a:b], want, away, size, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,keys", [(api.BF16, 3 << 27), (api.FP32, 1 << 27)], ids=["bf16", "fp32"])
def test_a_single_query_over_keys_for_seconds(kind, keys):
    """Longer than one role of a CTA waits for another within a step.  All weight is on the last key."""
    import torch
    k, v = (torch.zeros((keys, 1, 8), dtype=torch_type(kind), device="cuda") for _ in range(2))
    k[-1], v[-1] = 40, 3
    # heads enough that CTAs do not share the keys
    got = prompt(torch.ones((1, 96, 8), dtype=torch_type(kind), device="cuda"), k, v, [0, 1], [0, keys], kind, False, 0.5)
    assert (got == 3).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [api.FP32, api.BF16], ids=ids)
def test_a_prompt_inside_a_fused_projection(kind):
    """Queries, keys and values as columns of one matrix, outputs with a gap between heads."""
    import torch
    rng = np.random.default_rng(12)
    heads, kv, dim, n = 4, 2, 64, 150
    width = (heads + 2 * kv) * dim + 32
    fused = rounded(rng.standard_normal((n, width)), kind)
    x = to_device(fused, kind)
    size_of = x.element_size()
    out = torch.full((n, heads, dim + 16), math.nan, dtype=x.dtype, device="cuda")
    starts = ints([0, 47, n])
    args = api.PromptArgs(type=kind, heads=heads, kv_heads=kv, head_dim=dim, masked=1, scale=0.125, sequences=2, q_rows=n, kv_rows=n, q_starts=starts.data_ptr(), kv_starts=starts.data_ptr(),
                          q=x.data_ptr(), k=x.data_ptr() + heads * dim * size_of, v=x.data_ptr() + (heads + kv) * dim * size_of, out=out.data_ptr(),
                          q_row_stride=width, k_row_stride=width, v_row_stride=width, out_row_stride=heads * (dim + 16), out_head_stride=dim + 16)
    api.attention_prompt(args)
    torch.cuda.synchronize()
    q, k, v = fused[:, :heads * dim].reshape(n, heads, dim), fused[:, heads * dim:(heads + kv) * dim].reshape(n, kv, dim), fused[:, (heads + kv) * dim:(heads + 2 * kv) * dim].reshape(n, kv, dim)
    for a, b in ((0, 47), (47, n)):
        want, away, size = attend(q[a:b], k[a:b], v[a:b], 0.125, seen_by(b - a, b - a, True))
        check(out[a:b, :, :dim], want, away, size, kind)
    assert out[:, :, dim:].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [api.FP32, api.FP16], ids=ids)
def test_starts_that_are_no_starts_read_and_write_nothing_outside(kind):
    rng = np.random.default_rng(13)
    q, k, v = (rounded(rng.standard_normal((90, 2, 64)), kind) for _ in range(3))
    got = prompt(*(to_device(a, kind) for a in (q, k, v)), [-5, 40, 30, 2**31 - 1], [-2**31, 40, 95, 7], kind, True, 0.125)
    # rows 0 ... 39 with keys 0 ... 39; an empty sequence; rows 30 ... 89 with no key at all: what lies in both may be either's
    want, away, size = attend(q[:30], k[:40], v[:40], 0.125, seen_by(40, 40, True)[:30])
    check(got[:30], want, away, size, kind)
    assert (got[40:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES, ids=ids)
def test_scores_far_apart_and_equal_ones(kind):
    """Weights that underflow, rows of equal scores (every weight counts), and a maximum that comes last."""
    rng = np.random.default_rng(14)
    n, dim = 400, 64
    q, k, v = (rng.standard_normal((n, 1, dim)) for _ in range(3))
    q[:100] *= 30
    q[100:200] = 0
    k[:] = np.where(np.arange(n)[:, None, None] % 97 == 96, 3 * k, k)
    q, k, v = (rounded(a, kind) for a in (q, k, v))
    got = prompt(*(to_device(a, kind) for a in (q, k, v)), [0, n], [0, n], kind, True, 0.125)
    want, away, size = attend(q, k, v, 0.125, seen_by(n, n, True))
    check(got, want, away, size, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES, ids=ids)
@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-30])
def test_any_finite_scale(scale, kind):
    rng = np.random.default_rng(23)
    n = 150
    q, k, v = (rounded(rng.standard_normal((n, 2, 64)), kind) for _ in range(3))
    got = prompt(*(to_device(a, kind) for a in (q, k, v)), [0, n], [0, n], kind, True, scale)
    want, away, size = attend(q, k, v, scale, seen_by(n, n, True))
    check(got, want, away, size, kind)
    pool = Pool(kind, 2, 64, 16, 12, 1, 11)
    pool.fill([n], rng)
    want, away, size = decode_want(pool, q[:1], [0], [n], scale)
    check(decode(pool, to_device(q[:1], kind), 2, scale=scale), want, away, size, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 256])
def test_heads_more_than_32_bits_of_elements_apart(dim):
    """Keys, values and outputs with one head behind the other, 2^29 - 64 elements apart: head 9 lies behind 2^32."""
    import torch
    rng = np.random.default_rng(24)
    n, heads, apart, kind = 100, 10, 2 ** 29 - 64, api.BF16
    q, k = (rounded(rng.standard_normal((n, heads, dim)), kind) for _ in range(2))
    flat = torch.zeros((heads - 1) * apart + n * dim, dtype=torch.bfloat16, device="cuda")
    out = torch.zeros_like(flat)
    for h in range(heads):
        flat[h * apart:h * apart + n * dim] = to_device(k[:, h], kind).reshape(-1)
    dq, starts = to_device(q, kind), ints([0, n])
    api.attention_prompt(api.PromptArgs(type=kind, heads=heads, kv_heads=heads, head_dim=dim, masked=1, scale=0.1, sequences=1, q_rows=n, kv_rows=n, q_starts=starts.data_ptr(),
                                        kv_starts=starts.data_ptr(), q=dq.data_ptr(), k=flat.data_ptr(), v=flat.data_ptr(), out=out.data_ptr(), k_row_stride=dim, k_head_stride=apart,
                                        v_row_stride=dim, v_head_stride=apart, out_row_stride=dim, out_head_stride=apart))
    torch.cuda.synchronize()
    want, away, size = attend(q, k, k, 0.1, seen_by(n, n, True))
    got = torch.stack([out[h * apart:h * apart + n * dim].view(n, dim) for h in range(heads)], 1)
    check(got, want, away, size, kind)
    del flat, out
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dim", [(api.FP32, 64), (api.FP32, 128), (api.BF16, 64), (api.FP16, 128)], ids=str)
def test_a_captured_prompt_follows_the_starts(kind, dim):
    """Captured once on a stream of its own, replayed with other sequences in the same rows."""
    import torch
    rng = np.random.default_rng(25)
    n, heads, kv = 400, 4, 2
    q, k, v = (rounded(rng.standard_normal((n, h, dim)), kind) for h in (heads, kv, kv))
    dq, dk, dv = (to_device(a, kind) for a in (q, k, v))
    out, starts = torch.full_like(dq, math.nan), ints([0] * 6)
    args = api.PromptArgs(type=kind, heads=heads, kv_heads=kv, head_dim=dim, masked=1, scale=0.2, sequences=5, q_rows=n, kv_rows=n, q_starts=starts.data_ptr(), kv_starts=starts.data_ptr(),
                          q=dq.data_ptr(), k=dk.data_ptr(), v=dv.data_ptr(), out=out.data_ptr())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        api.attention_prompt(args, torch.cuda.current_stream().cuda_stream)
    for ends in ([400, 400, 400, 400, 400], [1, 130, 131, 131, 390], [0, 0, 0, 0, 257]):
        out.fill_(math.nan)
        starts.copy_(ints([0] + ends))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip([0] + ends, ends):
            want, away, size = attend(q[a:b], k[a:b], v[a:b], 0.2, seen_by(b - a, b - a, True))
            check(out[a:b], want, away, size, kind)
        assert out[ends[-1]:].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dim", [(api.FP32, 64), (api.BF16, 128)], ids=str)
def test_a_captured_call_of_few_rows_follows_the_starts(kind, dim):
    """Two calls in a row in the graph, the second of which attends to what the first has written; CTAs share the keys of a block."""
    import torch
    rng = np.random.default_rng(31)
    q, k, v = (rounded(rng.standard_normal((n, 2, dim)), kind) for n in (20, 2100, 2100))
    dq, dk, dv = (to_device(a, kind) for a in (q, k, v))
    first, second, q_starts, kv_starts = torch.full_like(dq, math.nan), torch.full_like(dq, math.nan), ints([0, 0, 0]), ints([0, 0, 0])
    def args(q, out):
        return api.PromptArgs(type=kind, heads=2, kv_heads=2, head_dim=dim, masked=1, scale=0.2, sequences=2, q_rows=20, kv_rows=2100, q_starts=q_starts.data_ptr(), kv_starts=kv_starts.data_ptr(),
                              q=q.data_ptr(), k=dk.data_ptr(), v=dv.data_ptr(), out=out.data_ptr())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        api.attention_prompt(args(dq, first), torch.cuda.current_stream().cuda_stream)
        api.attention_prompt(args(first, second), torch.cuda.current_stream().cuda_stream)
    for qs, ks in (([0, 20, 20], [0, 2100, 2100]), ([0, 1, 20], [0, 900, 930]), ([0, 0, 7], [5, 5, 1800])):
        first.fill_(math.nan); second.fill_(math.nan)
        q_starts.copy_(ints(qs)); kv_starts.copy_(ints(ks))
        graph.replay()
        torch.cuda.synchronize()
        between = first.float().cpu().numpy().astype(np.float64)
        for s in range(2):
            a, b, x, y = qs[s], qs[s + 1], ks[s], ks[s + 1]
            for given, got in ((q, first), (between, second)):
                want, away, size = attend(given[a:b], k[x:y], v[x:y], 0.2, seen_by(b - a, y - x, True))
                check(got[a:b], want, away, size, kind)
        assert first[qs[2]:].isnan().all() and second[qs[2]:].isnan().all()


# ---- the pool's books --------------------------------------------------------------------------------------------------------

class Books:
    """What the calls on the pool do, entry by entry."""

    def __init__(self, pool):
        self.page = pool.shape[3]
        self.table, self.lengths, self.refs, self.status = pool.books()

    def free_pages(self):
        return list(np.nonzero(self.refs == 0)[0])

    def extend(self, slots, counts):
        need, seen, why = 0, set(), 0
        for s, n in zip(slots, counts):
            if not 0 <= s < len(self.lengths) or n < 0 or s in seen:
                why |= api.CACHE_BAD_INDEX
                continue
            seen.add(s)
            then = self.lengths[s] + n
            if then > self.table.shape[1] * self.page:
                why |= api.CACHE_TOO_LONG
            else:
                need += -(-then // self.page) - -(-self.lengths[s] // self.page)
        free = self.free_pages()
        if not why and need > len(free):
            why = api.CACHE_NO_PAGES
        self.status |= why | (api.CACHE_REFUSED if why else 0)
        if why:
            return
        for s, n in zip(slots, counts):
            for i in range(-(-self.lengths[s] // self.page), -(-(self.lengths[s] + n) // self.page)):
                self.table[s, i] = p = free.pop(0)
                self.refs[p] = 1
            self.lengths[s] += n

    def fork(self, sources, to):
        """Returns (source page, new page, tokens) of what is copied."""
        why, copies, free, before = 0, [], self.free_pages(), self.lengths.copy()
        ok = lambda s: 0 <= s < len(self.lengths)
        if any(not ok(a) or not ok(b) or before[b] != 0 for a, b in zip(sources, to)) or len(set(to)) < len(to):
            why = api.CACHE_BAD_INDEX
        elif sum(before[a] % self.page != 0 for a in sources) > len(free):
            why = api.CACHE_NO_PAGES
        self.status |= why
        if why:
            return copies
        for a, b in zip(sources, to):
            full, rest = divmod(before[a], self.page)
            self.table[b] = -1
            self.table[b, :full] = self.table[a, :full]
            for p in self.table[a, :full]:
                self.refs[p] += 1
            if rest:
                self.table[b, full] = p = free.pop(0)
                self.refs[p] = 1
                copies.append((self.table[a, full], p, rest))
            self.lengths[b] = before[a]
        return copies

    def free(self, slots):
        for s in slots:
            if not 0 <= s < len(self.lengths):
                self.status |= api.CACHE_BAD_INDEX
                continue
            for i in range(-(-self.lengths[s] // self.page)):
                self.refs[self.table[s, i]] -= 1
                self.table[s, i] = -1
            self.lengths[s] = 0

    def compact(self):
        live = (self.refs > 0).sum()
        moves = list(zip([p for p in range(len(self.refs)) if p >= live and self.refs[p] > 0], [p for p in range(live) if self.refs[p] == 0]))
        where = dict(moves)
        for a, b in moves:
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = np.vectorize(lambda p: where.get(p, p), otypes=[np.int32])(self.table)
        return moves

    def same(self, pool):
        import torch
        torch.cuda.synchronize()
        for name, mine, theirs in zip(("page_table", "lengths", "refs", "status"), (self.table, self.lengths, self.refs, self.status), pool.books()):
            np.testing.assert_array_equal(theirs, mine, err_msg=name)


def bits(t):
    import torch
    return t.view(torch.int32 if t.element_size() == 4 else torch.int16).cpu().numpy().copy()


@pytest.mark.gpu
@pytest.mark.parametrize("page,pages,sequences", [(1, 300, 5), (16, 40, 6), (7, 9000, 1200), (256, 3, 2)])
def test_extend_takes_the_lowest_pages_in_order_or_changes_nothing(page, pages, sequences):
    rng = np.random.default_rng(page)
    pool = Pool(api.FP16, 1, 8, page, pages, sequences, 20)
    books = Books(pool)
    for turn in range(12):
        slots = rng.permutation(sequences)[:rng.integers(1, sequences + 1)]
        counts = rng.integers(0, 2 * page + 2, len(slots))
        if turn in (4, 7):
            slots[0] = slots[-1] if turn == 4 and len(slots) > 1 else sequences
        starts = ints(np.concatenate([[turn], turn + np.cumsum(counts)]))
        dev = ints(slots)
        pool.cache.extend(dev.data_ptr(), starts.data_ptr(), len(slots), *pool.space(len(slots)))
        books.extend(slots, counts)
        books.same(pool)
        gone = rng.permutation(sequences)[:max(1, sequences // 3)]
        if turn % 3 == 2:
            dev = ints(gone)
            pool.cache.free(dev.data_ptr(), len(gone))
            books.free(gone)
            books.same(pool)
    # one token for each sequence, without lists; and a sequence that gets too long
    pool.cache.extend(0, 0, sequences, *pool.space(sequences))
    books.extend(range(sequences), [1] * sequences)
    books.same(pool)
    many, slot = ints([0, 20 * page + 1]), ints([1])
    pool.cache.extend(slot.data_ptr(), many.data_ptr(), 1, *pool.space(1))
    books.extend([1], [20 * page + 1])
    books.same(pool)
    assert books.status[0] & api.CACHE_TOO_LONG


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES, ids=ids)
@pytest.mark.parametrize("kv_heads,dim,page,counts,order", [(2, 64, 16, [5, 0, 40, 16], [3, 0, 2, 1]), (1, 8, 1, [1, 2], [0, 1]), (3, 80, 7, [100], [4]), (8, 128, 64, [1, 1, 1, 1, 1], [0, 1, 2, 3, 4]),
                                                            (1, 24, 5, [3] * 100, list(range(100)))])
def test_append_writes_each_token_where_its_sequence_goes_on(kv_heads, dim, page, counts, order, kind):
    import torch
    rng = np.random.default_rng(15)
    sequences = max(order) + 2
    pool = Pool(kind, kv_heads, dim, page, sequences * 45, sequences, 45, layers=2)      # three times 100 tokens are 43 pages of seven
    slots = ints(order)
    where = {s: [] for s in order}
    for turn in range(3):
        starts = np.concatenate([[0], np.cumsum(counts)])
        dev = ints(starts)
        pool.cache.extend(slots.data_ptr(), dev.data_ptr(), len(order), *pool.space(len(order)))
        for layer in range(2):
            k, v = (torch.randn(sum(counts), kv_heads, dim, device="cuda").to(torch_type(kind)) for _ in range(2))
            pool.cache.append(layer, api.AppendArgs(k=k.data_ptr(), v=v.data_ptr(), slots=slots.data_ptr(), starts=dev.data_ptr(), entries=len(order), rows=sum(counts)))
            torch.cuda.synchronize()
            for s, a, b in zip(order, starts, starts[1:]):
                where[s] += [(layer, k[r].clone(), v[r].clone()) for r in range(a, b)]
    assert pool.status.item() == 0
    table = pool.table.cpu().numpy()
    used = torch.zeros(pool.shape, dtype=torch.bool)
    for s, rows in where.items():
        for layer in range(2):
            for t, (_, k, v) in enumerate(r for r in rows if r[0] == layer):
                p, r = table[s, t // page], t % page
                assert pool.k[layer, p, :, r].equal(k) and pool.v[layer, p, :, r].equal(v)
                used[layer, p, :, r] = True
    assert pool.k[~used].isnan().all() and pool.v[~used].isnan().all()


@pytest.mark.gpu
def test_append_leaves_out_rows_that_have_no_place():
    import torch
    pool = Pool(api.FP16, 1, 8, 4, 6, 3, 2)
    pool.table.copy_(ints([[0, 1], [6, -1], [2, 3]]))
    pool.lengths.copy_(ints([2, 8, 100]))
    before = bits(pool.k)
    k = torch.ones(9, 1, 8, dtype=torch.float16, device="cuda")
    # three rows for a sequence of two tokens; a page that is none; a sequence that is none; a length behind the table's end; rows behind the last start
    slots, starts = ints([0, 1, 9, 2]), ints([1, 4, 6, 7, 8])
    pool.cache.append(0, api.AppendArgs(k=k.data_ptr(), v=k.data_ptr(), slots=slots.data_ptr(), starts=starts.data_ptr(), entries=4, rows=9))
    torch.cuda.synchronize()
    got, want = bits(pool.k), before
    one = bits(torch.ones(8, dtype=torch.float16))
    want[0, 0, 0, 0], want[0, 0, 0, 1], want[0, 3, 0, 3] = one, one, one
    np.testing.assert_array_equal(got, want)
    assert pool.status.item() == api.CACHE_BAD_INDEX


@pytest.mark.gpu
def test_append_behind_a_refused_extend_writes_nothing():
    """The last places of the sequence are old tokens' then."""
    import torch
    pool = Pool(api.BF16, 1, 16, 4, 2, 2, 3)
    pool.fill([7], np.random.default_rng(22))
    before, starts, slots = bits(pool.k), ints([0, 2]), ints([0])
    k = torch.ones(2, 1, 16, dtype=torch.bfloat16, device="cuda")
    rows = api.AppendArgs(k=k.data_ptr(), v=k.data_ptr(), slots=slots.data_ptr(), starts=starts.data_ptr(), entries=1, rows=2)
    pool.cache.extend(slots.data_ptr(), starts.data_ptr(), 1, *pool.space(1))
    pool.cache.append(0, rows)
    torch.cuda.synchronize()
    assert pool.status.item() == api.CACHE_NO_PAGES | api.CACHE_REFUSED and pool.lengths[0].item() == 7
    np.testing.assert_array_equal(bits(pool.k), before)
    pool.status.zero_()
    one = ints([0, 1])
    pool.cache.extend(slots.data_ptr(), one.data_ptr(), 1, *pool.space(1))
    pool.cache.append(0, api.AppendArgs(k=k.data_ptr(), v=k.data_ptr(), slots=slots.data_ptr(), starts=one.data_ptr(), entries=1, rows=1))
    torch.cuda.synchronize()
    page = pool.table[0, 1].item()
    assert pool.status.item() == 0 and (pool.k[0, page, 0, 3] == 1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES, ids=ids)
@pytest.mark.parametrize("kv_heads,dim,page,layers,lengths", [(2, 64, 16, 3, [40, 16, 0, 5]), (1, 8, 1, 1, [3, 1]), (3, 80, 7, 2, [20, 50]), (4, 128, 64, 2, [63, 200, 64])])
def test_fork_shares_full_pages_and_copies_the_last(kv_heads, dim, page, layers, lengths, kind):
    rng = np.random.default_rng(16)
    n = len(lengths)
    pool = Pool(kind, kv_heads, dim, page, 2 * sum(-(-x // page) for x in lengths) + 3 * n, 5 * n, 60, layers)
    pool.fill(lengths, rng)
    k, v, books = bits(pool.k), bits(pool.v), Books(pool)
    sources, to = list(range(n)) * 3, [int(x) for x in n + rng.permutation(4 * n)[:3 * n]]
    a, b = ints(sources), ints(to)
    pool.cache.fork(a.data_ptr(), b.data_ptr(), len(to), *pool.space(len(to)))
    for x, y, tokens in books.fork(sources, to):
        for c in (k, v):
            c[:, y, :, :tokens] = c[:, x, :, :tokens]
    books.same(pool)
    np.testing.assert_array_equal(bits(pool.k), k)
    np.testing.assert_array_equal(bits(pool.v), v)
    # not onto one that is taken, not twice, not onto one that is none: nothing changes
    for f, t in (([0], [to[0] if lengths[0] else 0]), ([0, 1], [5 * n - 1, 5 * n - 1]), ([0], [5 * n]), ([-1], [5 * n - 1]), ([0, 0], [5 * n - 1, -3])):
        a, b = ints(f), ints(t)
        pool.cache.fork(a.data_ptr(), b.data_ptr(), len(f), *pool.space(len(f)))
        books.fork(f, t)
        books.same(pool)
    # the originals leave: their pages stay with the forks
    a = ints(list(range(n)) + [0, 0])
    pool.cache.free(a.data_ptr(), n + 2)
    books.free(list(range(n)) + [0, 0])
    books.same(pool)
    a = ints(to)
    pool.cache.free(a.data_ptr(), len(to))
    books.free(to)
    books.same(pool)
    assert (books.refs == 0).all()


@pytest.mark.gpu
def test_fork_without_pages_changes_nothing():
    pool = Pool(api.FP16, 1, 8, 4, 3, 4, 3)
    pool.fill([9], np.random.default_rng(17))
    k, books = bits(pool.k), Books(pool)
    a, b = ints([0]), ints([2])
    pool.cache.fork(a.data_ptr(), b.data_ptr(), 1, *pool.space(1))
    books.fork([0], [2])
    books.same(pool)
    assert books.status[0] == api.CACHE_NO_PAGES
    np.testing.assert_array_equal(bits(pool.k), k)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [api.FP32, api.BF16], ids=ids)
@pytest.mark.parametrize("kv_heads,dim,page,layers,pages,sequences", [(2, 64, 16, 2, 50, 6), (1, 8, 1, 1, 9000, 40), (3, 80, 7, 3, 30, 4), (1, 128, 256, 1, 5, 2)])
def test_compact_moves_the_highest_pages_into_the_lowest_holes(kv_heads, dim, page, layers, pages, sequences, kind):
    rng = np.random.default_rng(18)
    most = pages // sequences
    pool = Pool(kind, kv_heads, dim, page, pages, 2 * sequences, most + 1, layers)
    pool.fill([int(rng.integers(1, most * page + 1)) for _ in range(sequences)], rng)
    books = Books(pool)
    a, b = ints([1]), ints([sequences])
    if (books.refs == 0).any():
        pool.cache.fork(a.data_ptr(), b.data_ptr(), 1, *pool.space(1))
        books.fork([1], [sequences])
    gone = [0] + ([2, 3] if sequences > 3 else [])
    a = ints(gone)
    pool.cache.free(a.data_ptr(), len(gone))
    books.free(gone)
    books.same(pool)
    k, v = bits(pool.k), bits(pool.v)
    for turn in range(2):               # the second time there is nothing to move
        pool.cache.compact(*pool.space(0))
        moves = books.compact()
        assert (turn == 1) <= (not moves)
        for x, y in moves:
            k[:, y], v[:, y] = k[:, x], v[:, x]
        books.same(pool)
        np.testing.assert_array_equal(bits(pool.k), k)
        np.testing.assert_array_equal(bits(pool.v), v)
    assert books.refs[books.refs > 0].size == 0 or np.nonzero(books.refs)[0].max() == (books.refs > 0).sum() - 1


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [api.FP32, api.FP16], ids=ids)
def test_copy_takes_pages_of_all_layers_and_leaves_out_those_that_are_none(kind):
    import torch
    rng = np.random.default_rng(19)
    pool = Pool(kind, 3, 40, 9, 12, 2, 6, layers=4)
    pool.fill([50, 40], rng)
    k, v = bits(pool.k), bits(pool.v)
    a, b = ints([3, 3, 7, -1, 12, 2, 5]), ints([1, 0, 9, 4, 6, 12, -9])
    pool.cache.copy(a.data_ptr(), b.data_ptr(), 7)
    torch.cuda.synchronize()
    for x, y in ((3, 1), (3, 0), (7, 9)):
        k[:, y], v[:, y] = k[:, x], v[:, x]
    np.testing.assert_array_equal(bits(pool.k), k)
    np.testing.assert_array_equal(bits(pool.v), v)
    assert pool.status.item() == api.CACHE_BAD_INDEX


# ---- together ----------------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES, ids=ids)
def test_a_prompt_and_the_tokens_behind_it_through_the_cache(kind):
    """Two prompts, a fork of one, five tokens each, a sequence that leaves, a compaction: every token's row is what attention over all tokens
    before it gives.  The steps are captured once and replayed while the lengths grow."""
    import torch
    rng = np.random.default_rng(20)
    heads, kv, dim, page, scale = 4, 2, 64, 8, 0.125
    pool = Pool(kind, kv, dim, page, 40, 4, 12)
    T = torch_type(kind)
    lens = [21, 40]
    starts = ints([0, 21, 61])
    q, k, v = (rounded(rng.standard_normal((61, h, dim)), kind) for h in (heads, kv, kv))
    dq, dk, dv = (to_device(a, kind) for a in (q, k, v))
    out = torch.full_like(dq, math.nan)
    pool.cache.extend(0, starts.data_ptr(), 2, *pool.space(2))
    pool.cache.append(0, api.AppendArgs(k=dk.data_ptr(), v=dv.data_ptr(), starts=starts.data_ptr(), entries=2, rows=61))
    api.attention_prompt(api.PromptArgs(type=kind, heads=heads, kv_heads=kv, head_dim=dim, masked=1, scale=scale, sequences=2, q_rows=61, kv_rows=61, q_starts=starts.data_ptr(),
                                        kv_starts=starts.data_ptr(), q=dq.data_ptr(), k=dk.data_ptr(), v=dv.data_ptr(), out=out.data_ptr()))
    torch.cuda.synchronize()
    for a, b in ((0, 21), (21, 61)):
        want, away, size = attend(q[a:b], k[a:b], v[a:b], scale, seen_by(b - a, b - a, True))
        check(out[a:b], want, away, size, kind)
    history = {0: (k[:21], v[:21]), 1: (k[21:], v[21:])}
    a, b = ints([0]), ints([3])
    fork_space = torch.empty(pool.cache.workspace(1), dtype=torch.uint8, device="cuda")
    pool.cache.fork(a.data_ptr(), b.data_ptr(), 1, fork_space.data_ptr(), fork_space.numel())
    history[3] = history[0]
    # one step for sequences 3, 0, 1, captured on a stream of its own
    order = [3, 0, 1]
    slots = ints(order)
    tq, tk, tv = (torch.zeros(3, h, dim, dtype=T, device="cuda") for h in (heads, kv, kv))
    step_out = torch.full((3, heads, dim), math.nan, dtype=T, device="cuda")
    need = pool.cache.decode_workspace(3, heads)
    book_space, space = torch.empty(pool.cache.workspace(3), dtype=torch.uint8, device="cuda"), torch.empty(need, dtype=torch.uint8, device="cuda")
    append = api.AppendArgs(k=tk.data_ptr(), v=tv.data_ptr(), slots=slots.data_ptr(), entries=3, rows=3)
    call = api.DecodeArgs(entries=3, heads=heads, scale=scale, q=tq.data_ptr(), out=step_out.data_ptr(), slots=slots.data_ptr(), workspace=space.data_ptr(), workspace_bytes=need)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        stream = torch.cuda.current_stream().cuda_stream
        pool.cache.extend(slots.data_ptr(), 0, 3, book_space.data_ptr(), book_space.numel(), stream)
        pool.cache.append(0, append, stream)
        pool.cache.decode(0, call, stream)

    def step():
        new = [rounded(rng.standard_normal((3, h, dim)), kind) for h in (heads, kv, kv)]
        for d, h in zip((tq, tk, tv), new):
            d.copy_(to_device(h, kind))
        graph.replay()
        torch.cuda.synchronize()
        for i, s in enumerate(order):
            if s in history:
                history[s] = tuple(np.concatenate([h, x[i:i + 1]]) for h, x in zip(history[s], new[1:]))
                want, away, size = attend(new[0][i:i + 1], *history[s], scale, np.ones((1, len(history[s][0])), bool))
                check(step_out[i:i + 1], want, away, size, kind)

    for _ in range(5):
        step()
    gone = ints([0])
    pool.cache.free(gone.data_ptr(), 1)
    del history[0]
    compact_space = torch.empty(pool.cache.workspace(0), dtype=torch.uint8, device="cuda")
    pool.cache.compact(compact_space.data_ptr(), compact_space.numel())
    for _ in range(12):
        step()
    assert pool.status.item() == 0


@pytest.mark.gpu
def test_calls_on_two_streams_do_not_disturb_each_other():
    import torch
    rng = np.random.default_rng(21)
    pools, queries, wants = [], [], []
    for i in range(2):
        lengths = [int(x) for x in rng.integers(1, 3000, 6)]
        pool = Pool(api.BF16, 2, 128, 16, 1300, 6, 200)
        pool.fill(lengths, rng)
        q = rounded(rng.standard_normal((6, 8, 128)), api.BF16)
        pools.append(pool); queries.append(to_device(q, api.BF16)); wants.append(decode_want(pool, q, range(6), lengths, 0.1))
    streams = [torch.cuda.Stream() for _ in range(2)]
    spaces = [torch.empty(p.cache.decode_workspace(6, 8), dtype=torch.uint8, device="cuda") for p in pools]
    outs = [torch.full_like(q, math.nan) for q in queries]
    torch.cuda.synchronize()
    for _ in range(20):
        for p, q, s, w, o in zip(pools, queries, streams, spaces, outs):
            p.cache.decode(0, api.DecodeArgs(entries=6, heads=8, scale=0.1, q=q.data_ptr(), out=o.data_ptr(), workspace=w.data_ptr(), workspace_bytes=w.numel()), s.cuda_stream)
    torch.cuda.synchronize()
    for o, (want, away, size) in zip(outs, wants):
        check(o, want, away, size, api.BF16)


# ---- refusals and what comes behind them -------------------------------------------------------------------------------------

def with_refused(pool):
    pool.refused = ints(np.zeros(pool.lengths.numel()))
    pool.cache.refused = pool.refused.data_ptr()
    return pool


class Sequences:
    """Tokens with keys and values of their own, given to a pool call by call; `kept`: what each sequence has to hold."""

    def __init__(self, pool):
        self.pool, self.kept, self.next = pool, {s: [] for s in range(pool.lengths.numel())}, 1

    def extend(self, slots, counts):
        """The extend alone; returns its append."""
        import torch
        kv_heads, dim = self.pool.shape[2], self.pool.shape[4]
        values = np.arange(self.next, self.next + sum(counts))
        self.next += sum(counts)
        at, starts = ints(slots), ints(np.concatenate([[0], np.cumsum(counts)]))
        rows = torch.from_numpy(values).to(torch_type(self.pool.kind)).cuda()[:, None, None].expand(-1, kv_heads, dim).contiguous()
        self.pool.cache.extend(at.data_ptr(), starts.data_ptr(), len(slots), *self.pool.space(len(slots)))

        def append():
            if len(values):
                for layer in range(self.pool.shape[0]):
                    self.pool.cache.append(layer, api.AppendArgs(k=rows.data_ptr(), v=rows.data_ptr(), slots=at.data_ptr(), starts=starts.data_ptr(), entries=len(slots), rows=len(values)))
            torch.cuda.synchronize()
        append.rows = [list(x) for x in np.split(values, np.cumsum(counts)[:-1])]
        return append

    def give(self, slots, counts, ok):
        append = self.extend(slots, counts)
        append()
        if ok:
            for s, rows in zip(slots, append.rows):
                self.kept[s] += rows

    def check(self):
        table, lengths = self.pool.table.cpu().numpy(), self.pool.lengths.cpu().numpy()
        page = self.pool.shape[3]
        for s, rows in self.kept.items():
            assert lengths[s] == len(rows), s
            for c in (self.pool.k, self.pool.v):
                held = c.float().cpu().numpy()
                for t, x in enumerate(rows):
                    assert (held[:, table[s, t // page], :, t % page] == x).all(), (s, t)


@pytest.mark.gpu
@pytest.mark.parametrize("why", ["pages", "length", "index", "twice"])
def test_a_refused_extend_stops_its_sequences_and_no_others(why):
    bit = dict(pages=api.CACHE_NO_PAGES, length=api.CACHE_TOO_LONG, index=api.CACHE_BAD_INDEX, twice=api.CACHE_BAD_INDEX)[why] | api.CACHE_REFUSED
    pool = with_refused(Pool(api.FP16, 2, 8, 4, 6, 4, 4, layers=2))
    s = Sequences(pool)
    s.give([0, 1, 2], [3, 5, 2], True)
    assert pool.status.item() == 0
    bad = dict(pages=([0, 2], [10, 6]), length=([0, 2], [14, 1]), index=([0, 2, 4], [1, 1, 1]), twice=([0, 2, 0], [1, 1, 1]))[why]
    late = s.extend([1], [1])                      # one that went through before, and is written behind the refusal
    s.kept[1] += late.rows[0]
    refused = s.extend(*bad)
    late()
    # the others go on, whatever the order of the calls; the refused ones' rows are not written
    other = s.extend([1, 3], [1, 2])
    refused()
    other()
    for x, rows in zip([1, 3], other.rows):
        s.kept[x] += rows
    s.check()
    assert pool.status.item() == bit and pool.refused.tolist() == [1, 0, 1, 0]
    # they stay as they are, and so does who is named with them, until the host has seen it
    pool.status.zero_()
    s.give([3, 2], [1, 1], False)
    s.check()
    assert pool.status.item() == api.CACHE_REFUSED and pool.refused.tolist() == [1, 0, 1, 1]
    s.give([1], [1], True)
    s.check()
    pool.refused.zero_()
    s.give([0, 3, 2], [1, 1, 1], True)
    s.check()
    assert pool.refused.tolist() == [0] * 4


@pytest.mark.gpu
def test_a_freed_sequence_is_no_longer_refused():
    pool = with_refused(Pool(api.BF16, 1, 16, 4, 2, 3, 2))
    s = Sequences(pool)
    s.give([0], [5], True)
    s.give([1, 2], [1, 1], False)
    s.give([1], [0], False)
    s.check()
    assert pool.refused.tolist() == [0, 1, 1] and pool.status.item() == api.CACHE_NO_PAGES | api.CACHE_REFUSED
    slots = ints([0, 1, 1])
    pool.cache.free(slots.data_ptr(), 3)
    s.kept[0] = []
    s.give([1, 0], [4, 3], True)
    s.check()
    assert pool.refused.tolist() == [0, 0, 1]


@pytest.mark.gpu
def test_tokens_behind_a_refused_fork_go_nowhere():
    pool = with_refused(Pool(api.FP32, 1, 8, 4, 3, 4, 2))
    s = Sequences(pool)
    s.give([0], [6], True)

    def fork(sources, to):
        a, b = ints(sources), ints(to)
        pool.cache.fork(a.data_ptr(), b.data_ptr(), len(to), *pool.space(len(to)))

    fork([0, 0], [2, 3])                           # one page is free, two are needed
    s.give([2, 3], [1, 1], False)
    s.give([0], [1], True)
    s.check()
    assert pool.status.item() == api.CACHE_NO_PAGES | api.CACHE_REFUSED and pool.refused.tolist() == [0, 0, 1, 1]
    got = decode(pool, to_device(np.ones((4, 1, 8)), api.FP32), 1)
    assert got[0].isfinite().all() and (got[0] != 0).all() and (got[1:] == 0).all()
    # neither onto a refused one nor from one
    pool.status.zero_()
    fork([0], [2])
    pool.refused[2] = 0
    pool.refused[0] = 1
    fork([0], [1])
    s.check()
    assert pool.status.item() == api.CACHE_REFUSED and pool.refused.tolist() == [1, 1, 0, 1]
    pool.refused.zero_()
    fork([0], [2])
    s.kept[2] = list(s.kept[0])
    s.check()
    s.give([2], [1], True)
    s.check()
    assert pool.refused.tolist() == [0] * 4


@pytest.mark.gpu
def test_captured_steps_go_on_behind_a_refusal():
    """Two batches in one pool, a captured step each, replayed without a look at the status: the one that finds no pages stands still, also when there are pages again, until its sequences
    are freed or set to go on."""
    import torch
    pool = with_refused(Pool(api.BF16, 1, 8, 2, 6, 4, 4))
    kept, steps = {s: [] for s in range(4)}, []
    for slots in ([0, 1], [2, 3]):
        at, row = ints(slots), torch.zeros(2, 1, 8, dtype=torch.bfloat16, device="cuda")
        space = torch.empty(pool.cache.workspace(2), dtype=torch.uint8, device="cuda")
        args = api.AppendArgs(k=row.data_ptr(), v=row.data_ptr(), slots=at.data_ptr(), entries=2, rows=2)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            stream = torch.cuda.current_stream().cuda_stream
            pool.cache.extend(at.data_ptr(), 0, 2, space.data_ptr(), space.numel(), stream)
            pool.cache.append(0, args, stream)
        steps.append((slots, row, graph, at, space, args))

    def step(which, x, ok):
        slots, row, graph = steps[which][:3]
        row.copy_(torch.tensor([x, x + 100.0]).to(torch.bfloat16)[:, None, None].expand(2, 1, 8))
        graph.replay()
        torch.cuda.synchronize()
        if ok:
            for s, v in zip(slots, (x, x + 100)):
                kept[s].append(v)
        table, page = pool.table.cpu().numpy(), pool.shape[3]
        for s, rows in kept.items():
            assert pool.lengths[s].item() == len(rows)
            for t, v in enumerate(rows):
                assert (pool.k[0, table[s, t // page], 0, t % page] == v).all() and (pool.v[0, table[s, t // page], 0, t % page] == v).all()

    for x, which, ok in [(1, 0, True), (2, 0, True), (3, 1, True), (4, 0, True), (5, 0, True), (6, 1, True), (7, 1, False), (8, 0, False)]:      # six pages of two tokens
        step(which, x, ok)
    slots = ints([0])
    pool.cache.free(slots.data_ptr(), 1)
    kept[0] = []
    step(1, 9, False)                # two pages are free now
    step(0, 10, False)               # sequence 1 stands still
    pool.refused[2:] = 0
    step(1, 11, True)
    assert pool.refused.tolist() == [1, 1, 0, 0] and pool.status.item() == api.CACHE_NO_PAGES | api.CACHE_REFUSED


@pytest.mark.gpu
def test_a_list_of_refused_sequences_in_host_memory_is_refused():
    import torch
    host, d = torch.zeros(64, dtype=torch.int32), torch.zeros(1 << 20, dtype=torch.uint8, device="cuda").data_ptr()
    L, c = api.lib(), good_cache(refused=host.data_ptr(), **{name: d for name in ("k", "v", "page_table", "lengths", "refs", "status")})
    rows = api.AppendArgs(k=d, v=d, entries=1, rows=1)
    assert L.aspen_b200_cache_extend(C.byref(c), None, None, 1, d, 1 << 20, None) == -1 and "refused" in api.last_error()
    assert L.aspen_b200_cache_append(C.byref(c), 0, C.byref(rows), None) == -1
    assert L.aspen_b200_cache_fork(C.byref(c), d, d, 1, d, 1 << 20, None) == -1
    assert L.aspen_b200_cache_free(C.byref(c), d, 1, None) == -1


# ---- small weights beside a large one ----------------------------------------------------------------------------------------
#
# One key takes nearly all weight and has values of zero, the others share 2^-24 or 2^-20 of it each, so an output is as exact as their weights.
# Off by at most: u |o| its own rounding, u A the weights' (16 bits), 2 delta A the scores', and sums of n terms: products 16 at a time, cut off at 2^-23 of
# the sum, and weights four to a thread and 16 keys at most, rounded to 2^-24: n (2^-27 + 2^-26) < n 2^-25; joins and exp2 2^-20.

def sink_and_tail(keys, kv_heads, dim, apart, kind):
    """k, v of `keys` tokens, the first one `apart` above the others for a query of (1, 0, 0 ...)."""
    rng = np.random.default_rng(int(apart * 1000) + keys)
    k, v = rng.standard_normal((keys, kv_heads, dim)), 64 * (1 + rng.random((keys, kv_heads, dim)))
    k[:, :, 0] = 0
    k[0, :, 0], v[0] = apart, 0
    return rounded(k, kind), rounded(v, kind)


def check_tail(got, q, k, v, kind):
    want, _, size = attend(q, k, v, 1.0, np.ones((len(q), len(k)), bool))
    away = size * (2 * np.abs(k[:, :, 0]).max() * (q.shape[2] * 2.0 ** -23 + 2.0 ** -20) + len(k) * 2.0 ** -25 + 2.0 ** -20)
    check(got, want, away, size, kind)


APART = [pytest.param(14.03125, id="2^-20"), pytest.param(16.875, id="2^-24")]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES, ids=ids)
@pytest.mark.parametrize("apart", APART)
@pytest.mark.parametrize("heads,dim,q_len,kv_len", [(12, 64, [512], [4000]), (12, 128, [512], [4000]), (8, 64, [1], [60000]), (2, 256, [1], [9000]), (8, 256, [1] * 64, [1000] * 64), (24, 32, [3] * 40, [50] * 40)])
def test_prompts_weigh_many_small_keys_beside_a_large_one(heads, dim, q_len, kv_len, apart, kind):
    k, v = sink_and_tail(kv_len[0], heads, dim, apart, kind)
    q = np.zeros((q_len[0], heads, dim))
    q[:, :, 0] = 1
    n = len(q_len)
    got = prompt(*(to_device(np.concatenate([a] * n), kind) for a in (q, k, v)), np.arange(n + 1) * q_len[0], np.arange(n + 1) * kv_len[0], kind, False, 1.0)
    for s in (0, n // 2, n - 1):
        check_tail(got[s * q_len[0]:(s + 1) * q_len[0]], q, k, v, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES, ids=ids)
@pytest.mark.parametrize("apart", APART)
@pytest.mark.parametrize("heads,kv_heads,dim,tokens,entries", [(4, 4, 64, 320, 600), (8, 4, 128, 320, 600), (4, 4, 256, 320, 400), (16, 1, 64, 700, 3), (2, 2, 64, 60000, 1)])
def test_a_token_weighs_many_small_keys_beside_a_large_one(heads, kv_heads, dim, tokens, entries, apart, kind):
    """Many entries: a warp walks a whole sequence; few: it is shared."""
    rng = np.random.default_rng(30)
    pool = Pool(kind, kv_heads, dim, 16, -(-tokens // 16), 1, -(-tokens // 16))
    pool.fill([tokens], rng)
    k, v = sink_and_tail(tokens, kv_heads, dim, apart, kind)
    for t in range(tokens):
        p, r = pool.host_table[0, t // 16], t % 16
        pool.host_k[0, p, :, r], pool.host_v[0, p, :, r] = k[t], v[t]
    pool.k.copy_(to_device(pool.host_k, kind)); pool.v.copy_(to_device(pool.host_v, kind))
    q = np.zeros((1, heads, dim))
    q[:, :, 0] = 1
    got = decode(pool, to_device(np.concatenate([q] * entries), kind), heads, slots=[0] * entries, scale=1.0)
    for i in (0, entries // 2, entries - 1):
        check_tail(got[i:i + 1], q, k, v, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("page,lengths,broken,value", [(4, [9, 6], (0, 0), -1), (4, [9, 6], (0, 1), 13), (4, [8, 6], (0, 1), 2**31 - 1), (1, [3000, 2], (0, 2999), -7), (4, [9, 6], (1, 1), -1), (4, [9, 6], (0, 2), -1)])
def test_fork_of_a_sequence_with_a_page_that_is_none_changes_nothing(page, lengths, broken, value):
    """Its neighbours in the call are not forked either."""
    pool = Pool(api.FP16, 1, 8, page, 8 + sum(-(-n // page) for n in lengths), 6, -(-max(lengths) // page) + 1)
    pool.fill(lengths, np.random.default_rng(31))
    table = pool.host_table.copy()
    table[broken] = value
    pool.table.copy_(ints(table))
    k, books = bits(pool.k), Books(pool)
    a, b = ints([1, 0, 1]), ints([2, 3, 5])
    pool.cache.fork(a.data_ptr(), b.data_ptr(), 3, *pool.space(3))
    books.status |= api.CACHE_BAD_INDEX
    books.same(pool)
    np.testing.assert_array_equal(bits(pool.k), k)
    # the pool goes on: pages taken for nothing are free
    pool.status.zero_(); pool.table.copy_(ints(pool.host_table))
    books = Books(pool)
    pool.cache.fork(a.data_ptr(), b.data_ptr(), 3, *pool.space(3))
    copied = books.fork([1, 0, 1], [2, 3, 5])
    books.same(pool)
    for x, y, tokens in copied:
        k[:, y, :, :tokens] = k[:, x, :, :tokens]
    np.testing.assert_array_equal(bits(pool.k), k)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES, ids=ids)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_status_word_of_prompts_stays_as_it_was_where_nothing_stalls(dim, kind):
    import torch
    rng = np.random.default_rng(40)
    q, k, v = (rounded(rng.standard_normal((300, 8, dim)), kind) for _ in range(3))
    status = ints([6])
    got = prompt(*(to_device(a, kind) for a in (q, k, v)), [0, 300], [0, 300], kind, True, 0.1, status=status.data_ptr())
    want, away, size = attend(q, k, v, 0.1, seen_by(300, 300, True))
    check(got, want, away, size, kind)
    assert status.item() == 6
    d, host = got.data_ptr(), torch.zeros(4, dtype=torch.int32)
    good = dict(type=kind, heads=1, kv_heads=1, head_dim=8, scale=1.0, sequences=1, q_rows=1, kv_rows=1, q_starts=status.data_ptr(), kv_starts=status.data_ptr(), q=d, k=d, v=d, out=d + 4096)
    assert api.lib().aspen_b200_attention_prompt(C.byref(api.PromptArgs(**good, status=host.data_ptr())), None) == -1 and "status" in api.last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES, ids=ids)
@pytest.mark.parametrize("heads,kv_heads,dim,q_len,kv_len", [(2, 2, 64, [300, 40], [50, 200]), (2, 2, 32, [40, 300, 130], [200, 50, 2]), (2, 2, 128, [300, 40], [50, 200]), (16, 2, 64, [60, 5], [20, 40])])
def test_masked_prompts_whose_first_tile_sees_no_key(heads, kv_heads, dim, q_len, kv_len, kind):
    """Its second tile does, in the same piece of work: 48 short sequences beside them, so that the calls run in tiles."""
    rng = np.random.default_rng(dim + heads)
    q_len, kv_len = q_len + [300] * 48, kv_len + [50] * 48
    qs, ks = np.concatenate([[0], np.cumsum(q_len)]), np.concatenate([[0], np.cumsum(kv_len)])
    q, k, v = (rounded(rng.standard_normal((n, h, dim)), kind) for n, h in ((qs[-1], heads), (ks[-1], kv_heads), (ks[-1], kv_heads)))
    got = prompt(*(to_device(a, kind) for a in (q, k, v)), qs, ks, kind, True, dim ** -0.5)
    for s in range(len(q_len)):
        a, b, x, y = qs[s], qs[s + 1], ks[s], ks[s + 1]
        want, away, size = attend(q[a:b], k[x:y], v[x:y], dim ** -0.5, seen_by(b - a, y - x, True))
        check(got[a:b], want, away, size, kind)
        assert (got[a:b][:max(0, (b - a) - (y - x))] == 0).all()


# ---- more refusals -----------------------------------------------------------------------------------------------------------

def test_words_off_a_4_byte_boundary_are_refused():
    L, good = api.lib(), good_cache()
    for name in ("page_table", "lengths", "refs", "status", "refused"):
        c = good_cache(**{name: 66})
        call, rows = api.DecodeArgs(entries=1, heads=2, scale=1.0, q=4096, out=4096, workspace=4096, workspace_bytes=1 << 30), api.AppendArgs(k=4096, v=4096, entries=1, rows=1)
        assert L.aspen_b200_attention_decode(C.byref(c), 0, C.byref(call), None) == -1 and name in api.last_error()
        assert L.aspen_b200_cache_append(C.byref(c), 0, C.byref(rows), None) == -1
        assert L.aspen_b200_cache_extend(C.byref(c), None, None, 1, 4096, 1 << 30, None) == -1
        assert L.aspen_b200_cache_fork(C.byref(c), 64, 64, 1, 4096, 1 << 30, None) == -1
        assert L.aspen_b200_cache_free(C.byref(c), 64, 1, None) == -1
        assert L.aspen_b200_cache_compact(C.byref(c), 4096, 1 << 30, None) == -1
        assert L.aspen_b200_cache_copy(C.byref(c), 64, 64, 1, None) == -1
    c = C.byref(good)
    for at in (65, 66, 67):
        assert L.aspen_b200_cache_extend(c, at, None, 1, 4096, 1 << 30, None) == L.aspen_b200_cache_extend(c, None, at, 1, 4096, 1 << 30, None) == -1
        assert L.aspen_b200_cache_fork(c, at, 64, 1, 4096, 1 << 30, None) == L.aspen_b200_cache_fork(c, 64, at, 1, 4096, 1 << 30, None) == -1
        assert L.aspen_b200_cache_copy(c, at, 64, 1, None) == L.aspen_b200_cache_copy(c, 64, at, 1, None) == -1
        assert L.aspen_b200_cache_free(c, at, 1, None) == -1
        for name in ("slots", "starts"):
            assert L.aspen_b200_cache_append(c, 0, C.byref(api.AppendArgs(k=4096, v=4096, entries=1, rows=1, **{name: at})), None) == -1 and name in api.last_error()
        assert L.aspen_b200_attention_decode(c, 0, C.byref(api.DecodeArgs(entries=1, heads=2, scale=1.0, q=4096, out=4096, slots=at, workspace=4096, workspace_bytes=1 << 30)), None) == -1
        for name in ("q_starts", "kv_starts", "status"):
            args = dict(type=api.FP16, heads=4, kv_heads=2, head_dim=64, scale=1.0, sequences=1, q_rows=3, kv_rows=3, q_starts=64, kv_starts=64, q=4096, k=4096, v=4096, out=8192)
            args[name] = at
            assert L.aspen_b200_attention_prompt(C.byref(api.PromptArgs(**args)), None) == -1 and name in api.last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES, ids=ids)
@pytest.mark.parametrize("heads,kv_heads,dim,scale", [(12, 6, 64, 0.2), (4, 4, 128, -0.1), (6, 2, 256, 0.1), (3, 3, 40, 0.2)])
def test_hundreds_of_short_prompts(heads, kv_heads, dim, scale, kind):
    """A CTA takes several blocks of queries, of one sequence and of the next ones.  Among 700 sequences of up to five tokens are empty ones, one of 200, and a first one that would end
    before it starts."""
    rng = np.random.default_rng(heads)
    lengths = rng.integers(0, 6, 700)
    lengths[350] = 200
    starts = np.concatenate([[0], np.cumsum(lengths)]) + 2
    q, k, v = (rounded(rng.standard_normal((starts[-1] + 3, h, dim)), kind) for h in (heads, kv_heads, kv_heads))
    starts[0] = 9
    got = prompt(*(to_device(a, kind) for a in (q, k, v)), starts, starts, kind, True, scale)
    for s in range(1, 700):
        a, b = starts[s], starts[s + 1]
        want, away, size = attend(q[a:b], k[a:b], v[a:b], scale, seen_by(b - a, b - a, True))
        check(got[a:b], want, away, size, kind)
    assert got[:starts[1]].isnan().all() and got[starts[-1]:].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,dim,n", [(12, 64, 512), (2, 64, 40), (12, 128, 200)])
def test_fp32_values_of_any_size(heads, dim, n):
    """An operand is off by 2^-22 of itself, which the usual tolerance has, or by 2^-126; so is a mean of values, and it may lose 2^-126 when it is written.  2^128 - 2^120 is a value, too."""
    rng = np.random.default_rng(50)
    q, k, base = (rounded(rng.standard_normal((n, heads, dim)), api.FP32) for _ in range(3))
    q[0] = 0
    for power in (-126, -116, -108, -100, 100, 127):
        v = rounded(base * 2.0 ** min(power, 100), api.FP32)
        if power == 127:
            v[0, :, ::3] = 2.0 ** 128 - 2.0 ** 120
        got = prompt(*(to_device(a, api.FP32) for a in (q, k, v)), [0, n], [0, n], api.FP32, True, 0.1).cpu().numpy().astype(np.float64)
        want, away, _ = attend(q, k, v, 0.1, seen_by(n, n, True))
        assert (np.abs(got - want) <= away + 2.0 ** -24 * np.abs(want) + 2.0 ** -125).all(), power
        pool = Pool(api.FP32, heads, dim, 16, n // 16 + 1, 1, n // 16 + 1)
        pool.fill([n], rng)
        pool.host_v = rounded(np.nan_to_num(pool.host_v) * 2.0 ** min(power, 100), api.FP32)
        if power == 127:
            pool.host_v[0, pool.host_table[0, 0], :, 0, ::3] = 2.0 ** 128 - 2.0 ** 120
        pool.v.copy_(to_device(pool.host_v, api.FP32))
        got = decode(pool, to_device(q[1:2], api.FP32), heads, slots=[0]).cpu().numpy().astype(np.float64)
        want, away, _ = decode_want(pool, q[1:2], [0], [n], dim ** -0.5)
        assert (np.abs(got - want) <= away + 2.0 ** -24 * np.abs(want) + 2.0 ** -125).all(), power
