"""A paged cache of keys and values, and what a layer does with it between its qkv projection and its o_proj: new tokens
enter it rotated (`PagedKV.append`), and attend over it (`PagedKV.attend`).

The reference keeps one arena per request and runs these as Triton kernels: QK-norm + RoPE + KV write
(dlmrt/ops/triton/core.py, dlmrt/models/sdar/model.py:211-243) and flash attention split over the keys with a combine pass
(dlmrt/ops/triton/attention.py, dlmrt/models/sdar/engine.py:127-132). Here the cache is a pool of fixed-size pages that
sequences share, each sequence listing its pages; a block of a denoise round and a single decoded token are the same call.

    cache = PagedKV(keys, values)                      # one layer's pool: [pages, kv heads, page size, head dim] each
    table = rotary_table(head_dim, 32768, theta=1e6, device=device)
    q = cache.append(k, v, positions, slots, table, q=q, q_norm=w_q, k_norm=w_k)
    a = cache.attend(q.view(batch, tokens, heads, head_dim), pages, lengths)
    group.reduce_norm(o_proj(a.view(rows, -1), out=group.partial(...)), ...)

Everything runs on the current stream of the cache's device, can be captured, and allocates only its results and scratch
from torch's allocator. Indices (slots, positions, pages, lengths) live on the device and are checked there: one that lies
outside its table touches no memory, and `PagedKV.check()` raises IndexError for the first of them.
"""

from contextlib import nullcontext
from struct import Struct

import torch

from .. import _lib
from .._lib import DlmAppend, DlmAttend, DlmPages

# The pointers that every call brings, which lie side by side in the descriptors.
_APPEND, _APPEND_AT = Struct("9Q"), DlmAppend.q.offset
_ATTEND, _ATTEND_AT = Struct("7Q"), DlmAttend.q.offset
_MOST_INT = (1 << 31) - 1  # what a larger page is reported as
_MOST_PLANS = 4096  # of one cache: sizes of calls that are remembered

_INDEX = {1: "slot", 2: "position", 3: "page", 4: "length", 5: "adapter"}


def rotary_table(rotated, positions, theta=10000.0, device="cuda", inverse_frequencies=None):
    """[positions, rotated] FP32 for `PagedKV.append`: the cosines of position * theta^(-2 i / rotated) for i < rotated / 2,
    then the sines. The angles are formed in 64 bits: in 32 bits an angle of 10^5 is off by 2^-8. `inverse_frequencies`
    [rotated / 2] replaces the powers of theta (stretched or scaled rotations)."""
    half = rotated // 2
    if inverse_frequencies is None:
        inverse_frequencies = theta ** (-torch.arange(half, device=device, dtype=torch.float64) / half)
    if inverse_frequencies.shape != (half,):
        raise ValueError(f"expected {half} inverse frequencies, got {tuple(inverse_frequencies.shape)}")
    angle = torch.arange(positions, device=device, dtype=torch.float64).view(-1, 1) * inverse_frequencies.to(device).double()
    return torch.cat((angle.cos(), angle.sin()), 1).float()


def _index_error(status, where, page_size=0):
    """Reads `status` (and clears it); IndexError where a kernel met an index outside its table."""
    read = _lib.read_status(status, where)
    if read.code == _lib.ERR_INDEX:
        kind, value = _INDEX.get(read.slot, "index"), str(read.epoch)
        if kind == "slot":  # as a page and the place in it, which is how a slot is made up
            value = f"{'at least ' if read.epoch == _MOST_INT else ''}{read.epoch} * {page_size} + {read.phase}"
        raise IndexError(f"{where}: row {read.block}: {kind} {value} lies outside its table")
    _lib.check(read.code, where)


class PagedKV:
    """One layer's pool of pages.

    `keys`, `values`: [pages, kv heads, page size, head dim], BF16 or FP16 (the type of the queries, too) or FP8 E4M3 with
    `k_scale`, `v_scale` [kv heads] FP32: a code counts for code * scale of its head. The head dimension (64, 128 or 256) is
    contiguous, the other strides are free (multiples of 16 bytes), the page size is a power of two from 8 to
    4096."""

    def __init__(self, keys, values, k_scale=None, v_scale=None):
        if keys.dim() != 4 or keys.shape != values.shape or keys.dtype != values.dtype or keys.device != values.device:
            raise ValueError(f"keys {tuple(keys.shape)} {keys.dtype} and values {tuple(values.shape)} {values.dtype} must be "
                             "[pages, kv heads, page size, head dim] alike")
        if keys.dtype not in _lib.TYPES:
            raise ValueError(f"a cache holds BF16, FP16 or FP8 E4M3, not {keys.dtype}")
        if keys.stride(3) != 1 or values.stride(3) != 1:
            raise ValueError("keys and values must have a contiguous head dimension")
        pages, heads, page_size, head_dim = keys.shape
        if head_dim not in (64, 128, 256) or page_size & (page_size - 1) or not _lib.MIN_PAGE <= page_size <= _lib.MAX_PAGE:
            raise ValueError(f"head dimension {head_dim}, page size {page_size}: expected 64, 128 or 256, and a power of two "
                             f"from {_lib.MIN_PAGE} to {_lib.MAX_PAGE}")
        coded = keys.dtype == torch.float8_e4m3fn
        for scale in (k_scale, v_scale):
            if coded != (scale is not None):
                raise ValueError("an FP8 cache, and no other, has a scale per kv head for keys and for values")
            if scale is not None and (scale.dtype != torch.float32 or scale.shape != (heads,) or not scale.is_contiguous()
                                      or scale.device != keys.device):
                raise ValueError(f"scales must be contiguous FP32 [{heads}] tensors on {keys.device}")
        self.keys, self.values, self.k_scale, self.v_scale = keys, values, k_scale, v_scale
        self.device, self.dtype, self.heads, self.page_size, self.head_dim = keys.device, keys.dtype, heads, page_size, head_dim
        self.status = torch.zeros(_lib.STATUS_WORDS, device=keys.device, dtype=torch.int32)
        p = DlmPages()
        p.keys, p.values, p.status = keys.data_ptr(), values.data_ptr(), self.status.data_ptr()
        p.k_scale = k_scale.data_ptr() if coded else None
        p.v_scale = v_scale.data_ptr() if coded else None
        p.k_strides[:], p.v_strides[:] = keys.stride()[:3], values.stride()[:3]
        p.pages, p.page_size, p.heads, p.head_dim, p.type = pages, page_size, heads, head_dim, _lib.TYPES[keys.dtype]
        self._append, self._attend = DlmAppend(), DlmAttend()  # what every call starts from
        self._append.cache = self._attend.cache = p
        self._append.pdl = self._attend.pdl = 1
        # Everything of a call's arguments but addresses -> its descriptor, checked and filled in but for these. Calls copy
        # it, so concurrent callers share nothing. Checking and filling anew took 10 of a small call's 16 us. The last one of
        # each kind is compared first: that spares hashing thirty attributes.
        self._plans = {}
        self._last_append = self._last_attend = (None, None)
        _lib.lib()

    def check(self):
        """Raises IndexError for the first slot, position, page or length outside its table since the last check
        (synchronises the current stream)."""
        _index_error(self.status, "PagedKV", self.page_size)

    def _given(self, name, t, dtype, shape):
        if t.dtype != dtype or t.shape != shape or t.device != self.device:
            raise ValueError(f"{name}: expected {dtype} {tuple(shape)} on {self.device}, got {t.dtype} {tuple(t.shape)} on "
                             f"{t.device}")

    def _type(self, t):
        if t.dtype not in (torch.bfloat16, torch.float16) or (t.dtype != self.dtype and self.dtype != torch.float8_e4m3fn):
            raise ValueError(f"{t.dtype} tokens for a cache of {self.dtype}")
        return _lib.TYPES[t.dtype]

    def append(self, k, v, positions, slots, table=None, q=None, q_out=None, q_norm=None, k_norm=None, eps=1e-6,
               interleaved=False):
        """Stores the keys and values of n new tokens in their slots and returns the rotated queries (None without `q`).

        `k`, `v` [n, kv heads, head dim], `q` [n, query heads, head dim]: BF16 or FP16, any strides that are multiples of 8
        with a contiguous head dimension (slices of one qkv projection). `slots` [n] int64: page * page size + place in the
        page, each at most once in a call; negative: a padded row, which stores nothing. `positions` [n] int32: row of
        `table` (see `rotary_table`, whose width says how many elements of a head are rotated; None: no rotation, and positions are
        not looked at).
        `interleaved`: pairs are neighbours, not a half apart. `q_norm`, `k_norm` [head dim]: weights of an RMSNorm over each
        head in front of the rotation. `q_out` may be `q`, but no other
        tensor that shares elements with `q`, `k` or `v`; by default a new contiguous tensor. `k` and `v` are not part of the
        cache."""
        if table is not None and positions is None:
            raise ValueError("a rotation by `table` needs positions")
        key = (k.shape, k.stride(), k.dtype, k.device, v.shape, v.stride(), v.dtype, v.device, slots.shape, slots.stride(),
               slots.dtype, slots.device, eps, interleaved,
               None if table is None else (table.shape, table.stride(), table.dtype, table.device, positions.shape,
                                           positions.stride(), positions.dtype, positions.device),
               None if q is None else (q.shape, q.stride(), q.dtype, q.device),
               None if q_out is None else (q_out.shape, q_out.stride(), q_out.dtype, q_out.device),
               None if q_norm is None else (q_norm.shape, q_norm.stride(), q_norm.dtype, q_norm.device),
               None if k_norm is None else (k_norm.shape, k_norm.stride(), k_norm.dtype, k_norm.device))
        last, plan = self._last_append
        if key != last:
            plan = self._plans.get(key)
            if plan is None:
                plan = self._plan_append(k, v, positions, slots, table, q, q_out, q_norm, k_norm, eps, interleaved)
                self._remember(key, plan)
            self._last_append = key, plan
        if q is not None and q_out is None:
            q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        a = DlmAppend.from_buffer_copy(plan)
        _APPEND.pack_into(a, _APPEND_AT, 0 if q is None else q.data_ptr(), k.data_ptr(), v.data_ptr(),
                          0 if q is None else q_out.data_ptr(), 0 if table is None else positions.data_ptr(), slots.data_ptr(),
                          0 if table is None else table.data_ptr(), 0 if q_norm is None else q_norm.data_ptr(),
                          0 if k_norm is None else k_norm.data_ptr())
        code = _lib.launch("dlm_paged_append", a, self.device)
        if code:
            _lib.check(code, f"PagedKV.append of {k.shape[0]} tokens")
        return q_out

    def _remember(self, key, plan):
        if len(self._plans) >= _MOST_PLANS:
            self._plans.clear()
        self._plans[key] = plan

    def _plan_append(self, k, v, positions, slots, table, q, q_out, q_norm, k_norm, eps, interleaved):
        """The checked descriptor of an append, without addresses."""
        n = k.shape[0]
        shape = (n, self.heads, self.head_dim)
        a = DlmAppend.from_buffer_copy(self._append)
        a.type = self._type(k)
        self._given("k", k, k.dtype, shape)
        self._given("v", v, k.dtype, shape)
        self._given("slots", slots, torch.int64, (n,))
        kt, kh, k1 = k.stride()
        vt, vh, v1 = v.stride()
        if k1 != 1 or v1 != 1 or not slots.is_contiguous():
            raise ValueError("k and v must have a contiguous head dimension, slots must be contiguous")
        a.n, a.eps = n, eps
        a.k_strides[:], a.v_strides[:] = (kt, kh), (vt, vh)
        if table is not None:
            self._given("table", table, torch.float32, table.shape)
            self._given("positions", positions, torch.int32, (n,))
            if table.dim() != 2 or not table.is_contiguous() or not positions.is_contiguous():
                raise ValueError("table must be contiguous [positions, rotated], positions contiguous")
            if not table.shape[0] or not 16 <= table.shape[1] <= self.head_dim or table.shape[1] % 16:
                raise ValueError(f"table {tuple(table.shape)}: its width is a multiple of 16 up to {self.head_dim}")
            a.table_rows, a.rotated = table.shape
            a.interleaved = bool(interleaved)
        for name, norm in (("q_norm", q_norm), ("k_norm", k_norm)):
            if norm is not None:
                self._given(name, norm, k.dtype, (self.head_dim,))
                if not norm.is_contiguous():
                    raise ValueError(f"{name} must be contiguous")
        if q is not None:
            if q.dim() != 3:
                raise ValueError(f"q must be [n, query heads, head dim], got {tuple(q.shape)}")
            self._given("q", q, k.dtype, (n, q.shape[1], self.head_dim))
            if q_out is not None:
                self._given("q_out", q_out, q.dtype, q.shape)
            qt, qh, q1 = q.stride()
            ot, oh, o1 = (q.shape[1] * q.shape[2], q.shape[2], 1) if q_out is None else q_out.stride()
            if q1 != 1 or o1 != 1:
                raise ValueError("q and q_out must have a contiguous head dimension")
            a.q_heads = q.shape[1]
            a.q_strides[:], a.out_strides[:] = (qt, qh), (ot, oh)
        elif q_out is not None or q_norm is not None:
            raise ValueError("q_out and q_norm come with q")
        return a

    def attend(self, q, pages, lengths, out=None, lse=None, scale=None, window=0, causal=False):
        """Attention of the last `tokens` tokens of each sequence over its cached keys; returns `out`, shaped like `q`.

        `q` [batch, tokens, query heads, head dim] (or [batch, query heads, head dim] for one token each), already rotated,
        its keys and values appended. `pages` [batch, most pages] int32 lists each sequence's pages (entries past its length
        are not read), `lengths` [batch] int32 how many keys it has, the new tokens included. Every token sees all of them
        (a block refined as a whole), with `causal` those up to its own; with `window` only keys less than that many
        positions before it. A token that sees none gets zeros. `scale`: of the scores, head dim ** -0.5 by default. `out`
        may be `q`, but no other tensor that shares elements with it. `lse` [batch, tokens, query heads] FP32, if given, takes the logarithm of the softmax's denominator
        (-inf for a token that sees no key): what is needed to join the result with attention over other keys."""
        key = (q.shape, q.stride(), q.dtype, q.device, pages.shape, pages.stride(), pages.dtype, pages.device, lengths.shape,
               lengths.stride(), lengths.dtype, lengths.device, scale, window, causal,
               None if out is None else (out.shape, out.stride(), out.dtype, out.device),
               None if lse is None else (lse.shape, lse.stride(), lse.dtype, lse.device))
        last, plan = self._last_attend
        if key != last:
            plan = self._plans.get(key)
            if plan is None:
                plan = self._plan_attend(q, pages, lengths, out, lse, scale, window, causal)
                self._remember(key, plan)
            self._last_attend = key, plan
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        a = DlmAttend.from_buffer_copy(plan)
        room = plan.workspace_bytes
        # Scratch is of this call alone: calls on other streams, and captured graphs, have their own.
        scratch = torch.empty(room, device=self.device, dtype=torch.uint8) if room else None
        _ATTEND.pack_into(a, _ATTEND_AT, q.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(), pages.data_ptr(),
                          lengths.data_ptr(), scratch.data_ptr() if room else 0, room)
        code = _lib.launch("dlm_paged_attend", a, self.device)
        if code:
            _lib.check(code, f"PagedKV.attend of {tuple(q.shape)} over {tuple(pages.shape)} pages")
        return out

    def _plan_attend(self, q, pages, lengths, out, lse, scale, window, causal):
        """The checked descriptor of an attention call, without addresses; its workspace_bytes are what the call needs."""
        single = q.dim() == 3
        q4 = q.unsqueeze(1) if single else q
        if q4.dim() != 4 or q4.shape[3] != self.head_dim:
            raise ValueError(f"q must be [batch, tokens, query heads, {self.head_dim}], got {tuple(q.shape)}")
        b, t, hq, d = q4.shape
        a = DlmAttend.from_buffer_copy(self._attend)
        a.type = self._type(q)
        if hq % self.heads or not hq:
            raise ValueError(f"{hq} query heads do not share {self.heads} kv heads evenly")
        if q.device != self.device:
            raise ValueError(f"q is on {q.device}, the cache on {self.device}")
        if pages.dim() != 2 or pages.shape[0] != b:
            raise ValueError(f"pages must be [{b}, most pages], got {tuple(pages.shape)}")
        self._given("pages", pages, torch.int32, pages.shape)
        self._given("lengths", lengths, torch.int32, (b,))
        if out is not None:
            self._given("out", out, q.dtype, q.shape)
            out4 = out.unsqueeze(1) if single else out
        (qb, qt, qh, q1), (pb, p1) = q4.stride(), pages.stride()
        ob, ot, oh, o1 = (t * hq * d, hq * d, d, 1) if out is None else out4.stride()
        if q1 != 1 or o1 != 1 or (p1 != 1 and pages.shape[1] > 1) or not lengths.is_contiguous():
            raise ValueError("q and out must have a contiguous head dimension, pages contiguous rows; lengths are contiguous")
        if lse is not None:
            self._given("lse", lse, torch.float32, (b, hq) if single else (b, t, hq))
            if not lse.is_contiguous():
                raise ValueError("lse must be contiguous")
        if window < 0:
            raise ValueError(f"window {window}: expected the number of keys, or 0 for all")
        a.q_strides[:], a.out_strides[:] = (qb, qt, qh), (ob, ot, oh)
        a.table_stride, a.table_pages = pb, pages.shape[1]
        # A cache has at most 2^30 keys: a longer window is all of them.
        a.batch, a.tokens, a.q_heads, a.window, a.causal = b, t, hq, min(window, 1 << 30), bool(causal)
        a.scale = d ** -0.5 if scale is None else scale
        with torch.cuda.device(self.device) if self.device.type == "cuda" else nullcontext():  # it asks how many SMs there are
            a.workspace_bytes = _lib.lib().dlm_paged_attend_workspace_bytes(a)
        return a
