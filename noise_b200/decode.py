"""Operators that let the trained GPT answer, several tokens a step, on libnoise_b200.so.

The reference trains only; these continue its block (utils/model.py:81-97) and head (utils/model.py:202-209) past a
prompt. A step takes a tree of up to 64 tokens a sequence: the last sampled token as its root and drafted ones under it
(``parents``, -1 for the root, an earlier node for the others, -2 for padding); a single node is plain decoding.

- ``head_norm_rope(q, k, cos, sin, positions, ...)``: the per-head norm and the rotation of queries and keys in one
  pass; differentiable (``head_norm_rope_backward`` is its gradient as a call).
- ``KVCache``: a paged cache of keys and values in bf16 or in 8 bits, quantised as it is written (``write``), read back
  by ``read`` and by ``tree_attention``.
- ``tree_plan(parents)``: the nodes' masks and depths.
- ``tree_attention(q, k, v, cache, table, lengths, mask, depth, ...)``: the tree's attention over the cache and itself.
- ``verify_tree(logits, tokens, parents, u, race, probs, ...)``: how many drafts the target accepts, and the next token.

Each call runs on the current stream of its tensors' device, allocates with torch and reads nothing back. Arguments are
checked before a pointer reaches the library (TypeError for a dtype, ValueError for a shape, layout or device).
"""
import ctypes
import math

import torch

from . import _lib

MAX_NODES = 64
KINDS = {'bf16': 0, 'e4m3': 1, 'int8': 2}
CODES = {'bf16': torch.bfloat16, 'e4m3': torch.float8_e4m3fn, 'int8': torch.int8}
DTYPES = {torch.float32: 0, torch.bfloat16: 1}


def _need(ok, message):
    if not ok:
        raise ValueError(message)


def _rows(name, t, dims, device=None):
    """The checks every floating operand of ``dims`` dimensions gets; the last dimension is contiguous."""
    if t.dim() != dims or (t.stride(-1) != 1 and t.shape[-1] > 1):
        raise ValueError(f'{name}: {dims} dimensions, the last one contiguous; got {tuple(t.shape)}, strides {t.stride()}')
    if device is not None and t.device != device:
        raise ValueError(f'{name}: on {t.device}, expected {device}')


def _ints(name, t, dtype, shape, device):
    if t.dtype != dtype:
        raise TypeError(f'{name}: {dtype}, got {t.dtype}')
    if tuple(t.shape) != shape or not t.is_contiguous() or t.device != device:
        raise ValueError(f'{name}: contiguous {shape} on {device}, got {tuple(t.shape)} on {t.device}')


class _On:
    """The device's current stream handle, with the device current while the call is made."""

    def __init__(self, device):
        self.device = device
        self.guard = torch.cuda.device(device) if torch.cuda.current_device() != device.index else None

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        return _lib.stream_handle(self.device)

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)
        return False


# ---- head norm and rotation -----------------------------------------------------------------------------------


def _head_args(q, k, cos, sin, positions, q_weight, k_weight, eps):
    _lib.require_cuda(q, k, cos, sin, positions)
    dev = q.device
    if q.dtype not in DTYPES or k.dtype != q.dtype:
        raise TypeError(f'q and k: fp32 or bf16, alike; got {q.dtype}, {k.dtype}')
    if cos.dtype not in DTYPES or sin.dtype != cos.dtype:
        raise TypeError(f'cos and sin: fp32 or bf16, alike; got {cos.dtype}, {sin.dtype}')
    _rows('q', q, 3)
    _rows('k', k, 3, dev)
    tokens, heads, dim = q.shape
    _need(k.shape[0] == tokens and k.shape[2] == dim, f'q [tokens, heads, D] and k [tokens, k heads, D]: got '
          f'{tuple(q.shape)}, {tuple(k.shape)}')
    _need(2 <= dim <= 256 and dim % 2 == 0, f'D: even, 2 to 256; got {dim}')
    _need(0 < heads <= 4096 and 0 < k.shape[1] <= 4096, 'heads: 1 to 4096')
    _need(cos.dim() == 2 and cos.shape == sin.shape and cos.shape[1] == dim // 2 and cos.shape[0] > 0 and
          cos.is_contiguous() and sin.is_contiguous() and cos.device == dev and sin.device == dev,
          f'cos, sin: contiguous [positions, {dim // 2}] on {dev}, got {tuple(cos.shape)}, {tuple(sin.shape)}')
    _ints('positions', positions, torch.int32, (tokens,), dev)
    for name, w in (('q_weight', q_weight), ('k_weight', k_weight)):
        if w is not None:
            if w.dtype != q.dtype:
                raise TypeError(f'{name}: {q.dtype}, got {w.dtype}')
            _need(tuple(w.shape) == (dim,) and w.is_contiguous() and w.device == dev,
                  f'{name}: contiguous [{dim}] on {dev}, got {tuple(w.shape)}')
    if eps is None:
        eps = torch.finfo(q.dtype).eps
    _need(math.isfinite(eps) and eps >= 0, f'eps: {eps}')
    return tokens, dim, float(eps)


def _heads(t):
    return ctypes.byref(_lib.Heads(t.data_ptr(), t.stride(0), t.stride(1), t.shape[1]))


def _ptr(t):
    return None if t is None else t.data_ptr()


def _head_forward(q, k, cos, sin, positions, q_weight, k_weight, eps):
    tokens, dim, eps = _head_args(q, k, cos, sin, positions, q_weight, k_weight, eps)
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    k_out = torch.empty(k.shape, dtype=q.dtype, device=q.device)
    with _On(q.device) as stream:
        _lib.check(_lib.lib().noise_head_norm_rope(
            _heads(q), _heads(k), cos.data_ptr(), sin.data_ptr(), DTYPES[cos.dtype], cos.shape[0],
            positions.data_ptr(), tokens, dim, DTYPES[q.dtype], _ptr(q_weight), _ptr(k_weight), eps,
            q_out.data_ptr(), k_out.data_ptr(), stream), 'noise_head_norm_rope')
    return q_out, k_out


def head_norm_rope_backward(dq, dk, q, k, cos, sin, positions, q_weight=None, k_weight=None, eps=None):
    """Gradient of ``head_norm_rope``: (q's, k's, q_weight's, k_weight's) from the outputs' gradients dq, dk and the call's
    own arguments. The weights' are fp32 [D], summed over tokens and heads in a fixed order, None without a weight."""
    tokens, dim, eps = _head_args(q, k, cos, sin, positions, q_weight, k_weight, eps)
    dev = q.device
    for name, d, x in (('dq', dq, q), ('dk', dk, k)):
        if d.dtype != q.dtype:
            raise TypeError(f'{name}: {q.dtype}, got {d.dtype}')
        _rows(name, d, 3, dev)
        _need(d.shape == x.shape, f'{name}: {tuple(x.shape)}, got {tuple(d.shape)}')
    gq = torch.empty(q.shape, dtype=q.dtype, device=dev)
    gk = torch.empty(k.shape, dtype=q.dtype, device=dev)
    gqw = None if q_weight is None else torch.empty(dim, dtype=torch.float32, device=dev)
    gkw = None if k_weight is None else torch.empty(dim, dtype=torch.float32, device=dev)
    L, nbytes, ws = _lib.lib(), 0, None
    if gqw is not None or gkw is not None:
        nbytes = L.noise_head_norm_rope_backward_workspace_bytes(dim)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    with _On(dev) as stream:
        _lib.check(L.noise_head_norm_rope_backward(
            _heads(dq), _heads(dk), _heads(q), _heads(k), cos.data_ptr(), sin.data_ptr(), DTYPES[cos.dtype],
            cos.shape[0], positions.data_ptr(), tokens, dim, DTYPES[q.dtype], _ptr(q_weight), _ptr(k_weight), eps,
            gq.data_ptr(), gk.data_ptr(), _ptr(gqw), _ptr(gkw), _ptr(ws), nbytes, stream),
            'noise_head_norm_rope_backward')
    return gq, gk, gqw, gkw


class _HeadNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, eps):
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.eps = eps
        return _head_forward(q, k, cos, sin, positions, q_weight, k_weight, eps)

    @staticmethod
    def backward(ctx, dq, dk):
        q, k, q_weight, k_weight, cos, sin, positions = ctx.saved_tensors
        dq, dk = (d if d.stride(-1) == 1 else d.contiguous() for d in (dq, dk))  # (an expanded gradient)
        gq, gk, gqw, gkw = head_norm_rope_backward(dq, dk, q, k, cos, sin, positions, q_weight, k_weight, ctx.eps)
        return (gq, gk, None if gqw is None else gqw.to(q_weight.dtype),
                None if gkw is None else gkw.to(k_weight.dtype), None, None, None, None)


def head_norm_rope(q, k, cos, sin, positions, q_weight=None, k_weight=None, eps=None):
    """(q', k'): each head's row divided by its RMS (eps: finfo(dtype).eps, as F.rms_norm), times a weight if given,
    rotated by its position: norm and apply_rotary_emb of utils/model.py:46-47, 55-58 in one pass.

    q [tokens, heads, D], k [tokens, k heads, D]: fp32 or bf16, views of one projection's rows as they are; cos, sin
    [positions, D / 2] fp32 or bf16; positions int32 [tokens] (one outside the tables gives NaN); weights [D], shared by
    the heads. Outputs are contiguous, of q's dtype. Gradients reach q, k and the weights."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        return _HeadNormRope.apply(q, k, q_weight, k_weight, cos, sin, positions, eps)
    return _head_forward(q, k, cos, sin, positions, q_weight, k_weight, eps)


# ---- the cache ------------------------------------------------------------------------------------------------


class KVCache:
    """Keys and values of ``pages`` pages of ``page_size`` tokens for ``layers`` layers of ``heads`` heads of ``dim``.

    kind: 'bf16'; 'e4m3' or 'int8': 8-bit codes under a power of two for each (token, head) of K and of V. Which page
    holds which positions is the caller's: every call takes ``table`` int32 [sequences, pages of a sequence].

    ``k`` [layers, pages, heads, page_size, dim], ``v`` [layers, pages, heads, page_size / 4, dim, 4] and, in 8 bits,
    ``k_scale``, ``v_scale`` uint8 [layers, pages, heads, page_size] (value = code * 2^(byte - 127)) are plain tensors;
    ``status`` is the device's error word: ``check()`` raises if a call met an index out of range."""

    def __init__(self, layers, pages, heads, dim, kind='e4m3', page_size=64, device='cuda'):
        _need(kind in KINDS, f'kind: one of {sorted(KINDS)}')
        _need(min(layers, pages, heads) > 0 and heads <= 4096, 'layers, pages, heads: at least 1; at most 4096 heads')
        _need(16 <= page_size <= 4096 and page_size & (page_size - 1) == 0, 'page_size: a power of two, 16 to 4096')
        _need(16 <= dim <= 256 and dim % 16 == 0, 'dim: a multiple of 16, 16 to 256')
        raw = CODES[kind] if kind != 'e4m3' else torch.uint8  # (zeros of a float8 type are made as bytes)
        k = torch.zeros(layers, pages, heads, page_size, dim, dtype=raw, device=device).view(CODES[kind])
        v = torch.zeros(layers, pages, heads, page_size // 4, dim, 4, dtype=raw, device=device).view(CODES[kind])
        scales = (None, None) if kind == 'bf16' else (
            torch.zeros(layers, pages, heads, page_size, dtype=torch.uint8, device=device) for _ in range(2))
        self._set(k, v, *scales)

    @classmethod
    def of(cls, k, v, k_scale=None, v_scale=None):
        """A cache over tensors that are there already (of the shapes above)."""
        self = cls.__new__(cls)
        self._set(k, v, k_scale, v_scale)
        return self

    def _set(self, k, v, k_scale, v_scale):
        _lib.require_cuda(k, v)
        kinds = [n for n, t in CODES.items() if t == k.dtype]
        if not kinds or v.dtype != k.dtype:
            raise TypeError(f'k, v: one of {sorted(map(str, CODES.values()))}; got {k.dtype}, {v.dtype}')
        self.kind = kinds[0]
        _need(k.dim() == 5, f'k: [layers, pages, heads, page_size, dim], got {tuple(k.shape)}')
        layers, pages, heads, page, dim = k.shape
        _need(min(k.shape) > 0 and heads <= 4096 and 16 <= page <= 4096 and page & (page - 1) == 0 and
              16 <= dim <= 256 and dim % 16 == 0, f'k: pages of a power of two of tokens, 16 to 4096, dim a multiple of '
              f'16, 16 to 256; got {tuple(k.shape)}')
        _need(tuple(v.shape) == (layers, pages, heads, page // 4, dim, 4), f'v: [.., page_size / 4, dim, 4], got '
              f'{tuple(v.shape)}')
        scales = (k_scale, v_scale)
        if self.kind == 'bf16':
            _need(k_scale is None and v_scale is None, 'a bf16 cache has no scales')
        else:
            for name, t in zip(('k_scale', 'v_scale'), scales):
                _need(t is not None and t.dtype == torch.uint8 and t.shape == k.shape[:4] and t.is_contiguous() and
                      t.device == k.device, f'{name}: contiguous uint8 {tuple(k.shape[:4])} on {k.device}')
        _need(k.is_contiguous() and v.is_contiguous() and v.device == k.device, 'k, v: contiguous, on one device')
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.layers, self.pages, self.heads, self.page_size, self.dim = layers, pages, heads, page, dim
        self.device = k.device
        self.status = torch.zeros(64, dtype=torch.int32, device=k.device)
        for t in (k, v) + tuple(s for s in scales if s is not None):
            _need(t.data_ptr() % 16 == 0, 'the cache\'s tensors: on 16-byte boundaries')
        self._struct = _lib.KVCache(k.data_ptr(), v.data_ptr(), _ptr(k_scale), _ptr(v_scale), self.status.data_ptr(),
                                    layers, pages, heads, page, dim, KINDS[self.kind])
        self._ref = ctypes.byref(self._struct)

    def _places(self, seq, pos, table, layer):
        tokens = seq.shape[0]
        _ints('seq', seq, torch.int32, (tokens,), self.device)
        _ints('pos', pos, torch.int32, (tokens,), self.device)
        _need(table.dim() == 2, f'table: [sequences, pages], got {tuple(table.shape)}')
        _ints('table', table, torch.int32, tuple(table.shape), self.device)
        _need(layer is None or 0 <= layer < self.layers, f'layer: 0 to {self.layers - 1}, or None for all')
        return tokens, (0, self.layers) if layer is None else (layer, 1)

    def write(self, k, v, seq, pos, table, layer=0, rows=None):
        """Write keys and values of token i at position pos[i] of sequence seq[i] (int32 [tokens]; negative: skipped).

        k, v [source rows, heads, D], fp32 or bf16, any strides but the last; entry i takes row rows[i] (int32 [tokens];
        negative: skipped), or row i. layer None: all layers at once, k, v [layers, source rows, heads, D]. An entry out of range is
        skipped and reported by ``check()``."""
        _lib.require_cuda(k, v, seq, pos, table)
        tokens, (first, layers) = self._places(seq, pos, table, layer)
        if k.dtype not in DTYPES or v.dtype != k.dtype:
            raise TypeError(f'k and v: fp32 or bf16, alike; got {k.dtype}, {v.dtype}')
        dims = 4 if layer is None else 3
        _rows('k', k, dims, self.device)
        _rows('v', v, dims, self.device)
        source = k.shape[-3]
        want = ((self.layers,) if layer is None else ()) + (source, self.heads, self.dim)
        _need(tuple(k.shape) == want and tuple(v.shape) == want, f'k, v: {want}, got {tuple(k.shape)}, {tuple(v.shape)}')
        if rows is None:
            _need(source >= tokens, f'{tokens} tokens, but {source} rows')
        else:
            _ints('rows', rows, torch.int32, (tokens,), self.device)
        with _On(self.device) as stream:
            _lib.check(_lib.lib().noise_kv_write(
                self._ref, first, layers, k.data_ptr(), k.stride(0) if dims == 4 else 0, k.stride(-3), k.stride(-2),
                v.data_ptr(), v.stride(0) if dims == 4 else 0, v.stride(-3), v.stride(-2), source, DTYPES[k.dtype],
                tokens, seq.data_ptr(), pos.data_ptr(), _ptr(rows), table.data_ptr(), table.shape[0], table.shape[1],
                stream), 'noise_kv_write')

    def read(self, seq, pos, table, layer=0, dtype=torch.bfloat16):
        """(k, v) [tokens, heads, D] at those places, or [layers, ...] for layer None. bf16 holds every value of every kind
        exactly. Negative seq or pos: zeros; out of range: NaN."""
        _lib.require_cuda(seq, pos, table)
        tokens, (first, layers) = self._places(seq, pos, table, layer)
        if dtype not in DTYPES:
            raise TypeError(f'dtype: fp32 or bf16, got {dtype}')
        shape = ((layers,) if layer is None else ()) + (tokens, self.heads, self.dim)
        k, v = (torch.empty(shape, dtype=dtype, device=self.device) for _ in range(2))
        with _On(self.device) as stream:
            _lib.check(_lib.lib().noise_kv_read(
                self._ref, first, layers, k.data_ptr(), v.data_ptr(), DTYPES[dtype], tokens, seq.data_ptr(),
                pos.data_ptr(), table.data_ptr(), table.shape[0], table.shape[1], stream), 'noise_kv_read')
        return k, v

    def check(self):
        """Raise if a call since the last check met an index out of range (synchronises the current stream)."""
        with _On(self.device) as stream:
            code = _lib.read_status(self.status)
            if code:
                _lib.check(_lib.lib().noise_clear_status(self.status.data_ptr(), stream), 'noise_clear_status')
                raise _lib.NoiseError(f'a cache call met a sequence, position, row or page out of range (status {code})')


# ---- the tree -------------------------------------------------------------------------------------------------


def tree_plan(parents):
    """(mask int64, depth int32) [B, N] of trees ``parents`` int32 [B, N]: bit j of mask[b, i] is set if node i sees node
    j (its ancestors and itself); depth is the distance from the root. Padding (-2, or a parent that is not an earlier
    node of the tree): mask 0, depth -1."""
    _lib.require_cuda(parents)
    _need(parents.dim() == 2 and 1 <= parents.shape[1] <= MAX_NODES, f'parents: [B, N], N 1 to {MAX_NODES}; got '
          f'{tuple(parents.shape)}')
    _ints('parents', parents, torch.int32, tuple(parents.shape), parents.device)
    mask = torch.empty(parents.shape, dtype=torch.int64, device=parents.device)
    depth = torch.empty(parents.shape, dtype=torch.int32, device=parents.device)
    with _On(parents.device) as stream:
        _lib.check(_lib.lib().noise_tree_plan(parents.data_ptr(), parents.shape[0], parents.shape[1],
                                              mask.data_ptr(), depth.data_ptr(), stream), 'noise_tree_plan')
    return mask, depth


def tree_attention(q, k, v, cache, table, lengths, mask, depth, layer=0, window=-1, scale=None):
    """Attention of the trees' nodes over each sequence's ``lengths[b]`` cached tokens and over the trees themselves.

    q [B, N, heads, D], k, v [B, N, cache.heads, D] bf16 (the nodes' own, not yet in the cache), D 64 or 128; table
    int32 [B, pages]; lengths int32 [B]; mask, depth: ``tree_plan``'s, or any mask int64 [B, N] of the nodes that each node
    sees. Node n stands at position lengths[b] + depth[b, n] and sees what is at most ``window`` positions back
    (negative: all), as utils/model.py:17-21. scale: 1 / sqrt(D). Returns bf16 [B, N, heads, D]; rows of padding
    (depth below 0) and of nodes that see nothing are 0."""
    _lib.require_cuda(q, k, v, table, lengths, mask, depth)
    dev = cache.device
    for name, t in (('q', q), ('k', k), ('v', v)):
        if t.dtype != torch.bfloat16:
            raise TypeError(f'{name}: bf16, got {t.dtype}')
        _rows(name, t, 4, dev)
    seqs, nodes, heads, dim = q.shape
    want = (seqs, nodes, cache.heads, cache.dim)
    _need(dim == cache.dim and dim in (64, 128), f'D: the cache\'s, 64 or 128; got {dim}, the cache has {cache.dim}')
    _need(tuple(k.shape) == want and tuple(v.shape) == want, f'k, v: {want}, got {tuple(k.shape)}, {tuple(v.shape)}')
    _need(1 <= nodes <= MAX_NODES, f'nodes: 1 to {MAX_NODES}, got {nodes}')
    _need(heads >= cache.heads and heads % cache.heads == 0 and heads // cache.heads <= 64,
          f'q heads: a multiple of the cache\'s {cache.heads}, at most 64 times it; got {heads}')
    _need(table.dim() == 2 and table.shape[0] == seqs, f'table: [{seqs}, pages], got {tuple(table.shape)}')
    _ints('table', table, torch.int32, tuple(table.shape), dev)
    _ints('lengths', lengths, torch.int32, (seqs,), dev)
    _ints('mask', mask, torch.int64, (seqs, nodes), dev)
    _ints('depth', depth, torch.int32, (seqs, nodes), dev)
    _need(0 <= layer < cache.layers, f'layer: 0 to {cache.layers - 1}, got {layer}')
    # the kernel loads four values of q and of k at once
    if q.data_ptr() % 16 or any(x % 4 for x in q.stride()[:3]):
        q = q.contiguous()
    if k.data_ptr() % 8 or any(x % 4 for x in k.stride()[:3]):
        k = k.contiguous()
    out = torch.empty((seqs, nodes, heads, dim), dtype=torch.bfloat16, device=dev)
    L = _lib.lib()
    nbytes = L.noise_tree_attention_workspace_bytes(seqs, nodes, heads, cache.heads, dim)
    ws = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=dev)
    with _On(dev) as stream:
        _lib.check(L.noise_tree_attention(
            cache._ref, layer, q.data_ptr(), q.stride(0), q.stride(1), q.stride(2), heads, k.data_ptr(), k.stride(0),
            k.stride(1), k.stride(2), v.data_ptr(), v.stride(0), v.stride(1), v.stride(2), seqs, nodes,
            table.data_ptr(), table.shape[1], lengths.data_ptr(), mask.data_ptr(), depth.data_ptr(), window,
            dim ** -0.5 if scale is None else scale, out.data_ptr(), ws.data_ptr(), nbytes, stream),
            'noise_tree_attention')
    return out


def verify_tree(logits, tokens, parents, u, race, probs=None, temperature=1.0, softcap=0.0):
    """(count int32 [B], path int32 [B, N], token int64 [B]): the drafts that the target accepts, the nodes gone through
    (the root first, then -1), and the next token. Accepted and next tokens are distributed as the target's own.

    logits [B, N, V] fp32 or bf16: the target's at each node (row n: after node n's token), softcapped here as the
    framework's head does if ``softcap`` is given (15 for its GPT, 0: none) and divided by ``temperature`` (0: the
    largest logit, no random numbers); tokens int64, parents int32 [B, N]; u fp32 [B, N] uniform in [0, 1); race fp32
    [B, V] exponential; probs fp32 [B, N, V]: the draft's distribution at each node, from which its children were
    drawn, or None for drafts that were picked."""
    _lib.require_cuda(logits, tokens, parents)
    dev = logits.device
    if logits.dtype not in DTYPES:
        raise TypeError(f'logits: fp32 or bf16, got {logits.dtype}')
    _rows('logits', logits, 3)
    seqs, nodes, vocab = logits.shape
    _need(1 <= nodes <= MAX_NODES, f'nodes: 1 to {MAX_NODES}, got {nodes}')
    _need(1 <= vocab <= 393216, f'vocabulary: 1 to 393216, got {vocab}')
    _need(math.isfinite(temperature) and temperature >= 0, f'temperature: {temperature}')
    _need(math.isfinite(softcap) and softcap >= 0, f'softcap: {softcap}')
    _ints('tokens', tokens, torch.int64, (seqs, nodes), dev)
    _ints('parents', parents, torch.int32, (seqs, nodes), dev)
    if temperature > 0:
        _ints('u', u, torch.float32, (seqs, nodes), dev)
        _ints('race', race, torch.float32, (seqs, vocab), dev)
        if probs is not None:
            if probs.dtype != torch.float32:
                raise TypeError(f'probs: fp32, got {probs.dtype}')
            _rows('probs', probs, 3, dev)
            _need(probs.shape == logits.shape, f'probs: {tuple(logits.shape)}, got {tuple(probs.shape)}')
    else:
        u = race = probs = None
    count = torch.empty(seqs, dtype=torch.int32, device=dev)
    path = torch.empty((seqs, nodes), dtype=torch.int32, device=dev)
    token = torch.empty(seqs, dtype=torch.int64, device=dev)
    with _On(dev) as stream:
        _lib.check(_lib.lib().noise_verify_tree(
            logits.data_ptr(), DTYPES[logits.dtype], logits.stride(0), logits.stride(1), tokens.data_ptr(),
            parents.data_ptr(), _ptr(u), _ptr(race), _ptr(probs), 0 if probs is None else probs.stride(0),
            0 if probs is None else probs.stride(1), seqs, nodes, vocab, temperature, softcap, count.data_ptr(),
            path.data_ptr(), token.data_ptr(), stream), 'noise_verify_tree')
    return count, path, token
