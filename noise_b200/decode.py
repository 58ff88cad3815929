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
import functools
import math

import torch

from . import _lib

MAX_NODES = 64
MAX_VOCAB = 393216
KINDS = {'bf16': 0, 'e4m3': 1, 'int8': 2}
CODES = {'bf16': torch.bfloat16, 'e4m3': torch.float8_e4m3fn, 'int8': torch.int8}
DTYPES = {torch.float32: 0, torch.bfloat16: 1}
EPS = {t: torch.finfo(t).eps for t in DTYPES}  # F.rms_norm's


def _need(ok, message):
    if not ok:
        raise ValueError(message)


def _rows(name, t, dims, device):
    """The checks every floating operand of ``dims`` dimensions gets; the last dimension is contiguous."""
    if t.dim() != dims or (t.stride(-1) != 1 and t.shape[-1] > 1):
        raise ValueError(f'{name}: {dims} dimensions, the last one contiguous; got {tuple(t.shape)}, strides {t.stride()}')
    if t.device != device:
        raise ValueError(f'{name}: on {t.device}, expected {device}')


def _ints(name, t, dtype, shape, device):
    if t.dtype != dtype:
        raise TypeError(f'{name}: {dtype}, got {t.dtype}')
    if t.shape != shape or not t.is_contiguous() or t.device != device:
        raise ValueError(f'{name}: contiguous {tuple(shape)} on {device}, got {tuple(t.shape)} on {t.device}')


def _call(name, device, *args):
    """The entry point on the device's current stream, with the device current."""
    fn = getattr(_lib.lib(), name)
    if torch.cuda.current_device() == device.index:
        rc = fn(*args, _lib.stream_handle(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _lib.stream_handle(device))
    if rc:
        _lib.check(rc, name)


# ---- head norm and rotation -----------------------------------------------------------------------------------


def _head_args(q, k, cos, sin, positions, q_weight, k_weight, eps):
    """The checks of both directions; (tokens, D, the arguments that both calls share)."""
    _lib.require_cuda(q, k, cos, sin, positions)
    dev, dtype, table = q.device, q.dtype, cos.dtype
    if dtype not in DTYPES or k.dtype != dtype:
        raise TypeError(f'q and k: fp32 or bf16, alike; got {dtype}, {k.dtype}')
    if table not in DTYPES or sin.dtype != table:
        raise TypeError(f'cos and sin: fp32 or bf16, alike; got {table}, {sin.dtype}')
    _rows('q', q, 3, dev)
    _rows('k', k, 3, dev)
    (tokens, heads, dim), (k_tokens, k_heads, k_dim) = q.shape, k.shape
    if k_tokens != tokens or k_dim != dim:
        raise ValueError(f'q [tokens, heads, D], k [tokens, k heads, D]: got {tuple(q.shape)}, {tuple(k.shape)}')
    if dim < 2 or dim > 256 or dim % 2:
        raise ValueError(f'D: even, 2 to 256; got {dim}')
    if not (0 < heads <= 4096 and 0 < k_heads <= 4096):
        raise ValueError(f'heads: 1 to 4096; got {heads}, {k_heads}')
    shape = cos.shape
    if (len(shape) != 2 or shape[1] * 2 != dim or shape[0] < 1 or sin.shape != shape or not cos.is_contiguous() or
            not sin.is_contiguous() or cos.device != dev or sin.device != dev):
        raise ValueError(f'cos, sin: contiguous [positions, {dim // 2}] on {dev}, got {tuple(shape)}, {tuple(sin.shape)}')
    _ints('positions', positions, torch.int32, (tokens,), dev)
    weights = [None, None]
    for i, w in enumerate((q_weight, k_weight)):
        if w is not None:
            name = 'qk'[i] + '_weight'
            if w.dtype != dtype:
                raise TypeError(f'{name}: {dtype}, got {w.dtype}')
            if w.shape != (dim,) or not w.is_contiguous() or w.device != dev:
                raise ValueError(f'{name}: contiguous [{dim}] on {dev}, got {tuple(w.shape)} on {w.device}')
            weights[i] = w.data_ptr()
    eps = EPS[dtype] if eps is None else float(eps)
    if not 0 <= eps < math.inf:
        raise ValueError(f'eps: {eps}')
    return (_heads(q), _heads(k), cos.data_ptr(), sin.data_ptr(), DTYPES[table], shape[0], positions.data_ptr(),
            tokens, dim, DTYPES[dtype], *weights, eps)


def _heads(t):
    return _lib.Heads(t.data_ptr(), t.stride(0), t.stride(1), t.shape[1])


def _ptr(t):
    return None if t is None else t.data_ptr()


def _head_forward(q, k, cos, sin, positions, q_weight, k_weight, eps):
    args = _head_args(q, k, cos, sin, positions, q_weight, k_weight, eps)
    q_out, k_out = q.new_empty(q.shape), k.new_empty(k.shape)
    _call('noise_head_norm_rope', q.device, *args, q_out.data_ptr(), k_out.data_ptr())
    return q_out, k_out


def head_norm_rope_backward(dq, dk, q, k, cos, sin, positions, q_weight=None, k_weight=None, eps=None):
    """Gradient of ``head_norm_rope``: (q's, k's, q_weight's, k_weight's) from the outputs' gradients dq, dk and the call's
    own arguments. The weights' are fp32 [D], summed over tokens and heads in a fixed order, None without a weight."""
    args = _head_args(q, k, cos, sin, positions, q_weight, k_weight, eps)
    _lib.require_cuda(dq, dk)
    dev, dim = q.device, q.shape[2]
    if dq.dtype != q.dtype or dk.dtype != q.dtype:
        raise TypeError(f'dq and dk: {q.dtype}, got {dq.dtype}, {dk.dtype}')
    _rows('dq', dq, 3, dev)
    _rows('dk', dk, 3, dev)
    if dq.shape != q.shape or dk.shape != k.shape:
        raise ValueError(f'dq, dk: {tuple(q.shape)}, {tuple(k.shape)}; got {tuple(dq.shape)}, {tuple(dk.shape)}')
    gq, gk = q.new_empty(q.shape), k.new_empty(k.shape)
    gqw = None if q_weight is None else torch.empty(dim, dtype=torch.float32, device=dev)
    gkw = None if k_weight is None else torch.empty(dim, dtype=torch.float32, device=dev)
    nbytes, ws = 0, None
    if gqw is not None or gkw is not None:
        nbytes = _lib.lib().noise_head_norm_rope_backward_workspace_bytes(dim)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _call('noise_head_norm_rope_backward', dev, _heads(dq), _heads(dk), *args, gq.data_ptr(), gk.data_ptr(),
          _ptr(gqw), _ptr(gkw), _ptr(ws), nbytes)
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

    def _places(self, seq, pos, table, layer):
        _lib.require_cuda(seq, pos, table)
        shape = seq.shape
        if len(shape) != 1 or table.dim() != 2:
            raise ValueError(f'seq [tokens], table [sequences, pages]: got {tuple(shape)}, {tuple(table.shape)}')
        _ints('seq', seq, torch.int32, shape, self.device)
        _ints('pos', pos, torch.int32, shape, self.device)
        _ints('table', table, torch.int32, table.shape, self.device)
        if layer is None:
            return shape[0], 0, self.layers
        if not 0 <= layer < self.layers:
            raise ValueError(f'layer: 0 to {self.layers - 1}, or None for all; got {layer}')
        return shape[0], layer, 1

    def write(self, k, v, seq, pos, table, layer=0, rows=None):
        """Write keys and values of token i at position pos[i] of sequence seq[i] (int32 [tokens]; negative: skipped).

        k, v [source rows, heads, D], fp32 or bf16, any strides but the last; entry i takes row rows[i] (int32 [tokens];
        negative: skipped), or row i. layer None: all layers at once, k, v [layers, source rows, heads, D]. An entry out
        of range is skipped and reported by ``check()``; no two entries of a call may share a place."""
        _lib.require_cuda(k, v)
        tokens, first, layers = self._places(seq, pos, table, layer)
        if k.dtype not in DTYPES or v.dtype != k.dtype:
            raise TypeError(f'k and v: fp32 or bf16, alike; got {k.dtype}, {v.dtype}')
        dims = 4 if layer is None else 3
        _rows('k', k, dims, self.device)
        _rows('v', v, dims, self.device)
        source = k.shape[-3]
        want = (self.layers, source, self.heads, self.dim) if layer is None else (source, self.heads, self.dim)
        if k.shape != want or v.shape != want:
            raise ValueError(f'k, v: {want}, got {tuple(k.shape)}, {tuple(v.shape)}')
        if rows is not None:
            _lib.require_cuda(rows)
            _ints('rows', rows, torch.int32, seq.shape, self.device)
            rows = rows.data_ptr()
        elif source < tokens:
            raise ValueError(f'{tokens} tokens, but {source} rows')
        _call('noise_kv_write', self.device, self._struct, first, layers, k.data_ptr(), k.stride(0), k.stride(-3),
              k.stride(-2), v.data_ptr(), v.stride(0), v.stride(-3), v.stride(-2), source, DTYPES[k.dtype], tokens,
              seq.data_ptr(), pos.data_ptr(), rows, table.data_ptr(), table.shape[0], table.shape[1])

    def read(self, seq, pos, table, layer=0, dtype=torch.bfloat16):
        """(k, v) [tokens, heads, D] at those places, or [layers, ...] for layer None. bf16 holds every value of every kind
        exactly. Negative seq or pos: zeros; out of range: NaN."""
        tokens, first, layers = self._places(seq, pos, table, layer)
        if dtype not in DTYPES:
            raise TypeError(f'dtype: fp32 or bf16, got {dtype}')
        shape = (layers, tokens, self.heads, self.dim) if layer is None else (tokens, self.heads, self.dim)
        k = torch.empty(shape, dtype=dtype, device=self.device)
        v = torch.empty(shape, dtype=dtype, device=self.device)
        _call('noise_kv_read', self.device, self._struct, first, layers, k.data_ptr(), v.data_ptr(), DTYPES[dtype],
              tokens, seq.data_ptr(), pos.data_ptr(), table.data_ptr(), table.shape[0], table.shape[1])
        return k, v

    def check(self):
        """Raise if a call since the last check met an index out of range (synchronises the current stream)."""
        with torch.cuda.device(self.device):
            code = _lib.read_status(self.status)
        if code:
            _call('noise_clear_status', self.device, self.status.data_ptr())
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
    _call('noise_tree_plan', parents.device, parents.data_ptr(), *parents.shape, mask.data_ptr(), depth.data_ptr())
    return mask, depth


@functools.lru_cache(maxsize=256)
def _attention_bytes(*sizes):
    return max(_lib.lib().noise_tree_attention_workspace_bytes(*sizes), 16)


def tree_attention(q, k, v, cache, table, lengths, mask, depth, layer=0, window=-1, scale=None):
    """Attention of the trees' nodes over each sequence's ``lengths[b]`` cached tokens and over the trees themselves.

    q [B, N, heads, D], k, v [B, N, cache.heads, D] bf16 (the nodes' own, not yet in the cache), D 64 or 128; table
    int32 [B, pages]; lengths int32 [B]; mask, depth: ``tree_plan``'s, or any mask int64 [B, N] of the nodes that each node
    sees. Node n stands at position lengths[b] + depth[b, n] and sees what is at most ``window`` positions back
    (negative: all), as utils/model.py:17-21. scale: 1 / sqrt(D). Returns bf16 [B, N, heads, D]; rows of padding
    (depth below 0) and of nodes that see nothing are 0."""
    _lib.require_cuda(q, k, v, table, lengths, mask, depth)
    dev = cache.device
    if not q.dtype == k.dtype == v.dtype == torch.bfloat16:
        raise TypeError(f'q, k, v: bf16, got {q.dtype}, {k.dtype}, {v.dtype}')
    _rows('q', q, 4, dev)
    _rows('k', k, 4, dev)
    _rows('v', v, 4, dev)
    (seqs, nodes, heads, dim), k_heads = q.shape, cache.heads
    if dim != cache.dim or dim not in (64, 128):
        raise ValueError(f'D: the cache\'s, 64 or 128; got {dim}, the cache has {cache.dim}')
    want = (seqs, nodes, k_heads, dim)
    if k.shape != want or v.shape != want:
        raise ValueError(f'k, v: {want}, got {tuple(k.shape)}, {tuple(v.shape)}')
    if not 1 <= nodes <= MAX_NODES:
        raise ValueError(f'nodes: 1 to {MAX_NODES}, got {nodes}')
    if heads < k_heads or heads % k_heads or heads // k_heads > 64:
        raise ValueError(f'q heads: a multiple of the cache\'s {k_heads}, at most 64 times it; got {heads}')
    if table.dim() != 2 or table.shape[0] != seqs:
        raise ValueError(f'table: [{seqs}, pages], got {tuple(table.shape)}')
    _ints('table', table, torch.int32, table.shape, dev)
    _ints('lengths', lengths, torch.int32, (seqs,), dev)
    _ints('mask', mask, torch.int64, (seqs, nodes), dev)
    _ints('depth', depth, torch.int32, (seqs, nodes), dev)
    if not 0 <= layer < cache.layers:
        raise ValueError(f'layer: 0 to {cache.layers - 1}, got {layer}')
    # the kernel copies 16 bytes at a time
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    if q.data_ptr() % 16 or (qs[0] | qs[1] | qs[2]) % 8:
        q = q.contiguous()
        qs = q.stride()
    if k.data_ptr() % 16 or (ks[0] | ks[1] | ks[2]) % 8:
        k = k.contiguous()
        ks = k.stride()
    if v.data_ptr() % 16 or (vs[0] | vs[1] | vs[2]) % 8:
        v = v.contiguous()
        vs = v.stride()
    out = torch.empty((seqs, nodes, heads, dim), dtype=torch.bfloat16, device=dev)
    nbytes = _attention_bytes(seqs, nodes, heads, k_heads, dim)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _call('noise_tree_attention', dev, cache._struct, layer, q.data_ptr(), qs[0], qs[1], qs[2], heads, k.data_ptr(),
          ks[0], ks[1], ks[2], v.data_ptr(), vs[0], vs[1], vs[2], seqs, nodes, table.data_ptr(), table.shape[1],
          lengths.data_ptr(), mask.data_ptr(), depth.data_ptr(), window, dim ** -0.5 if scale is None else scale,
          out.data_ptr(), ws.data_ptr(), nbytes)
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
    dev, dtype = logits.device, logits.dtype
    if dtype not in DTYPES:
        raise TypeError(f'logits: fp32 or bf16, got {dtype}')
    _rows('logits', logits, 3, dev)
    seqs, nodes, vocab = logits.shape
    if not 1 <= nodes <= MAX_NODES:
        raise ValueError(f'nodes: 1 to {MAX_NODES}, got {nodes}')
    if not 1 <= vocab <= MAX_VOCAB:
        raise ValueError(f'vocabulary: 1 to {MAX_VOCAB}, got {vocab}')
    if not (0 <= temperature < math.inf and 0 <= softcap < math.inf):
        raise ValueError(f'temperature and softcap: at least 0; got {temperature}, {softcap}')
    shape = (seqs, nodes)
    _ints('tokens', tokens, torch.int64, shape, dev)
    _ints('parents', parents, torch.int32, shape, dev)
    u_ptr = race_ptr = q_ptr = None
    q_seq = q_node = 0
    if temperature > 0:
        _lib.require_cuda(u, race)
        _ints('u', u, torch.float32, shape, dev)
        _ints('race', race, torch.float32, (seqs, vocab), dev)
        u_ptr, race_ptr = u.data_ptr(), race.data_ptr()
        if probs is not None:
            _lib.require_cuda(probs)
            if probs.dtype != torch.float32:
                raise TypeError(f'probs: fp32, got {probs.dtype}')
            _rows('probs', probs, 3, dev)
            if probs.shape != logits.shape:
                raise ValueError(f'probs: {tuple(logits.shape)}, got {tuple(probs.shape)}')
            q_ptr, q_seq, q_node = probs.data_ptr(), probs.stride(0), probs.stride(1)
    count = torch.empty(seqs, dtype=torch.int32, device=dev)
    path = torch.empty(shape, dtype=torch.int32, device=dev)
    token = torch.empty(seqs, dtype=torch.int64, device=dev)
    _call('noise_verify_tree', dev, logits.data_ptr(), DTYPES[dtype], logits.stride(0), logits.stride(1),
          tokens.data_ptr(), parents.data_ptr(), u_ptr, race_ptr, q_ptr, q_seq, q_node, seqs, nodes, vocab, temperature,
          softcap, count.data_ptr(), path.data_ptr(), token.data_ptr())
    return count, path, token
