"""Cases of the operators that let the trained GPT answer several tokens a step: per-head norm and rotation, the
quantised cache, attention for a tree of drafted tokens over it, and the tokens' verification.

``run`` is the plain form (elementary torch operations, 32 bits, one rounding at the end), or with ``own`` the calls a
user makes of ``noise_b200.decode``. ``exact`` is the definition in 64 bits.

Shapes the operators share:
- a tree of N nodes a sequence: ``parents`` [B, N], the root (the last sampled token) first with parent -1, padding -2;
  ``mask`` [B, N] int64, bit j: the node sees node j (its ancestors and itself); ``depth`` [B, N], -1 for padding;
- the paged cache: K [layers, pages, heads, page, D], V [layers, pages, heads, page / 4, D, 4] (four tokens side by
  side), a scale byte e + 127 for each (token, head) of K and of V in the 8-bit kinds: value = code * 2^e;
  ``table`` [B, pages of a sequence] gives the page of each position.
"""
import math

import torch

own = False

QMAX = {'e4m3': 448.0, 'int8': 127.0}
CODE = {'e4m3': torch.float8_e4m3fn, 'int8': torch.int8, 'bf16': torch.bfloat16}
FLOAT = {'fp32': torch.float32, 'bf16': torch.bfloat16}
SIZE = {'fp32': 4, 'bf16': 2, 'e4m3': 1, 'int8': 1}


def listed():
    return [
        # one decoding step of 8 sequences of the framework's GPT: 8 heads of 64, queries and keys of one projection
        dict(name='heads_step', op='heads', tokens=8, q_heads=8, k_heads=8, dim=64, dtype='bf16', weights=False),
        # the prompts of a batch of 8 rows of 2,048 tokens, the same heads
        dict(name='heads_prompt', op='heads', tokens=16384, q_heads=8, k_heads=8, dim=64, dtype='bf16', weights=False),
        # gradient of the same rows kept in fp32, as the framework keeps its residual stream
        dict(name='heads_grad', op='heads_grad', tokens=2048, q_heads=8, k_heads=8, dim=64, dtype='fp32',
             weights=False),
        # a training step of wider, grouped heads with learned norms and an odd count of tokens
        dict(name='heads_grad_wide', op='heads_grad', tokens=12287, q_heads=32, k_heads=8, dim=128, dtype='bf16',
             weights=True),
        # a decoding step's 8 tokens written to the cache and read back
        dict(name='cache_step', op='cache', tokens=8, seqs=8, heads=8, dim=64, page=64, kind='e4m3'),
        # 8 prompts of 4,096 tokens of 8 wide heads
        dict(name='cache_prompt', op='cache', tokens=32768, seqs=8, heads=8, dim=128, page=64, kind='int8'),
        # one token a sequence of the framework's GPT in a windowed block, unquantised cache, ragged lengths
        dict(name='attend_token', op='attend', seqs=8, nodes=1, branch=1, shortest=100, longest=2048, q_heads=8,
             k_heads=8, dim=64, page=64, kind='bf16', window=1024),
        # a tree of 16 drafted tokens a sequence over rows of 2,048
        dict(name='attend_tree', op='attend', seqs=32, nodes=16, branch=2, shortest=1021, longest=2048, q_heads=8,
             k_heads=8, dim=64, page=64, kind='e4m3', window=-1),
        # single tokens over long documents, grouped heads
        dict(name='attend_long', op='attend', seqs=8, nodes=1, branch=1, shortest=8193, longest=65536, q_heads=32,
             k_heads=8, dim=128, page=64, kind='e4m3', window=-1),
        # the largest tree, 64 nodes, over grouped heads
        dict(name='attend_tree_wide', op='attend', seqs=8, nodes=64, branch=3, shortest=4000, longest=8192,
             q_heads=32, k_heads=8, dim=128, page=64, kind='int8', window=-1),
        # 4 sequences, chains of 5 nodes, the framework's vocabulary
        dict(name='verify_chain', op='verify', seqs=4, nodes=5, branch=1, vocab=4096, dtype='fp32', probs=True,
             temperature=1.0, softcap=15.0),
        # 32 sequences, trees of 32 nodes, a large odd vocabulary
        dict(name='verify_tree', op='verify', seqs=32, nodes=32, branch=3, vocab=50001, dtype='fp32', probs=True,
             temperature=0.8, softcap=0.0),
    ]


def draw(rng):
    """One more case of the listed ranges, none costlier than the largest listed one."""
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    op = rng.choice(['heads', 'heads_grad', 'cache', 'attend', 'attend', 'verify'])
    most = {'heads': 3.7e8, 'heads_grad': 3.7e8, 'cache': 4e8, 'attend': 6e8, 'verify': 2e8}[op]
    while True:
        if op in ('heads', 'heads_grad'):
            q_heads, k_heads = rng.choice([(8, 8), (8, 2), (32, 8), (12, 4)])
            case = dict(op=op, tokens=spread(1, 16384), q_heads=q_heads, k_heads=k_heads, dim=rng.choice([64, 128]),
                        dtype=rng.choice(['bf16', 'bf16', 'fp32']), weights=rng.random() < 0.5)
        elif op == 'cache':
            seqs = spread(1, 64)
            case = dict(op=op, tokens=seqs * spread(1, 4096), seqs=seqs, heads=rng.choice([2, 8]),
                        dim=rng.choice([64, 128]), page=rng.choice([16, 64]), kind=rng.choice(['bf16', 'e4m3', 'int8']))
        elif op == 'attend':
            q_heads, k_heads = rng.choice([(8, 8), (8, 2), (32, 8)])
            longest = spread(1, 65536)
            case = dict(op=op, seqs=spread(1, 64), nodes=rng.choice([1, 1, spread(2, 64)]), branch=rng.choice([1, 2, 3]),
                        shortest=rng.randint(0, longest), longest=longest, q_heads=q_heads, k_heads=k_heads,
                        dim=rng.choice([64, 128]), page=rng.choice([16, 64]),
                        kind=rng.choice(['bf16', 'e4m3', 'int8']), window=rng.choice([-1, -1, 1024]))
            rows = case['seqs'] * longest
            if rows * k_heads * case['dim'] > 4.2e8 or rows * q_heads * case['nodes'] > 1.35e8:
                continue  # the plain form's fp32 keys and scores stay within the listed cases' own
        else:
            case = dict(op=op, seqs=spread(1, 64), nodes=spread(1, 64), branch=rng.choice([1, 2, 3]),
                        vocab=spread(1000, 50001), dtype=rng.choice(['bf16', 'fp32']), probs=rng.random() < 0.7,
                        temperature=rng.choice([0.0, 0.8, 1.0]), softcap=rng.choice([0.0, 15.0]))
            if case['seqs'] * case['nodes'] * case['vocab'] > 5.1e7:
                continue
        if work(case)['bytes'] <= most:
            return case


def _lengths(case):
    """Cached tokens of each sequence: evenly from the longest down to the shortest."""
    n, lo, hi = case['seqs'], case['shortest'], case['longest']
    return [hi - (hi - lo) * b // max(1, n - 1) for b in range(n)]


def _tree(case):
    """parents [B, N]: a full tree of ``branch`` children a node; every third sequence drafted a node less."""
    n, f = case['nodes'], case['branch']
    rows = [[-1] + [(i - 1) // f for i in range(1, n)] for _ in range(case['seqs'])]
    for b in range(2, case['seqs'], 3):
        if n > 2:
            rows[b][-1] = -2
    return rows


def _visited(case):
    """Nodes whose logits a walk needs, on average: it goes on from a node with children about every other time."""
    depth = 0 if case['nodes'] == 1 else int(math.log(case['nodes'], case['branch'])) if case['branch'] > 1 else \
        case['nodes'] - 1
    return sum(0.5 ** i for i in range(depth + 1))


def work(case):
    op = case['op']
    if op in ('heads', 'heads_grad'):
        values = case['tokens'] * (case['q_heads'] + case['k_heads']) * case['dim']
        tables = case['tokens'] * 4 + min(case['tokens'], 2048) * case['dim'] * 2
        return {'bytes': values * SIZE[case['dtype']] * (2 if op == 'heads' else 3) + tables,
                'flops': values * (7 if op == 'heads' else 16)}
    if op == 'cache':
        rows = 2 * case['tokens'] * case['heads']  # of K and of V; read, written, read back, written out
        code = case['dim'] * SIZE[case['kind']] + (case['kind'] != 'bf16')
        return {'bytes': rows * (case['dim'] * 4 + 2 * code) + case['tokens'] * 8, 'flops': rows * case['dim'] * 4}
    if op == 'attend':
        seen = [min(n, case['window'] + 1) if case['window'] >= 0 else n for n in _lengths(case)]
        code = 2 * (case['dim'] * SIZE[case['kind']] + (case['kind'] != 'bf16'))
        new = case['seqs'] * case['nodes'] * case['dim'] * 2
        return {'bytes': sum(seen) * case['k_heads'] * code + new * 2 * (case['q_heads'] + case['k_heads']),
                'flops': 4 * case['nodes'] * case['q_heads'] * case['dim'] * sum(n + case['nodes'] for n in seen)}
    rows = case['seqs'] * _visited(case)
    row = case['vocab'] * (SIZE[case['dtype']] + (4 if case['probs'] and case['temperature'] > 0 else 0))
    race = case['seqs'] * case['vocab'] * 4 if case['temperature'] > 0 else 0
    return {'bytes': rows * row + race, 'flops': rows * case['vocab'] * 6}


# ---- inputs ---------------------------------------------------------------------------------------------------


def _split(codes):
    """V's rows [..., page, D] as the cache keeps them, four tokens side by side."""
    *lead, page, dim = codes.shape
    raw = codes.view(torch.int8) if codes.element_size() == 1 else codes
    return raw.reshape(*lead, page // 4, 4, dim).transpose(-1, -2).contiguous().view(codes.dtype)


def _joined(v):
    """The rows [..., page, D] of V as the cache keeps it."""
    *lead, quads, dim, _ = v.shape
    raw = v.view(torch.int8) if v.element_size() == 1 else v
    return raw.transpose(-1, -2).reshape(*lead, 4 * quads, dim).view(v.dtype)


def _quantised(x, kind):
    """(codes, scale bytes) of rows x [..., D]; the scale 2^e is the least with |x| <= 2^e * QMAX."""
    if kind == 'bf16':
        return x.to(torch.bfloat16), None
    x = x.float()
    m, e = torch.frexp(x.abs().amax(-1) / QMAX[kind])  # m in [0.5, 1): the least power of two is 2^e, or 2^(e - 1)
    e = torch.where(m == 0.5, e - 1, e)
    e = torch.where(m == 0, -126, e).clamp(-126, 127)
    y = torch.ldexp(x, -e[..., None])
    codes = y.round().to(torch.int8) if kind == 'int8' else y.to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8)


def _scaled(codes, scale):
    """fp32 values of codes [..., D] and their scale bytes (None: none)."""
    x = codes.float()
    return x if scale is None else torch.ldexp(x, scale[..., None].int() - 127)


def _table(case, pages, gen):
    """Pages of the sequences' positions, in no order; [B, pages of a sequence]."""
    return torch.randperm(case['seqs'] * pages, generator=gen, device='cuda').int().view(case['seqs'], pages)


def _masks(parents):
    """(mask, depth) of a tree's rows of parents."""
    mask, depth = [], []
    for i, p in enumerate(parents):
        mask.append(0 if p == -2 else (1 << i) | (mask[p] if p >= 0 else 0))
        depth.append(-1 if p == -2 else bin(mask[i]).count('1') - 1)
    return [m - (1 << 64) if m >= 1 << 63 else m for m in mask], depth


def prepare(case, seed):
    gen = torch.Generator('cuda').manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=gen, device='cuda').to(dtype)
    op, s = case['op'], {'case': case}
    if op in ('heads', 'heads_grad'):
        t, hq, hk, d, dt = case['tokens'], case['q_heads'], case['k_heads'], case['dim'], FLOAT[case['dtype']]
        qkv = normal(t, (hq + 2 * hk), d, dtype=dt) * 1.5  # queries, keys and values of one projection
        s['q'], s['k'] = qkv[:, :hq], qkv[:, hq:hq + hk]
        angle = torch.outer(torch.arange(2048, device='cuda').float(),
                            1e4 ** (-torch.arange(0, d, 2, device='cuda').float() / d))
        s['cos'], s['sin'] = angle.cos().bfloat16(), angle.sin().bfloat16()
        s['positions'] = torch.arange(t, device='cuda', dtype=torch.int32) % 2048 if t >= 2048 else \
            torch.randint(0, 2048, (t,), generator=gen, device='cuda', dtype=torch.int32)
        for n in ('q', 'k'):
            s[n + '_weight'] = (1 + 0.2 * normal(d)).to(dt) if case['weights'] else None
        if op == 'heads_grad':
            s['dq'], s['dk'] = normal(t, hq, d, dtype=dt), normal(t, hk, d, dtype=dt)
        return s
    if op == 'verify':
        b, n, v = case['seqs'], case['nodes'], case['vocab']
        s['parents'] = torch.tensor(_tree(case), dtype=torch.int32, device='cuda')
        draft = 2.5 * normal(b, n, v)
        s['logits'] = (draft + 0.7 * normal(b, n, v)).to(FLOAT[case['dtype']])  # the draft is near the target
        probs = torch.softmax(draft, -1)
        from_ = s['parents'].clamp(min=0).long()
        race = torch.empty(b, n, v, device='cuda').exponential_(generator=gen)
        s['tokens'] = (torch.gather(probs, 1, from_[..., None].expand(b, n, v)) / race).argmax(-1)
        s['probs'] = probs if case['probs'] else None
        del draft, race
        s['u'] = torch.rand(b, n, generator=gen, device='cuda')
        s['race'] = torch.empty(b, v, device='cuda').exponential_(generator=gen)
        return s
    b, d, page, kind = case['seqs'], case['dim'], case['page'], case['kind']
    if op == 'cache':
        t, h, each = case['tokens'], case['heads'], case['tokens'] // b
        pages = -(-(each + 7) // page)
        s['k'], s['v'] = normal(t, h, d, dtype=torch.bfloat16), normal(t, h, d, dtype=torch.bfloat16)
        s['seq'] = torch.arange(b, device='cuda', dtype=torch.int32).repeat_interleave(each)
        s['pos'] = torch.arange(each, device='cuda', dtype=torch.int32).repeat(b) + 7  # after a few earlier tokens
        store = (torch.zeros(1, b * pages, h, page, d, device='cuda', dtype=torch.bfloat16).to(CODE[kind]),
                 torch.zeros(1, b * pages, h, page // 4, d, 4, device='cuda', dtype=torch.bfloat16).to(CODE[kind]))
        scales = (None, None) if kind == 'bf16' else tuple(
            torch.zeros(1, b * pages, h, page, device='cuda', dtype=torch.uint8) for _ in range(2))
    else:
        n, hq, h = case['nodes'], case['q_heads'], case['k_heads']
        lengths = _lengths(case)
        pages = max(1, -(-max(lengths) // page))
        s['lengths'] = torch.tensor(lengths, dtype=torch.int32, device='cuda')
        plan = [_masks(p) for p in _tree(case)]
        s['mask'] = torch.tensor([m for m, _ in plan], dtype=torch.int64, device='cuda')
        s['depth'] = torch.tensor([x for _, x in plan], dtype=torch.int32, device='cuda')
        # queries and keys after their head norms (rows of norm sqrt(D)), sharper than the norm alone leaves them
        s['q'] = (1.5 * normal(b, n, hq, d)).bfloat16()
        s['k'], s['v'] = normal(b, n, h, d, dtype=torch.bfloat16), normal(b, n, h, d, dtype=torch.bfloat16)
        kc, ks = _quantised(normal(b * pages, h, page, d, dtype=torch.bfloat16), kind)
        vc, vs = _quantised(normal(b * pages, h, page, d, dtype=torch.bfloat16), kind)
        store, scales = (kc[None], _split(vc)[None]), (ks if ks is None else ks[None], vs if vs is None else vs[None])
    s['table'] = _table(case, pages, gen)
    s['store'], s['scales'] = store, scales
    if own:  # the handle a program keeps
        from noise_b200.decode import KVCache
        s['cache'] = KVCache.of(*store, *scales)
    return s


# ---- one pass -------------------------------------------------------------------------------------------------


def run(s):
    op = s['case']['op']
    if own:
        from noise_b200 import decode
        if op == 'heads':
            return decode.head_norm_rope(s['q'], s['k'], s['cos'], s['sin'], s['positions'], s['q_weight'],
                                         s['k_weight'])
        if op == 'heads_grad':
            return decode.head_norm_rope_backward(s['dq'], s['dk'], s['q'], s['k'], s['cos'], s['sin'],
                                                  s['positions'], s['q_weight'], s['k_weight'])
        if op == 'cache':
            s['cache'].write(s['k'], s['v'], s['seq'], s['pos'], s['table'])
            return s['cache'].read(s['seq'], s['pos'], s['table'])
        if op == 'attend':
            return decode.tree_attention(s['q'], s['k'], s['v'], s['cache'], s['table'], s['lengths'], s['mask'],
                                         s['depth'], window=s['case']['window'])
        return decode.verify_tree(s['logits'], s['tokens'], s['parents'], s['u'], s['race'], s['probs'],
                                  temperature=s['case']['temperature'], softcap=s['case']['softcap'])
    return {'heads': _heads, 'heads_grad': _heads_grad, 'cache': _cache, 'attend': _attend, 'verify': _verify}[op](s)


def _eps(x):
    return torch.finfo(x.dtype).eps


def _rotated(x, c, s):
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c + b * s, b * c - a * s], -1)


def _angles(s):
    at = s['positions'].long()
    return s['cos'][at].float()[:, None], s['sin'][at].float()[:, None]


def _heads(s):
    c, sn = _angles(s)

    def one(x, w):
        y = x.float()
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + _eps(x))
        return _rotated(y if w is None else y * w.float(), c, sn).to(x.dtype)
    return one(s['q'], s['q_weight']), one(s['k'], s['k_weight'])


def _heads_grad(s):
    c, sn = _angles(s)

    def one(dy, x, w):
        y = x.float()
        r = torch.rsqrt((y * y).mean(-1, keepdim=True) + _eps(x))
        y = y * r
        g = _rotated(dy.float(), c, -sn)  # the rotation back
        h = g if w is None else g * w.float()
        dx = r * (h - y * (h * y).mean(-1, keepdim=True))
        return dx.to(x.dtype), None if w is None else (g * y).sum((0, 1))
    (dq, wq), (dk, wk) = one(s['dq'], s['q'], s['q_weight']), one(s['dk'], s['k'], s['k_weight'])
    return dq, dk, wq, wk


def _cache(s):
    page, kind = s['case']['page'], s['case']['kind']
    pos = s['pos'].long()
    at, slot = s['table'][s['seq'].long(), pos // page].long(), pos % page
    out = []
    for i, x in enumerate((s['k'], s['v'])):
        codes, scale = _quantised(x, kind)
        store = s['store'][i][0]
        raw, new = (store.view(torch.int8), codes.view(torch.int8)) if kind != 'bf16' else (store, codes)
        if i == 0:
            raw[at, :, slot] = new
            back = raw[at, :, slot]
        else:
            raw[at, :, slot // 4, :, slot % 4] = new
            back = raw[at, :, slot // 4, :, slot % 4]
        if scale is not None:
            s['scales'][i][0][at, :, slot] = scale
            scale = s['scales'][i][0][at, :, slot]
        out.append(_scaled(back.view(CODE[kind]), scale).bfloat16())
    return tuple(out)


def _attend(s):
    case, table = s['case'], s['table'].long()
    b, n, hq, d = s['q'].shape
    h, group, room = case['k_heads'], case['q_heads'] // case['k_heads'], table.shape[1] * case['page']

    def cached(store, scale, back):  # [B, heads, positions, D]
        x = _scaled(back(store[0]), None if scale is None else scale[0])[table]
        return x.transpose(1, 2).reshape(b, h, room, d)
    k = torch.cat([cached(s['store'][0], s['scales'][0], lambda z: z), s['k'].float().transpose(1, 2)], 2)
    v = torch.cat([cached(s['store'][1], s['scales'][1], _joined), s['v'].float().transpose(1, 2)], 2)
    q = s['q'].float().view(b, n, h, group, d).permute(0, 2, 3, 1, 4)  # [B, heads, group, N, D]
    at = torch.arange(room, device='cuda')
    length, depth = s['lengths'][:, None, None], s['depth'][..., None]
    sees = (at < length).expand(b, n, room)
    node = torch.arange(n, device='cuda')
    tree = (s['mask'][..., None] >> node & 1).bool()
    if case['window'] >= 0:
        sees = sees & (length + depth - at <= case['window'])
        tree = tree & (depth - depth.transpose(1, 2) <= case['window'])
    sees = torch.cat([sees, tree], 2) & (depth >= 0)
    scores = q.reshape(b, h, group * n, d) @ k.transpose(2, 3) * d ** -0.5
    scores = scores.view(b, h, group, n, -1).masked_fill(~sees[:, None, None], float('-inf'))
    most = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(most == float('-inf'), 0.0, most))
    total = p.sum(-1, keepdim=True)
    o = (p.view(b, h, group * n, -1) @ v).view(b, h, group, n, d) / torch.where(total == 0, 1.0, total)
    return o.permute(0, 3, 1, 2, 4).reshape(b, n, hq, d).bfloat16()


def _capped(z, case):
    return case['softcap'] * torch.tanh(z / case['softcap']) if case['softcap'] > 0 else z


def _verify(s):
    """Every node's children are judged at once, a rank among the siblings at a time; then each node is reached if its
    parents were accepted."""
    case, parents, tokens = s['case'], s['parents'].long(), s['tokens']
    b, n = tokens.shape
    node = torch.arange(n, device='cuda')
    same = (parents[:, :, None] == parents[:, None]) & (parents[:, None] >= 0) & (node[:, None] > node)
    rank = torch.where(parents >= 0, same.sum(-1), -1)
    z = _capped(s['logits'].float(), case)
    won = torch.full((b, n), -1, device='cuda')  # the accepted child of each node
    rows = torch.arange(b, device='cuda')[:, None]
    greedy = case['temperature'] == 0
    if greedy:
        best = z.argmax(-1)
    else:
        z = z / case['temperature']
        p = torch.exp(z - z.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        left, mass = p.clone(), torch.ones(b, n, device='cuda')
    for r in range(case['branch']):
        is_r = (rank == r)[:, None] & (parents[:, None] == node[:, None])  # [B, parent, child]
        child = torch.where(is_r.any(-1), is_r.int().argmax(-1), -1)
        token = tokens[rows, child.clamp(min=0)]
        tried = (child >= 0) & (won < 0)
        if greedy:
            ok = token == best
        else:
            value = left.gather(2, token[..., None])[..., 0]
            chance = s['probs'].gather(2, token[..., None])[..., 0] if case['probs'] else 1.0
            ok = s['u'][rows, child.clamp(min=0)] * mass * chance < value
            lost = tried & ~ok
            q = s['probs'] if case['probs'] else torch.zeros_like(left).scatter_(2, token[..., None], 1.0)
            new = (left / torch.where(mass > 0, mass, 1.0)[..., None] - q).clamp(min=0)
            left = torch.where(lost[..., None], new, left)
            mass = torch.where(lost, new.sum(-1), mass)
        won = torch.where(tried & ok, child, won)
    at, path = torch.zeros(b, dtype=torch.int64, device='cuda'), [torch.zeros(b, dtype=torch.int64, device='cuda')]
    for _ in range(n - 1):  # down the accepted children
        nxt = torch.where(path[-1] >= 0, won[rows[:, 0], at], -1)
        at = torch.where(nxt >= 0, nxt, at)
        path.append(nxt)
    path = torch.stack(path, 1)
    if greedy:
        token = best[rows[:, 0], at]
    else:
        last, whole = left[rows[:, 0], at], p[rows[:, 0], at]
        last = torch.where((mass[rows[:, 0], at] > 0)[:, None], last, whole)
        token = (last / s['race']).argmax(-1)
    return (path >= 0).sum(1).int() - 1, path.int(), token


# ---- the definition in 64 bits --------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {'heads': _exact_heads, 'heads_grad': _exact_heads, 'cache': _exact_cache, 'attend': _exact_attend,
            'verify': _exact_verify}[case['op']](s, case)


def _exact_heads(s, case):
    """Rotation as a complex product; the gradient from torch's differentiation of the forward."""
    c, sn = (s[n].double()[s['positions'].long()] for n in ('cos', 'sin'))
    turn = torch.complex(c, -sn)[:, None]
    outs, grads = [], []
    for n in ('q', 'k'):
        x = s[n].double().requires_grad_()
        w = torch.ones(case['dim'], dtype=torch.float64, device='cuda') if s[n + '_weight'] is None else \
            s[n + '_weight'].double()
        w.requires_grad_()
        y = w * x / torch.sqrt(x.square().sum(-1, keepdim=True) / case['dim'] + torch.finfo(s[n].dtype).eps)
        half = case['dim'] // 2
        z = torch.complex(y[..., :half], y[..., half:]) * turn
        y = torch.cat([z.real, z.imag], -1)
        outs.append(y.detach())
        if case['op'] == 'heads_grad':
            grads.append(torch.autograd.grad((y * s['d' + n].double()).sum(), (x, w)))
    if case['op'] == 'heads':
        return tuple(outs)
    (dq, wq), (dk, wk) = grads
    return (dq, dk) + ((wq, wk) if case['weights'] else (None, None))


def _exact_cache(s, case):
    """The nearest value on the grid of a row's scale, ties to even."""
    out = []
    for x in (s['k'].double(), s['v'].double()):
        if case['kind'] != 'bf16':
            top = x.abs().amax(-1, keepdim=True) / QMAX[case['kind']]
            scale = torch.exp2(torch.ceil(torch.log2(top) - 1e-12).clamp(-126, 127))  # log2 is a last bit off
            step = torch.ones_like(x)
            if case['kind'] == 'e4m3':  # 3 bits after the leading one, from 2^-6 up
                step = torch.exp2(torch.floor(torch.log2((x / scale).abs().clamp(min=2.0 ** -6)) + 1e-12) - 3)
            x = torch.round(x / scale / step) * step * scale
        out.append(x)
    return tuple(out)


def _exact_attend(s, case):
    """One sequence and one key head at a time, over the keys that are there."""
    b, n, hq, d = s['q'].shape
    group, page = hq // case['k_heads'], case['page']
    out = torch.zeros(b, n, hq, d, dtype=torch.float64, device='cuda')
    for i, length in enumerate(_lengths(case)):
        pos = torch.arange(length, device='cuda')
        at, slot = s['table'][i].long()[pos // page], pos % page
        mask, depth = s['mask'][i], s['depth'][i].long()
        where = torch.cat([pos, length + depth])
        sees = torch.cat([torch.ones(n, length, dtype=torch.bool, device='cuda'),
                          (mask[:, None] >> torch.arange(n, device='cuda')) % 2 == 1], 1)
        if case['window'] >= 0:
            sees &= (length + depth)[:, None] <= where + case['window']
        real = depth >= 0
        for h in range(case['k_heads']):
            rows = []
            for j, new in enumerate((s['k'], s['v'])):
                store = s['store'][j][0]
                raw = store if case['kind'] == 'bf16' else store.view(torch.int8)
                x = raw[at, h, slot] if j == 0 else raw[at, h, slot // 4, :, slot % 4]
                x = x.contiguous().view(store.dtype).double()
                if case['kind'] != 'bf16':
                    x = x * torch.exp2(s['scales'][j][0][at, h, slot].double() - 127)[:, None]
                rows.append(torch.cat([x, new[i, :, h].double()]))
            q = s['q'][i, real, h * group:(h + 1) * group].double()
            a = torch.einsum('ngd,kd->ngk', q, rows[0]) / math.sqrt(d)
            a = a.masked_fill(~sees[real][:, None], float('-inf')).softmax(-1)
            out[i, real, h * group:(h + 1) * group] = torch.einsum('ngk,kd->ngd', a, rows[1])
    return out


def _exact_verify(s, case):
    """The walk itself, one sequence after another."""
    b, n = s['tokens'].shape
    counts, paths, tokens = [], [], []
    parents, drafted, u = (s[k].tolist() for k in ('parents', 'tokens', 'u'))
    for i in range(b):
        at, path = 0, [0]
        while True:
            z = s['logits'][i, at].double()
            if case['softcap'] > 0:
                z = case['softcap'] * torch.tanh(z / case['softcap'])
            if case['temperature'] > 0:
                p = (z / case['temperature']).softmax(-1)
            r, found = (p if case['temperature'] > 0 else None), None
            for c in (c for c in range(1, n) if parents[i][c] == at):
                x = drafted[i][c]
                if r is None:
                    found = c if x == int(z.argmax()) else None
                else:
                    q = s['probs'][i, at].double() if case['probs'] else torch.zeros_like(r).index_fill_(
                        0, torch.tensor([x], device='cuda'), 1.0)
                    if u[i][c] * float(r.sum()) * float(q[x]) < float(r[x]):
                        found = c
                    elif float(r.sum()) > 0:
                        r = (r / r.sum() - q).clamp(min=0)
                if found is not None:
                    break
            if found is None:
                break
            at = found
            path.append(at)
        if r is None:
            tokens.append(int(z.argmax()))
        else:
            tokens.append(int(((r if float(r.sum()) > 0 else p) / s['race'][i].double()).argmax()))
        counts.append(len(path) - 1)
        paths.append(path + [-1] * (n - len(path)))
    return (torch.tensor(counts, dtype=torch.int32), torch.tensor(paths, dtype=torch.int32), torch.tensor(tokens))
