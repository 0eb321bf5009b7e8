"""The surface-embedding operators under measurement: real calls over their real range.

Two operators on a table of embeddings, one row per face (or vertex) of a mesh:

- ``surface_embedding(index, embeddings, scale)``: the table looked up at an index image or at the
  faces' corners, ``out = scale * embeddings[index]`` (zeros where the index names no row), and
  the table's gradient, the sum of the incoming rows of each index;
- ``surface_cross_entropy(features, embeddings, labels, scale, reduction)``: the softmax cross
  entropy of pixel features against every row of the table, ``logits = scale * features @
  embeddings.T``, at the pixels whose label names a row, and the gradients of both.

``own`` False runs them as elementary torch operations; True runs the package's kernels.
"""
import math

import torch

own = False

_TYPES = {'f64': torch.float64, 'f32': torch.float32, 'f16': torch.float16,
          'bf16': torch.bfloat16}
_SIZES = {'f64': 8, 'f32': 4, 'f16': 2, 'bf16': 2}
_RADIUS = 0.8            # the rendered sphere's radius over half the image
_COVER = math.pi * _RADIUS * _RADIUS / 4  # the fraction of the pixels that it covers
_PIECE = 1 << 28         # logits held at a time by the plain form (1 GB in 32 bits)


def listed():
    return [
        # --- surface_embedding -----------------------------------------------------------------
        # picked pixels of one small view (a click, a few key points): latency
        dict(name='embed_points', op='embed', form='points', n=64, rows=1000, dim=32,
             dtype='f32', train=False),
        # a training step on four 256 x 256 views of 10,000 faces
        dict(name='embed_views', op='embed', form='image', views=4, size=256, rows=10000, dim=16,
             dtype='f32', train=True),
        # per-vertex features gathered at the corners of 200,000 faces, an odd number of channels
        dict(name='embed_corners', op='embed', form='corners', faces=200000, rows=100002, dim=37,
             dtype='f32', train=True),
        # a training step on eight 512 x 512 views of 50,000 faces, half precision
        dict(name='embed_step', op='embed', form='image', views=8, size=512, rows=50000, dim=64,
             dtype='bf16', train=True),
        # eight 1024 x 1024 views
        dict(name='embed_large', op='embed', form='image', views=8, size=1024, rows=50000, dim=32,
             dtype='f16', train=True),
        # --- surface_cross_entropy -------------------------------------------------------------
        # a hundred annotated points on a small mesh: latency of a training step
        dict(name='xent_points', op='xent', form='points', n=100, rows=1000, dim=16, dtype='f32',
             scale=10.0, reduction='mean', train=True),
        # one pixel against 200,000 faces: the interactive query
        dict(name='xent_pixel', op='xent', form='points', n=1, rows=200000, dim=256,
             dtype='bf16', scale=14.0, reduction='none', train=False),
        # odd sizes, half precision under a loss scale, a loss per pixel
        dict(name='xent_odd', op='xent', form='image', views=3, size=131, rows=997, dim=37,
             dtype='f16', scale=8.0, reduction='none', train=True),
        # a training step on four 256 x 256 views of 10,000 faces, 32 bits
        dict(name='xent_views', op='xent', form='image', views=4, size=256, rows=10000, dim=64,
             dtype='f32', scale=14.0, reduction='mean', train=True),
        # wide embeddings on one 512 x 512 view
        dict(name='xent_wide', op='xent', form='image', views=1, size=512, rows=10000, dim=256,
             dtype='bf16', scale=20.0, reduction='mean', train=True),
        # a training step on two 512 x 512 views of 50,000 faces
        dict(name='xent_step', op='xent', form='image', views=2, size=512, rows=50000, dim=64,
             dtype='bf16', scale=14.0, reduction='mean', train=True),
        # the validation loss map of eight 512 x 512 views
        dict(name='xent_eval', op='xent', form='image', views=8, size=512, rows=50000, dim=128,
             dtype='bf16', scale=16.0, reduction='none', train=False),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.4:
        form = rng.choice(['points', 'image', 'image', 'corners'])
        case = dict(op='embed', form=form, rows=_log_uniform(rng, 1, 200000),
                    dim=_log_uniform(rng, 1, 256), dtype=rng.choice(['f32', 'bf16', 'f16', 'f64']),
                    train=rng.random() < 0.75)
        if form == 'points':
            case['n'] = _log_uniform(rng, 1, 20000)
        elif form == 'corners':
            case['faces'] = _log_uniform(rng, 1, 200000)
        else:
            case['views'] = rng.randint(1, 8)
            case['size'] = _log_uniform(rng, 16, 1024)
            while _tokens(case) * case['dim'] * _SIZES[case['dtype']] > 1 << 29:
                case['size'] = max(16, case['size'] * 2 // 3)
        return case
    train = rng.random() < 0.7
    dtype = rng.choice(['f32', 'bf16', 'bf16', 'f16'])
    case = dict(op='xent', form=rng.choice(['points', 'image', 'image']),
                rows=_log_uniform(rng, 1, 200000), dim=_log_uniform(rng, 1, 256), dtype=dtype,
                scale=round(rng.uniform(4.0, 24.0), 3),
                reduction=rng.choice(['mean', 'sum', 'none']), train=train)
    if case['form'] == 'points':
        case['n'] = _log_uniform(rng, 1, 5000)
    else:
        case['views'] = rng.randint(1, 8)
        case['size'] = _log_uniform(rng, 16, 512)
        limit = 1.2e10 if train else 4.0e10
        while _tokens(case) * case['rows'] * max(1.0, case['dim'] / 64) > limit:
            case['size'] = max(16, case['size'] * 2 // 3)
    return case


def _tokens(case):
    if case['form'] == 'points':
        return case['n']
    if case['form'] == 'corners':
        return 3 * case['faces']
    return case['views'] * case['size'] * case['size']


def _grid(faces):
    """Bands and columns of a sphere's triangle grid with at most `faces` triangles."""
    bands = max(1, int(math.sqrt(faces / 5.0)))
    return bands, max(1, faces // (2 * bands))


def _rendered(views, size, faces, gen, dev):
    """face_idx of a sphere of `faces` triangles seen from random directions, -1 off it."""
    c = (torch.arange(size, device=dev, dtype=torch.float32) + 0.5) * (2.0 / size) - 1.0
    y, x = torch.meshgrid(-c / _RADIUS, c / _RADIUS, indexing='ij')
    z2 = 1.0 - x * x - y * y
    n = torch.stack([x, y, z2.clamp(min=0.0).sqrt()], dim=-1).reshape(1, -1, 3)
    rot, _ = torch.linalg.qr(torch.randn(views, 3, 3, generator=gen))
    n = (n.unsqueeze(2) * rot.to(dev).unsqueeze(1)).sum(-1)  # (views, pixels, 3)
    bands, cols = _grid(faces)
    v = torch.acos(n[..., 1].clamp(-1.0, 1.0)) * (bands / math.pi)
    u = (torch.atan2(n[..., 2], n[..., 0]) + math.pi) * (cols / (2 * math.pi))
    band = v.long().clamp(0, bands - 1)
    col = u.long().clamp(0, cols - 1)
    upper = ((u - col) + (v - band) > 1.0).long()
    idx = (2 * (band * cols + col) + upper).clamp(max=faces - 1)
    idx = torch.where((z2 > 0).reshape(1, -1), idx, torch.full_like(idx, -1))
    return idx.reshape(views, size, size)


def _corners(faces, rows, gen, dev):
    """(faces, 3) vertex indices of a triangle grid over `rows` vertices."""
    f = torch.arange(faces, device=dev)
    width = max(1, int(math.sqrt(rows)))
    a = (f // 2) % rows
    return torch.stack([a, (a + width + f % 2) % rows, (a + 1 + (f % 2) * (width - 1)) % rows],
                       dim=1).contiguous()


def _index(case, gen, dev):
    if case['form'] == 'points':
        return torch.randint(0, case['rows'], (case['n'],), generator=gen).to(dev)
    if case['form'] == 'corners':
        return _corners(case['faces'], case['rows'], gen, dev)
    return _rendered(case['views'], case['size'], case['rows'], gen, dev)


def prepare(case, seed):
    dev = torch.device('cuda')
    gen = torch.Generator().manual_seed(seed)
    dgen = torch.Generator(device=dev).manual_seed(seed)
    dt = _TYPES[case['dtype']]
    index = _index(case, gen, dev)
    rows, dim = case['rows'], case['dim']
    table = torch.randn(rows, dim, generator=dgen, device=dev)
    state = dict(case=case, index=index, scale=float(case.get('scale', math.sqrt(dim))))
    if case['op'] == 'embed':
        state['table'] = table.to(dt).requires_grad_(case['train'])
        if case['train']:
            state['grad'] = torch.randn(*index.shape, dim, generator=dgen, device=dev).to(dt)
        return state
    table = table / table.norm(dim=1, keepdim=True).clamp(min=1e-6)
    # a network half way through its training: towards the label's row, with noise
    noise = torch.randn(*index.shape, dim, generator=dgen, device=dev)
    x = table[index.clamp(min=0)] + noise * (0.9 / math.sqrt(dim))
    x = x / x.norm(dim=-1, keepdim=True).clamp(min=1e-6)
    state['table'] = table.to(dt).requires_grad_(case['train'])
    state['features'] = x.to(dt).requires_grad_(case['train'])
    if case['train']:
        # 16-bit floats are trained under a loss scale
        up = 1024.0 if case['dtype'] == 'f16' and case['reduction'] == 'mean' else 1.0
        if case['reduction'] == 'none':
            state['grad'] = torch.rand(index.shape, generator=dgen, device=dev) * up
        else:
            state['grad'] = torch.tensor(up, device=dev)
    return state


# ------------------------------------------------------------------------------------------------
# the calls a user makes
# ------------------------------------------------------------------------------------------------
def _own_embed(state):
    from kaolin_amd.render.mesh import surface_embedding
    out = surface_embedding(state['index'], state['table'], state['scale'])
    if not state['case']['train']:
        return out
    return out, torch.autograd.grad(out, state['table'], state['grad'])[0]


def _own_xent(state):
    from kaolin_amd.metrics.render import surface_cross_entropy
    loss = surface_cross_entropy(state['features'], state['table'], state['index'],
                                 state['scale'], state['case']['reduction'])
    if not state['case']['train']:
        return loss
    gx, ge = torch.autograd.grad(loss, [state['features'], state['table']], state['grad'])
    return loss, gx, ge


# ------------------------------------------------------------------------------------------------
# the plain forms
# ------------------------------------------------------------------------------------------------
def _wide(t):
    return t if t.dtype == torch.float64 else t.float()


def _plain_embed(state):
    index, table, scale = state['index'].reshape(-1), state['table'], state['scale']
    hit = torch.nonzero(index >= 0).squeeze(1)
    rows = index[hit]
    out = torch.zeros(index.numel(), table.shape[1], dtype=table.dtype, device=table.device)
    out[hit] = (_wide(table)[rows] * scale).to(table.dtype)
    out = out.reshape(*state['index'].shape, -1)
    if not state['case']['train']:
        return out
    g = _wide(state['grad'].reshape(index.numel(), -1)[hit])
    total = torch.zeros(table.shape, dtype=g.dtype, device=g.device).index_add_(0, rows, g)
    return out, (total * scale).to(table.dtype)


def _plain_xent(state):
    case, scale = state['case'], state['scale']
    labels = state['index'].reshape(-1)
    x_in, table = state['features'], state['table']
    hit = torch.nonzero(labels >= 0).squeeze(1)
    e = table.float()
    x = x_in.reshape(labels.numel(), -1)[hit].float()
    y = labels[hit]
    count = max(1, hit.numel())
    train, reduction = case['train'], case['reduction']
    if train:
        up = state['grad'].reshape(-1)
        up = up[hit] if reduction == 'none' else up.expand(hit.numel())
        if reduction == 'mean':
            up = up / count
        gx = torch.zeros_like(x)
        ge = torch.zeros_like(e)
    rows = torch.zeros(hit.numel(), dtype=torch.float32, device=x.device)
    piece = max(1, _PIECE // e.shape[0])
    for i in range(0, hit.numel(), piece):
        xs, ys = x[i:i + piece], y[i:i + piece, None]
        s = (xs @ e.t()) * scale
        s = s - s.max(dim=1, keepdim=True).values
        target = s.gather(1, ys)
        s = s.exp_()
        # without the label's own term, so that a probability next to 1 loses nothing
        s.scatter_(1, ys, torch.zeros_like(target))
        others = s.sum(dim=1, keepdim=True)
        rows[i:i + piece] = torch.logaddexp(others.log() - target,
                                            torch.zeros_like(target)).squeeze(1)
        if train:
            total = others + target.exp()
            p = s / total
            p.scatter_(1, ys, -others / total)
            p *= up[i:i + piece, None] * scale
            gx[i:i + piece] = p @ e
            ge += p.t() @ xs
    if reduction == 'none':
        loss = torch.zeros(labels.numel(), dtype=torch.float32, device=x.device)
        loss[hit] = rows
        loss = loss.reshape(state['index'].shape)
    else:
        loss = rows.sum(dtype=torch.float64)
        loss = (loss / count if reduction == 'mean' else loss).float()
    if not train:
        return loss
    full = torch.zeros(labels.numel(), x.shape[1], dtype=x_in.dtype, device=x.device)
    full[hit] = gx.to(x_in.dtype)
    return loss, full.reshape(x_in.shape), ge.to(table.dtype)


def run(state):
    if own:
        return _own_embed(state) if state['case']['op'] == 'embed' else _own_xent(state)
    with torch.no_grad():
        return _plain_embed(state) if state['case']['op'] == 'embed' else _plain_xent(state)


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        table = state['table'].double()
        index = state['index']
        if case['op'] == 'embed':
            padded = torch.cat([table * state['scale'], torch.zeros_like(table[:1])])
            where = torch.where(index < 0, torch.full_like(index, case['rows']), index)
            out = padded[where.reshape(-1)].reshape(*index.shape, case['dim'])
            if not case['train']:
                return out
            total = torch.zeros_like(padded)
            total.index_add_(0, where.reshape(-1),
                             state['grad'].double().reshape(-1, case['dim']))
            return out, total[:-1] * state['scale']
        flat = index.reshape(-1)
        x = state['features'].double().reshape(flat.numel(), -1)
        loss = torch.zeros(flat.numel(), dtype=torch.float64, device=x.device)
        gx, ge = torch.zeros_like(x), torch.zeros_like(table)
        kept = (flat >= 0).nonzero().reshape(-1)
        weight = torch.ones(flat.numel(), dtype=torch.float64, device=x.device)
        if case['train']:
            weight = weight * state['grad'].double().reshape(-1)
        if case['reduction'] == 'mean':
            weight = weight / max(1, kept.numel())
        scaled = table * state['scale']
        for part in kept.split(max(1, (1 << 27) // case['rows'])):
            logits = x[part] @ scaled.t()
            lse = torch.logsumexp(logits, dim=1)
            loss[part] = lse - (x[part] * scaled[flat[part]]).sum(1)
            if case['train']:
                prob = torch.exp(logits - lse[:, None])
                prob[torch.arange(part.numel(), device=x.device), flat[part]] -= 1.0
                prob = prob * weight[part, None]
                gx[part] = prob @ scaled
                ge += prob.t() @ (x[part] * state['scale'])
        if case['reduction'] == 'none':
            value = loss.reshape(index.shape)
        else:
            value = loss.sum()
            if case['reduction'] == 'mean':
                value = value / max(1, kept.numel())
        if not case['train']:
            return value
        return value, gx.reshape(*index.shape, case['dim']), ge


def work(case):
    n, rows, dim, size = _tokens(case), case['rows'], case['dim'], _SIZES[case['dtype']]
    kept = n * _COVER if case['form'] == 'image' else n
    touched = min(rows, kept) * dim * size  # the rows of the table that are looked at
    if case['op'] == 'embed':
        moved = n * 8 + touched + n * dim * size
        flops = kept * dim
        if case['train']:
            moved += kept * dim * size + rows * dim * size
            flops += kept * dim
        return {'bytes': moved, 'flops': flops}
    moved = n * 8 + kept * dim * size + rows * dim * size
    moved += 4 * n if case['reduction'] == 'none' else 4
    products = 1
    if case['train']:
        moved += n * dim * size + rows * dim * size
        moved += 4 * n if case['reduction'] == 'none' else 4
        products = 3
    return {'bytes': moved, 'flops': 2.0 * products * kept * rows * dim}
