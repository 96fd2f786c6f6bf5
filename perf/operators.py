"""Cases that measure the token scores (with their gradient) and the
orthogonalised weight update of mdlm_amd against plain torch forms.

Token scores.  A row of logits x (V columns, the mask token's column excluded)
has the log-probabilities l_v = x_v - log sum_u exp(x_u).  For a masked position
the operator returns l of the given token, the entropy -sum_v e^{l_v} l_v, the
row's log-sum-exp and the k best alternatives (by logit, ties to the lowest
index).  A position that is not masked is known: log-probability 0 for its own
token and -1e6 for any other, entropy 0, log-sum-exp 0, its own token first
among the alternatives and then the lowest other indices.  The gradient takes
d(loss)/d(log-probability), d(loss)/d(entropy) and d(loss)/d(alternatives).

Orthogonalised update.  X = G / (|G| + 1e-7), then `steps` times
X <- a X + (b A + c A^2) X with A = X X^T.  The weight update takes the momentum
of the clipped gradient, orthogonalises its Nesterov look-ahead and moves the
weights, their moving average and their bf16 copy.
"""
import math

import torch

own = False

COEFFS = (3.4445, -4.7750, 2.0315)
STEPS = 5
NORM_EPS = 1e-7
NEG = -1e6
MOMENTUM = 0.95
MAX_NORM = 1.0
GRAD_SCALE = 0.5        # two ranks' gradients, summed
EMA_OMD = 1e-4          # one minus the moving average's decay

LARGEST_LOGITS = 8192 * 50258
LARGEST_FLOPS = 5 * (3 * 4096 ** 2 * 8192 + 4096 ** 3)


def listed():
  return [
    # scoring, the smallest call: one position of one sequence is looked at
    dict(name='score one position', op='score', rows=1, masked=1, V=50258, k=8, dtype='bf16', padded=True),
    # a few positions of a 30522-token vocabulary, kept in fp32, rows not padded
    dict(name='score 37 rows fp32', op='score', rows=37, masked=37, V=30522, k=5, dtype='fp32', padded=False),
    # the first sampling step of 8 sequences of 1024: every position still masked
    dict(name='score 8 sequences', op='score', rows=8192, masked=8192, V=50258, k=8, dtype='bf16', padded=True),
    # the gradient for one 128-token sequence
    dict(name='score grad one sequence', op='score_grad', rows=128, masked=77, V=30522, k=0, dtype='bf16', padded=True),
    # fp32 logits of an unpadded odd vocabulary, the alternatives in the loss too
    dict(name='score grad fp32 odd', op='score_grad', rows=1001, masked=900, V=50257, k=4, dtype='fp32', padded=False),
    # the masked rows of a training step, already gathered: all of them masked
    dict(name='score grad batch', op='score_grad', rows=8192, masked=8192, V=50258, k=0, dtype='bf16', padded=True),
    # one square projection of a 768-wide block
    dict(name='orthogonalize 768', op='ortho', n=1, rows=768, cols=768, dtype='fp32'),
    # an odd tall pair
    dict(name='orthogonalize odd pair', op='ortho', n=2, rows=1291, cols=517, dtype='bf16'),
    # a large wide matrix
    dict(name='orthogonalize large', op='ortho', n=1, rows=4096, cols=8192, dtype='bf16'),
    # the update of the two-block 128-wide model's fused projections
    dict(name='update two small', op='update', n=2, rows=384, cols=128),
    # the update of all twelve fused projections of a 768-wide model
    dict(name='update twelve blocks', op='update', n=12, rows=2304, cols=768),
    # one wide matrix of a 1024-wide model
    dict(name='update 1024x4096', op='update', n=1, rows=1024, cols=4096),
  ]


def _log_int(rng, lo, hi):
  return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
  op = rng.choice(['score', 'score_grad', 'ortho', 'update'])
  if op in ('score', 'score_grad'):
    V = _log_int(rng, 300, 131072)
    rows = _log_int(rng, 1, max(1, min(8192, LARGEST_LOGITS // (2 * V))))
    k = rng.choice([0, rng.randint(1, 16)])
    # the -1e6 of a known position's alternatives would drown every other value
    masked = rows if k and op == 'score' else rng.randint((rows + 1) // 2, rows)
    return dict(op=op, rows=rows, masked=masked, V=V, k=k,
                dtype=rng.choice(['bf16', 'fp32']), padded=rng.random() < 0.5)
  while True:
    case = dict(op=op, n=rng.choice([1, 1, 2, 3, 5, 8, 12]), rows=_log_int(rng, 16, 6000),
                cols=_log_int(rng, 16, 6000))
    if op == 'ortho':
      case['dtype'] = rng.choice(['bf16', 'fp32'])
    if work(case)['flops'] <= LARGEST_FLOPS / 4:
      return case


def work(case):
  if case['op'] in ('score', 'score_grad'):
    rows, masked, V, k = case['rows'], case['masked'], case['V'], case['k']
    es = 2 if case['dtype'] == 'bf16' else 4
    small = rows * (16 + 12 + 12 * k)       # two token ids; three results; k alternatives
    if case['op'] == 'score':
      return dict(bytes=masked * V * es + small, flops=masked * V * 6)
    return dict(bytes=(masked + rows) * V * es + small, flops=masked * V * 8)
  n, r, c = case['n'], case['rows'], case['cols']
  s, l = min(r, c), max(r, c)
  flops = n * STEPS * (s * s * l + s * s * s + 2 * s * s * l)   # A and A^2 are symmetric: half of each
  if case['op'] == 'ortho':
    return dict(bytes=n * r * c * ((2 if case['dtype'] == 'bf16' else 4) + 2), flops=flops)
  return dict(bytes=n * r * c * (4 + 8 + 8 + 8 + 2), flops=flops)


# ------------------------------------------------------------------- inputs
def _logits(case, gen):
  rows, V = case['rows'], case['V']
  dt = torch.bfloat16 if case['dtype'] == 'bf16' else torch.float32
  ld = (V + 127) // 128 * 128 if case['padded'] else V
  buf = torch.empty(rows, ld, dtype=dt, device='cuda')
  # a frequency-shaped offset per token, noise, and a lift of the right token
  base = -1.2 * torch.log1p(torch.arange(V, device='cuda', dtype=torch.float32) / 20)
  base = base[torch.randperm(V, generator=gen, device='cuda')]
  x0 = torch.randint(0, V - 1, (rows,), generator=gen, device='cuda')
  lift = 9 * torch.rand(rows, generator=gen, device='cuda')
  for a in range(0, rows, 1024):
    b = min(rows, a + 1024)
    x = torch.randn(b - a, V, generator=gen, device='cuda') * 1.5 + base
    x[torch.arange(b - a, device='cuda'), x0[a:b]] += lift[a:b]
    buf[a:b, :V] = x.to(dt)
  if ld > V:
    buf[:, V:] = 0
  mask = V - 1
  xt = x0.clone()
  xt[torch.randperm(rows, generator=gen, device='cuda')[:case['masked']]] = mask
  return buf[:, :V], xt, x0, mask


def _matrices(n, r, c, gen):
  """Gradient-like: a decaying signal of rank min/16 plus the noise of a batch."""
  s = min(r, c)
  rk = max(1, s // 16)
  amp = 1.0 / torch.sqrt(torch.arange(1, rk + 1, device='cuda', dtype=torch.float32))
  g = torch.randn(n, r, rk, generator=gen, device='cuda') * amp @ torch.randn(n, rk, c, generator=gen, device='cuda')
  return (g + torch.randn(n, r, c, generator=gen, device='cuda')) * 1e-3


def prepare(case, seed):
  gen = torch.Generator(device='cuda').manual_seed(int(seed) * 7919 + 13)
  op = case['op']
  if op in ('score', 'score_grad'):
    logits, xt, x0, mask = _logits(case, gen)
    s = dict(op=op, logits=logits, xt=xt, x0=x0, mask=mask, k=case['k'])
    if op == 'score_grad':
      rows, k = case['rows'], case['k']
      f = _plain_scores(logits, xt, x0, mask, k)     # what the forward pass left
      s.update(lse=f['lse'], entropy=f['entropy'], top_ids=f.get('top_ids'))
      s['g_logp'] = -torch.rand(rows, generator=gen, device='cuda') / rows
      s['g_entropy'] = 0.1 * torch.randn(rows, generator=gen, device='cuda') / rows
      s['g_top'] = 0.3 * torch.randn(rows, k, generator=gen, device='cuda') / rows if k else None
    return s
  n, r, c = case['n'], case['rows'], case['cols']
  g = _matrices(n, r, c, gen)
  if op == 'ortho':
    return dict(op=op, g=g.to(torch.bfloat16 if case['dtype'] == 'bf16' else torch.float32))
  p = torch.randn(n, r, c, generator=gen, device='cuda') * 0.04
  m = 0.5 * _matrices(n, r, c, gen) + 0.3 * g
  return dict(op=op, p=p, g=g, m=m, ema=p + 1e-3 * torch.randn(n, r, c, generator=gen, device='cuda'),
              w16=p.to(torch.bfloat16), sumsq=4 * g.double().square().sum().float().reshape(1), lr=1e-4, wd=0.1)


# --------------------------------------------------------------- plain forms
def _masked_columns(x, mask):
  return torch.arange(x.shape[1], device=x.device) == mask


def _plain_scores(logits, xt, x0, mask, k):
  x = logits.float()
  rows, V = x.shape
  known = (xt != mask)
  x = torch.where(_masked_columns(x, mask), -math.inf, x)
  m = x.amax(1, keepdim=True)
  y = x - m
  e = torch.exp(y)
  z = e.sum(1, keepdim=True)
  lz = torch.log(z)
  ent = lz[:, 0] - torch.where(e > 0, e * y, 0.0).sum(1) / z[:, 0]
  lse = (m + lz)[:, 0]
  at = x0[:, None]
  logp = (y.gather(1, at) - lz)[:, 0]
  of_mask = (logits.gather(1, at).float()[:, 0] + NEG) - lse
  logp = torch.where(x0 == mask, of_mask, logp)
  out = dict(logp=torch.where(known, torch.where(x0 == xt, 0.0, NEG), logp),
             entropy=torch.where(known, 0.0, ent), lse=torch.where(known, 0.0, lse))
  if k:
    # unique 64-bit keys: the logit's order, then the lowest index
    bits = (x + 0.0).view(torch.int32).to(torch.int64)
    order = torch.where(bits < 0, -2147483649 - bits, bits)
    idx = torch.arange(V, device=x.device)
    key = order * 4294967296 + (4294967295 - idx)
    key = torch.where(known[:, None], torch.where(idx == xt[:, None], V, -idx - torch.where(idx == mask, V, 0)), key)
    ids = key.topk(k, dim=1).indices
    top = y.gather(1, ids) - lz
    out['top_logp'] = torch.where(known[:, None], torch.where(ids == xt[:, None], 0.0, NEG), top)
    out['top_ids'] = ids
  return out


def _plain_scores_grad(s):
  logits, xt, x0, mask = s['logits'], s['xt'], s['x0'], s['mask']
  l = logits.float() - s['lse'][:, None]
  l = torch.where(_masked_columns(l, mask), -math.inf, l)
  p = torch.exp(l)
  total = s['g_logp']
  if s['g_top'] is not None:
    total = total + s['g_top'].sum(1)
  bend = torch.where(p > 0, p * (l + s['entropy'][:, None]), 0.0)
  d = -total[:, None] * p - s['g_entropy'][:, None] * bend
  d = d.scatter_add(1, x0[:, None], s['g_logp'][:, None])
  if s['g_top'] is not None:
    d = d.scatter_add(1, s['top_ids'], s['g_top'])
  d = torch.where((xt != mask)[:, None] | _masked_columns(l, mask), 0.0, d)
  return d.to(logits.dtype)


def _plain_ortho(g):
  a, b, c = COEFFS
  x = g.float()
  tall = x.shape[-2] > x.shape[-1]
  if tall:
    x = x.transpose(-1, -2).contiguous()
  norm = x.double().square().sum((-2, -1), keepdim=True).sqrt()
  x = x / (norm + NORM_EPS).float()
  for _ in range(STEPS):
    gram = x @ x.transpose(-1, -2).contiguous()
    x = a * x + (b * gram + c * (gram @ gram)) @ x
  return x.transpose(-1, -2) if tall else x


def _plain_update(s):
  g, m, p = s['g'], s['m'], s['p']
  total = torch.sqrt(s['sumsq']) * GRAD_SCALE
  coef = GRAD_SCALE * torch.clamp(MAX_NORM / (total + 1e-6), max=1.0)
  g = g * coef
  m += (g - m) * (1 - MOMENTUM)
  o = _plain_ortho(g + MOMENTUM * (m - g))
  scale = 0.2 * math.sqrt(max(p.shape[-2:]))
  p.mul_(1 - s['lr'] * s['wd']).sub_(o * (s['lr'] * scale))
  s['ema'] -= EMA_OMD * (s['ema'] - p)
  s['w16'].copy_(p)
  return dict(p=p, m=m, ema=s['ema'], w16=s['w16'])


# ---------------------------------------------------------------------- run
def run(s):
  if own:
    from mdlm_amd import ops
    if s['op'] == 'score':
      t = ops.subs_scores(s['logits'], s['xt'], s['x0'], s['mask'], top_k=s['k'])
      out = dict(logp=t.logp, entropy=t.entropy, lse=t.lse)
      if s['k']:
        out.update(top_logp=t.top_logp, top_ids=t.top_ids)
      return out
    if s['op'] == 'score_grad':
      return dict(dlogits=ops.subs_scores_bwd(s['logits'], s['xt'], s['x0'], s['mask'], s['lse'], s['entropy'],
                                              g_logp=s['g_logp'], g_entropy=s['g_entropy'],
                                              top_ids=s['top_ids'], g_top=s['g_top']))
    if s['op'] == 'ortho':
      return dict(o=ops.orthogonalize(s['g'], steps=STEPS))
    ops.muon_update(s['p'], s['g'], s['m'], s['lr'], ema=s['ema'], w16=s['w16'], momentum=MOMENTUM,
                    weight_decay=s['wd'], steps=STEPS, sumsq=s['sumsq'], max_norm=MAX_NORM,
                    grad_scale=GRAD_SCALE, ema_one_minus_decay=EMA_OMD)
    return dict(p=s['p'], m=s['m'], ema=s['ema'], w16=s['w16'])
  if s['op'] == 'score':
    return _plain_scores(s['logits'], s['xt'], s['x0'], s['mask'], s['k'])
  if s['op'] == 'score_grad':
    return dict(dlogits=_plain_scores_grad(s))
  if s['op'] == 'ortho':
    return dict(o=_plain_ortho(s['g']).to(torch.bfloat16))
  return _plain_update(s)


# -------------------------------------------------------------- in 64 bits
def _exact_table(logits, mask):
  x = logits.to(torch.float64)
  x[:, mask] = -math.inf
  return torch.log_softmax(x, dim=1)


def _exact_ortho(g):
  a, b, c = COEFFS
  x = g.to(torch.float64)
  x = x / (torch.linalg.matrix_norm(x, keepdim=True) + NORM_EPS)
  wide = x.shape[-2] <= x.shape[-1]
  for _ in range(STEPS):
    xt = x.transpose(-1, -2).contiguous()
    q = torch.matmul(x, xt) if wide else torch.matmul(xt, x)
    y = b * q + c * torch.matmul(q, q)
    x = a * x + (torch.matmul(y, x) if wide else torch.matmul(x, y))
  return x


def exact(case, seed):
  s = prepare(case, seed)
  if case['op'] in ('score', 'score_grad'):
    mask, masked, k = s['mask'], s['xt'] == s['mask'], case['k']
    parts = []
    for a in range(0, case['rows'], 1024):        # by rows: the table is held in 64 bits
      sl = slice(a, a + 1024)
      t = _exact_table(s['logits'][sl], mask)
      p = t.exp()
      h = torch.special.entr(p).sum(1)
      here = masked[sl]
      if case['op'] == 'score':
        got = dict(logp=t.gather(1, s['x0'][sl, None])[:, 0] * here, entropy=h * here,
                   lse=torch.where(here, s['logits'][sl, 0].double() - t[:, 0], 0.0))
        if k:
          best = torch.sort(t, dim=1, descending=True).values[:, :k]
          rest = torch.cat([torch.zeros(1), torch.full((k - 1,), NEG)]).to(t)
          got['top_logp'] = torch.where(here[:, None], best, rest)
      else:
        gl, gh = s['g_logp'][sl].double(), s['g_entropy'][sl].double()
        up = torch.zeros_like(t)
        up.scatter_(1, s['x0'][sl, None], gl[:, None])
        if k:
          up.scatter_add_(1, s['top_ids'][sl], s['g_top'][sl].double())
        lp = torch.where(p > 0, t, 0.0)
        d = up - p * up.sum(1, keepdim=True) - gh[:, None] * (p * lp + p * h[:, None])
        got = dict(dlogits=d * here[:, None])
      parts.append(got)
    out = {n: torch.cat([q[n] for q in parts]) for n in parts[0]}
    if k and case['op'] == 'score':
      out['top_ids'] = None
    return out
  if case['op'] == 'ortho':
    return dict(o=_exact_ortho(s['g']))
  total = s['sumsq'].double().sqrt() * GRAD_SCALE
  g = s['g'].double() * (GRAD_SCALE * (MAX_NORM / (total + 1e-6)).clamp(max=1.0))
  m = MOMENTUM * s['m'].double() + (1 - MOMENTUM) * g
  o = _exact_ortho((1 - MOMENTUM) * g + MOMENTUM * m)
  p = s['p'].double() * (1 - s['lr'] * s['wd']) - s['lr'] * 0.2 * math.sqrt(max(case['rows'], case['cols'])) * o
  ema = (1 - EMA_OMD) * s['ema'].double() + EMA_OMD * p
  return dict(p=p, m=m, ema=ema, w16=p)
