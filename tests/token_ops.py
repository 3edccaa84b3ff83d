"""What the tests of group norm, rotary positions and attention share: calls of
the C ABI on torch tensors, and plain implementations in 64 bits."""
import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def types(L):
    return {torch.float32: L.IE_DT_F32, torch.bfloat16: L.IE_DT_BF16, torch.float16: L.IE_DT_F16}


def stream():
    return torch.cuda.current_stream().cuda_stream


def ptr(t):
    return None if t is None else t.data_ptr()


def split(x, c_store):
    """fp32 [..., c] -> bf16 [..., 2 * c_store], hi plane then lo plane."""
    c = x.shape[-1]
    y = torch.zeros(*x.shape[:-1], 2 * c_store, dtype=torch.bfloat16, device=x.device)
    y[..., :c] = x
    y[..., c_store:c_store + c] = x - y[..., :c].float()
    return y


def joined(y, c, c_store):
    return y[..., :c].double() + y[..., c_store:c_store + c].double()


# ------------------------------------------------------------ group norm

def group_norm_desc(L, x_shape, c, groups, eps, act, x_type, y_type):
    n, h, w, c_store = x_shape
    return L.GroupNormDesc(n=n, c=c, h=h, w=w, c_store=c_store, groups=groups, eps=eps,
                           act=act, x_type=x_type, y_type=y_type)


def run_group_norm(L, d, x, gamma, beta, y):
    need = int(L.lib.ie_cuda_group_norm_workspace_bytes(d))
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device=x.device)
    L.check(L.lib.ie_cuda_group_norm_nhwc(d, x.data_ptr(), ptr(gamma), ptr(beta), y.data_ptr(),
                                          ws.data_ptr(), need, stream()))
    return ws


def group_norm_64(x, groups, gamma, beta, eps, act):
    """x [n, h, w, c] in 64 bits -> (y, bound on |y|'s fp32 arithmetic scale)."""
    n, h, w, c = x.shape
    v = x.reshape(n, h * w, groups, c // groups)
    mean = v.mean(dim=(1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(((v - mean) ** 2).mean(dim=(1, 3), keepdim=True) + eps)
    g = gamma.double() if gamma is not None else torch.ones(c, dtype=torch.float64, device=x.device)
    b = beta.double() if beta is not None else torch.zeros(c, dtype=torch.float64, device=x.device)
    z = ((v - mean) * rstd).reshape(x.shape) * g + b
    size = ((v.abs() + v.abs().mean(dim=(1, 3), keepdim=True)) * rstd).reshape(x.shape) * g.abs() \
        + b.abs()
    if act == 1:
        y = z.clamp(min=0)
    elif act == 2:
        y = z.clamp(0, 6)
    elif act == 3:
        y = z * torch.sigmoid(z)
    elif act == 4:
        y = 0.5 * z * torch.erfc(-z / math.sqrt(2))
    else:
        y = z
    return y, size


# ---------------------------------------------------------------- rotary

def rotary_desc(L, x, y, rot_heads, section, layout, freq, positions, theta=10000.0, inverse=0,
                tokens=None):
    t = types(L)
    d = L.RotaryDesc(tokens=x.shape[0] if tokens is None else tokens,
                     x_token_stride=x.stride(0), x_head_stride=x.stride(1),
                     y_token_stride=y.stride(0), y_head_stride=y.stride(1),
                     pos_axis_stride=positions.stride(0), theta=theta, heads=x.shape[1],
                     rot_heads=rot_heads, head_dim=x.shape[2], axes=len(section), layout=layout,
                     freq=freq, inverse=inverse, x_type=t[x.dtype], y_type=t[y.dtype],
                     pos_bits=64 if positions.dtype == torch.int64 else 32)
    for i, s in enumerate(section):
        d.section[i] = s
    return d


def run_rotary(L, d, x, positions, y):
    plan = L.RotaryPlan()
    L.check(L.lib.ie_rotary_plan_init(d, plan))
    L.check(L.lib.ie_cuda_rotary(d, plan, x.data_ptr(), positions.data_ptr(), y.data_ptr(),
                                 stream()))


def rotary_pairs(section, layout, freq, theta):
    """Per pair: (axis, frequency, first element, second element)."""
    pairs, out, begin = sum(section), [], 0
    for a, size in enumerate(section):
        for j in range(size):
            i = begin + j
            f = theta ** (-i / pairs) if freq == 0 else theta ** (-j / size)
            uv = ((2 * i, 2 * i + 1), (i, i + pairs), (2 * begin + j, 2 * begin + size + j))[layout]
            out.append((a, f, *uv))
        begin += size
    return out


def rotary_64(x, positions, rot_heads, section, layout, freq, theta=10000.0, inverse=0):
    """-> (y, |u| + |v| of each rotated element: the scale of its arithmetic)."""
    y = x.double().clone()
    size = y.abs()
    for a, f, u, v in rotary_pairs(section, layout, freq, theta):
        t = positions[a].double() * f * (-1 if inverse else 1)
        c, s = torch.cos(t)[:, None], torch.sin(t)[:, None]
        xu, xv = x[:, :rot_heads, u].double(), x[:, :rot_heads, v].double()
        y[:, :rot_heads, u], y[:, :rot_heads, v] = xu * c - xv * s, xu * s + xv * c
        size[:, :rot_heads, u] = size[:, :rot_heads, v] = xu.abs() + xv.abs()
    return y, size


# ------------------------------------------------------------- attention

def attention_desc(L, q, k, v, o, scale, softcap=0.0, o_type=None):
    t = types(L)
    d = L.AttentionDesc(batch=q.shape[0], q_len=q.shape[1], kv_len=k.shape[1],
                        q_heads=q.shape[2], kv_heads=k.shape[2], head_dim=q.shape[3],
                        type=t[q.dtype], o_type=t[o.dtype] if o_type is None else o_type,
                        scale=scale, softcap=softcap)
    for i in range(3):
        d.q_stride[i], d.k_stride[i] = q.stride(i), k.stride(i)
        d.v_stride[i], d.o_stride[i] = v.stride(i), o.stride(i)
    return d


def attention_mask(L, causal=0, documents=0, kv_lens=None, prefix=None, q_offsets=None,
                   kv_offsets=None, slopes=None):
    return L.AttentionMask(causal=causal, documents=documents, kv_lens=ptr(kv_lens),
                           prefix_lens=ptr(prefix), q_offsets=ptr(q_offsets),
                           kv_offsets=ptr(kv_offsets), slopes=ptr(slopes))


def run_attention(L, d, m, q, k, v, o, lse=None, workspace=None):
    need = int(L.lib.ie_cuda_attention_workspace_bytes(d, m))
    ws = workspace
    if ws is None:
        ws = torch.empty(max(need, 1), dtype=torch.uint8, device=q.device)
    L.check(L.lib.ie_cuda_attention(d, m, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                                    ptr(lse), ws.data_ptr(), ws.numel(), stream()))
    return ws


def attention_64(q, k, v, scale, softcap=0.0, causal=0, kv_lens=None, prefix=None, q_offsets=None,
                 kv_offsets=None, slopes=None):
    """Sequence by sequence in 64 bits -> (o, lse, sum of p |v|, rows written)."""
    b, sq, hq, d = q.shape
    sk, hk = k.shape[1], k.shape[2]
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(o)
    lse = torch.full((b, hq, sq), -math.inf, dtype=torch.float64, device=q.device)
    rows = torch.zeros(b, sq, dtype=torch.bool, device=q.device)
    if q_offsets is not None:
        qo, ko = q_offsets.tolist(), kv_offsets.tolist()
        seqs = [(0, qo[r], qo[r + 1], ko[r], ko[r + 1], r) for r in range(len(qo) - 1)]
    else:
        seqs = [(r, 0, sq, 0, sk if kv_lens is None else int(kv_lens[r]), r) for r in range(b)]
    for n, q0, q1, k0, k1, r in seqs:
        rows[n, q0:q1] = True
        if q1 == q0 or k1 == k0:
            continue
        i = torch.arange(q1 - q0, device=q.device)[:, None] + (k1 - k0) - (q1 - q0)
        j = torch.arange(k1 - k0, device=q.device)[None]
        sees = torch.ones(q1 - q0, k1 - k0, dtype=torch.bool, device=q.device)
        if causal:
            sees = (j <= i) | (j < (int(prefix[r]) if prefix is not None else 0))
        kk, vv = (t[n, k0:k1].double().repeat_interleave(hq // hk, 1) for t in (k, v))
        x = torch.einsum("ihd,jhd->hij", q[n, q0:q1].double(), kk) * scale
        if softcap:
            x = softcap * torch.tanh(x / softcap)
        if slopes is not None:
            x = x - slopes.double()[:, None, None] * (i - j).abs()
        x = torch.where(sees, x, -math.inf)
        l = torch.logsumexp(x, -1)
        p = torch.exp(x - torch.where(torch.isinf(l), 0.0, l)[..., None])
        lse[n, :, q0:q1] = l
        o[n, q0:q1] = torch.einsum("hij,jhd->ihd", p, vv)
        size[n, q0:q1] = torch.einsum("hij,jhd->ihd", p, vv.abs())
    return o, lse, size, rows


def check_attention(o, lse, want, dtype, extra=0.0):
    """Tolerances.  With p = exp(s - max) rounded to the 16-bit type, each
    weight is off by at most half a step, so o by half_step * sum p |v|, and
    its own rounding is half_step * |o|.  Scores are sums of at most 128 fp32
    products and pass an fp32 exp (and tanh): off by less than 2^-13 here
    (|s| < 64, 2^-18 of that for the sums, 2^-19 * cap for the tanh), which
    moves every weight, and the sum of weights, by that much."""
    wo, wl, size, rows = want
    half = HALF_STEP[dtype]
    err = (o.double() - wo).abs()
    tol = half * (wo.abs() + size) + 2.0 ** -12 * size + 2.0 ** -24 + extra
    bad = (err > tol) & rows[:, :, None, None]
    assert not bad.any(), (float((err / tol)[rows].max()), bad.nonzero()[:4].tolist())
    if lse is not None:
        r = rows[:, None, :].expand_as(wl)
        a, b = lse.double()[r], wl[r]
        assert torch.equal(torch.isinf(a), torch.isinf(b)) and not torch.isnan(a).any()
        f = ~torch.isinf(b)
        if f.any():
            # beyond |s| = 64 the fp32 result itself has steps of 2^-23 * |lse|, and
            # the score's sum, its scaling and the logarithm's sum a few of them
            # (at 6394 half a step is 2^-12 already): 8 half steps
            assert not ((a[f] - b[f]).abs() > 2.0 ** -12 + 2.0 ** -21 * b[f].abs()).any()
