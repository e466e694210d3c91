"""64-bit references of the 4-bit cache and its attention (CPU, torch)."""
import numpy as np
import torch


def quantize(x):
    """Values that a cached fp16 tensor [..., D] stands for, in 64 bits, from the definition, block by block."""
    a = x.numpy().astype(np.float64).reshape(-1, 32)
    out = np.empty_like(a)
    for i, b in enumerate(a):
        if not np.isfinite(b).all():
            out[i] = np.nan
            continue
        m = b[np.argmax(np.abs(b))]                # the first of equals
        d = np.float64(np.float16(m / -8))
        out[i] = 0.0 if d == 0 else (np.clip(np.floor(b / d + 8.5), 0, 15) - 8) * d
    return torch.from_numpy(out.reshape(x.shape))


def attention(q, k, v, scale, see):
    """One head: q [n][D], k and v [t][D] (64 bits), see [n][t].  Returns o, the same sum over |v|, and the log of the
    softmax's sum; rows that see nothing: zeros and -inf."""
    s = (q.double() @ torch.nan_to_num(k).t() * scale).masked_fill(~see, float("-inf"))
    lse = torch.logsumexp(s, -1)
    p = torch.where(see, torch.exp(s - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)[:, None]), torch.zeros_like(s))
    v = torch.nan_to_num(v)
    return p @ v, p @ v.abs(), lse
