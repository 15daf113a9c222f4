"""Products in 8-bit integers in 64 bits: the definition the int8 operators are held to."""
import torch


def quantize_rows(x):
    """(q, scale) of rows in float64; q holds whole numbers. A row with an infinity or a NaN: zeros and NaN."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)          # NaN if the row has one
    fine = torch.isfinite(top)
    q = torch.where(fine & (top > 0), torch.round(127 * torch.where(fine, x, 0.0) / torch.where(top > 0, top, 1.0)), 0.0)
    return q, torch.where(fine, top / 127, float("nan"))[..., 0]


def linear(x, values, scales):
    q, scale = quantize_rows(x)
    return (q @ values.double().T) * scale[:, None] * scales.double()


def swiglu(gate, up):
    return gate * torch.sigmoid(gate) * up


def layer(x, gate_up, gate_up_scale, down, down_scale, ids, weights):
    """Routes one expert at a time; ids outside [0, E) contribute nothing."""
    q, scale = quantize_rows(x)
    out = torch.zeros(x.shape[0], down.shape[1], dtype=torch.float64)
    inter = down.shape[2]
    for e in range(gate_up.shape[0]):
        token, slot = torch.where(ids == e)
        if token.numel() == 0:
            continue
        both = (q[token] @ gate_up[e].double().T) * scale[token, None] * gate_up_scale[e].double()
        a, a_scale = quantize_rows(swiglu(both[:, :inter], both[:, inter:]))
        y = (a @ down[e].double().T) * a_scale[:, None] * down_scale[e].double()
        out.index_add_(0, token, weights[token, slot].double()[:, None] * y)
    return out
