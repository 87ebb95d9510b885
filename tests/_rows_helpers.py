"""Helpers of the tests of row operators: rounding-error bounds, inputs."""

import torch

ROW_DTYPES = [torch.float16, torch.bfloat16, torch.float32, torch.float64]
ROW_IDS = ["f16", "bf16", "f32", "f64"]
# unit roundoff of a type, and half of its smallest subnormal
UNIT = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24, torch.float64: 2.0**-53}
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134, torch.float32: 2.0**-150, torch.float64: 0.0}


def assert_sum(got, want, magnitude, terms, arithmetic=None):
    """got = a sum of `terms` products, each product and each addition rounded in
    32 bits (64 for float64), then rounded once to got's type: within
    (terms + 2) u * sum |product| of the 64-bit sum `want`, plus the last
    rounding of a value that is off by as much.  `arithmetic` names the sums'
    type where the result's does not.  The float64 oracle errs as much itself."""
    wide = torch.float64 if got.dtype == torch.float64 or arithmetic == torch.float64 else torch.float32
    sums = (terms + 2) * UNIT[wide] * (2 if wide == torch.float64 else 1) * magnitude.double().cpu()
    last = UNIT[got.dtype] if got.dtype != wide else 0.0
    want = want.double().cpu()
    bound = sums + last * (want.abs() + sums) + TINY[got.dtype] + 1e-300
    diff = (got.double().cpu() - want).abs()
    worst = (diff / bound).max().item() if diff.numel() else 0.0
    assert bool((diff <= bound).all()), f"{worst} times the bound"


def randn(shape, dtype, seed, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g, dtype=torch.float64).to(dtype).to(device)


def route_oracle(experts, num_experts):
    """(order, inverse, offsets) on the CPU, by the definition."""
    flat = experts.reshape(-1).cpu().tolist()
    key = [e if 0 <= e < num_experts else num_experts for e in flat]
    order = sorted(range(len(key)), key=lambda i: (key[i], i))
    inverse = [0] * len(key)
    for place, i in enumerate(order):
        inverse[i] = place
    offsets = [sum(k < e for k in key) for e in range(num_experts + 1)] if len(key) < 4096 else None
    if offsets is None:
        counts = [0] * (num_experts + 1)
        for k in key:
            counts[k] += 1
        offsets = [0]
        for e in range(num_experts):
            offsets.append(offsets[-1] + counts[e])
    return (torch.tensor(order, dtype=torch.int32), torch.tensor(inverse, dtype=torch.int32).reshape(experts.shape),
            torch.tensor(offsets, dtype=torch.int32))


def random_experts(n_tokens, slots, num_experts, seed, dropped=0.0, dtype=torch.int32):
    g = torch.Generator().manual_seed(seed)
    experts = torch.randint(0, num_experts, (n_tokens, slots), generator=g)
    if dropped:
        u = torch.rand((n_tokens, slots), generator=g)
        experts = torch.where(u < dropped, torch.where(u < dropped / 2, -1, num_experts + 3), experts)
    return experts.to(dtype).cuda()
