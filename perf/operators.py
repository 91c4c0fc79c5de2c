"""What the dense operators of a training step are measured on: the layer transform `spmm_cpp.linear` (a matrix product with
bias, activation and residual in its epilogue, and its gradients) and the optimiser `spmm_cpp.AdamW` (one pass over all
parameters, moments in 32 or 8 bits).

Where `own` is false, `run` computes the same from elementary torch operations in 32 bits, rounded once at the end."""
import math
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
BLOCK = 256                      # elements that share a scale where moments are held in 8 bits
TOP = 448.0                      # largest e4m3 value
LEAST = 2.0 ** -9                # smallest e4m3 value above zero
FLOOR = 2.0 ** -100              # a block's scale never goes below the one that this largest value would give
LR, BETA1, BETA2, EPS, DECAY = 0.01, 0.9, 0.999, 1e-8, 0.01


# ------------------------------------------------------------------------------------------------ the cases
def _linear(name, m, k, n, dtype, act, bias, residual, train, padded=False):
    """No 32-bit training case has relu: where x W + b is within rounding of zero its slope is 0 or 1 by the order of a sum, and
    one such value among ten million moves a gradient's norm by more than 32-bit outputs may differ. Forward it is continuous."""
    return dict(name=name, op="linear", m=m, k=k, n=n, dtype=dtype, act=act, bias=bias, residual=residual, train=train, padded=padded)


def _adamw(name, tensors, least, most, dtype, bits, master, step, salt=0):
    return dict(name=name, op="adamw", tensors=tensors, least=least, most=most, dtype=dtype, bits=bits, master=master, step=step, salt=salt)


def listed():
    return [
        # one node's features through the first layer of the Reddit model: what a served request costs
        _linear("one_row_f32", 1, 602, 256, "f32", "relu", True, False, False),
        # a few requests at once through a wide layer: the weights' bytes are all there is
        _linear("few_rows_bf16", 6, 4096, 4096, "bf16", "silu", True, True, False),
        # first layer of the Reddit model, all nodes, the input features at the aggregation's row pitch
        _linear("reddit_first_f32", 232965, 602, 256, "f32", "relu", True, False, False, padded=True),
        # a hidden layer over every node of the products graph with a skip connection, 16 bits
        _linear("products_hidden_bf16", 2449029, 256, 256, "bf16", "relu", True, True, False),
        # a hidden layer of the Reddit model in training, with a skip connection: output and all gradients
        _linear("reddit_hidden_f32_train", 232965, 256, 256, "f32", "gelu", True, True, True),
        # its last layer, 41 classes: a narrow, odd product, half precision
        _linear("reddit_classes_f16_train", 232965, 256, 41, "f16", "none", True, False, True),
        # the expanding half of a perceptron block over some thousand tokens
        _linear("mlp_bf16_train", 8192, 1024, 4096, "bf16", "gelu", True, False, True),
        # the Cora model's first layer: 1433 features, 16 hidden, few nodes
        _linear("cora_first_f32_train", 2708, 1433, 16, "f32", "silu", False, False, True),
        # the Reddit model's own weights and biases: a handful of small tensors, where the calls count
        _adamw("gcn_weights_f32", 6, 41, 602 * 256, "f32", 32, False, 10),
        # a deep model's many tensors, from a bias of some dozen elements to matrices of a million, 8-bit moments
        _adamw("many_bf16_8bit", 180, 64, 1 << 20, "bf16", 8, False, 1000),
        # learned node embeddings of the products graph (2449029 x 100), moments in 32 bits
        _adamw("embedding_f32", 1, 244902900, 244902900, "f32", 32, False, 100),
        # the same with 128 features in 16 bits, a 32-bit master copy and 8-bit moments
        _adamw("embedding_bf16_8bit_master", 1, 313475712, 313475712, "bf16", 8, True, 100),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """Another case of these ranges: rows from 1 to 2449029, widths from 1 to 4096; 1 to 180 tensors of 1 to 313475712 elements."""
    if rng.random() < 0.65:
        train = rng.random() < 0.5
        dtype = rng.choice(("f32", "bf16", "f16"))
        k, n = _log(rng, 1, 4096), _log(rng, 1, 4096)
        # at most the largest listed case's products (a third of them with the two of the gradients) and values
        most = min(2449029, 2449029 * 65536 // (k * n * (3 if train else 1)), 2449029 * 768 // ((k + 2 * n) * (4 if train else 2)))
        m = max(1, _log(rng, 1, max(1, most)))
        acts = ("none", "gelu", "silu") if train and dtype == "f32" else ("none", "relu", "gelu", "silu")
        return dict(op="linear", m=m, k=k, n=n, dtype=dtype, act=rng.choice(acts),
                    bias=rng.random() < 0.7, residual=rng.random() < 0.4, train=train, padded=rng.random() < 0.3)
    tensors = _log(rng, 1, 180)
    most = min(244902900, 244902900 // tensors)
    least = _log(rng, 1, most)
    dtype, bits = rng.choice(("f32", "bf16", "f16")), rng.choice((8, 32))
    return dict(op="adamw", tensors=tensors, least=least, most=_log(rng, least, most), dtype=dtype, bits=bits,
                master=dtype != "f32" and rng.random() < 0.5, step=_log(rng, 1, 100000), salt=rng.randrange(1 << 20))


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _linear_inputs(case, seed):
    """Features as a layer meets them: half of them zero behind the last activation, the rest positive; weights that keep the
    rows' scale; gradients around zero. A padded x is a view of rows that are a multiple of 32 wide, as aggregation leaves them."""
    gen, dtype = _generator(seed), DTYPES[case["dtype"]]
    m, k, n = case["m"], case["k"], case["n"]
    pitch = -(-k // 32) * 32 if case["padded"] else k
    x = torch.zeros(m, pitch, dtype=dtype, device="cuda")[:, :k]
    x.copy_(_normal(gen, m, k).relu_())
    s = {"case": case, "x": x, "dy": None, "bias": None, "residual": None}
    s["weight"] = (_normal(gen, k, n) / math.sqrt(k)).to(dtype)
    if case["bias"]:
        s["bias"] = (0.1 * _normal(gen, n)).to(dtype)
    if case["residual"]:
        s["residual"] = _normal(gen, m, n).relu_().to(dtype)
    if case["train"]:
        s["dy"] = (0.05 * _normal(gen, m, n)).to(dtype)
        for name in ("x", "weight", "bias", "residual"):
            if s[name] is not None:
                s[name].requires_grad_(True)
    return s


def _sizes(case):
    """Elements of each tensor: spread over the logarithm from the least to the most."""
    low, high, count = math.log(case["least"]), math.log(case["most"]), case["tensors"]
    at = torch.rand(count, generator=torch.Generator().manual_seed(case["salt"]), dtype=torch.float64)
    sizes = torch.exp(low + (high - low) * at).round().long().clamp(case["least"], case["most"])
    sizes[0], sizes[-1] = case["least"], case["most"]
    return sizes.tolist()


def _adamw_inputs(case, seed):
    """Parameters, gradients and moments in the middle of a training run. Parameters and gradients are views of one flat buffer
    each, as bucketed data-parallel training keeps them; a tensor starts at a multiple of 256 elements, gaps are zero."""
    gen, dtype = _generator(seed), DTYPES[case["dtype"]]
    sizes = _sizes(case)
    starts, total = [], 0
    for n in sizes:
        starts.append(total)
        total += -(-n // BLOCK) * BLOCK
    inside = torch.zeros(total, dtype=torch.bool, device="cuda")
    place = torch.zeros(total, dtype=torch.int32, device="cuda")                      # each element's index in its tensor
    for at, n in zip(starts, sizes):
        inside[at:at + n] = True
        if case["bits"] == 8:
            place[at:at + n] = torch.arange(n, dtype=torch.int32, device="cuda")
    wide = torch.exp(2.0 * _normal(gen, total // BLOCK)).repeat_interleave(BLOCK)     # gradients differ in size over the model
    grad = (1e-3 * wide * _normal(gen, total)).mul_(inside).to(dtype)
    m = (3e-4 * wide * _normal(gen, total)).mul_(inside)
    v = (1e-3 * wide * (0.2 + _normal(gen, total).abs_())).square_().mul_(inside)
    del wide
    w = (0.05 * _normal(gen, total)).mul_(inside)
    s = {"case": case, "sizes": sizes, "starts": starts, "param": w.to(dtype), "grad": grad, "place": place, "master": w if case["master"] else None}
    if case["bits"] == 32:
        s.update(exp_avg=m, exp_avg_sq=v)
    else:
        s["exp_avg"], s["exp_avg_scale"] = _to_codes(m, False)
        s["exp_avg_rms"], s["exp_avg_rms_scale"] = _to_codes(v.sqrt_(), True)
    return s


STATE = {32: ("exp_avg", "exp_avg_sq"), 8: ("exp_avg", "exp_avg_scale", "exp_avg_rms", "exp_avg_rms_scale")}


def _state_dict(s):
    """The optimiser's state_dict() for these moments."""
    case, states = s["case"], {}
    for i, (at, n) in enumerate(zip(s["starts"], s["sizes"])):
        one = {"step": case["step"]}
        for name in STATE[case["bits"]] + (("master",) if case["master"] else ()):
            one[name] = s[name][at // BLOCK:-(-(at + n) // BLOCK)] if name.endswith("_scale") else s[name][at:at + n]
        states[i] = one
    return states


def prepare(case, seed):
    if case["op"] == "linear":
        return _linear_inputs(case, seed)
    s = _adamw_inputs(case, seed)
    if own:                      # the optimiser that a training program makes once and keeps
        spmm_cpp = _package()
        params = [torch.nn.Parameter(s["param"][at:at + n]) for at, n in zip(s["starts"], s["sizes"])]
        for p, at, n in zip(params, s["starts"], s["sizes"]):
            p.grad = s["grad"][at:at + n]
        opt = spmm_cpp.AdamW(params, lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, state_bits=case["bits"],
                             master_weights=case["master"])
        given = opt.state_dict()
        opt.load_state_dict({"state": _state_dict(s), "param_groups": given["param_groups"]})
        for name, t in opt.state_buffers().items():
            t.copy_(s[name])     # what lies between the tensors too: it comes back with the buffers
        for name in STATE[case["bits"]] + ("master", "place"):
            s[name] = None       # the optimiser has its own now
        s["opt"], s["params"] = opt, params
    return s


# ------------------------------------------------------------------------------------------------ one pass
def _gelu(t):
    return 0.5 * t * (1.0 + torch.erf(t * math.sqrt(0.5)))


def _gelu_slope(t):
    return 0.5 * (1.0 + torch.erf(t * math.sqrt(0.5))) + t * torch.exp(-0.5 * t * t) * (1.0 / math.sqrt(2.0 * math.pi))


def _silu_slope(t):
    g = torch.sigmoid(t)
    return g * (1.0 + t * (1.0 - g))


ACT = {"none": lambda t: t, "relu": lambda t: torch.where(t <= 0, torch.zeros_like(t), t), "gelu": _gelu, "silu": lambda t: t * torch.sigmoid(t)}
SLOPE = {"relu": lambda t: (~(t <= 0)).to(t.dtype), "gelu": _gelu_slope, "silu": _silu_slope}


def _linear_plain(s, wide=torch.float32):
    """y = act(x W + b) + r, and with a gradient G of y: P = G act'(x W + b), dx = P W^T, dW = x^T P, db = sum of P's rows, dr = G."""
    case = s["case"]
    x, w = s["x"].to(wide), s["weight"].to(wide)
    pre = torch.mm(x, w)
    if s["bias"] is not None:
        pre = pre + s["bias"].to(wide)
    y = ACT[case["act"]](pre)
    if s["residual"] is not None:
        y = y + s["residual"].to(wide)
    got = {"y": y}
    if case["train"]:
        p = s["dy"].to(wide)
        if case["act"] != "none":
            p = p * SLOPE[case["act"]](pre)
        got["dx"], got["dw"] = torch.mm(p, w.t()), torch.mm(x.t(), p)
        if s["bias"] is not None:
            got["db"] = p.sum(0)
        if s["residual"] is not None:
            got["dr"] = s["dy"].to(wide)
    return got


def _package():
    if "dist-gnn_amd" not in sys.path:
        sys.path.insert(0, "dist-gnn_amd")
    import spmm_cpp
    return spmm_cpp


def _linear_own(s):
    spmm_cpp = _package()
    case = s["case"]
    y = spmm_cpp.linear(s["x"], s["weight"], s["bias"], activation=case["act"], residual=s["residual"])
    got = {"y": y}
    if case["train"]:
        names = [n for n in ("x", "weight", "bias", "residual") if s[n] is not None]
        grads = torch.autograd.grad(y, [s[n] for n in names], s["dy"])
        got.update(zip([{"x": "dx", "weight": "dw", "bias": "db", "residual": "dr"}[n] for n in names], grads))
    return got


def _dither(place, step, along, ahead):
    """Where in its gap a value is rounded up: the fraction, in 16 bits, of (place x along + step x ahead) / 2^32, both odd parts
    of irrational numbers. Over the steps it fills [0, 1) evenly, so what a slow average loses to one rounding the next returns."""
    ahead = (step * ahead + (1 << 31)) % (1 << 32) - (1 << 31)
    return (place * along).add_(ahead).bitwise_right_shift_(16).bitwise_and_(0xFFFF).float().mul_(2.0 ** -16)


M_ALONG, M_AHEAD, R_ALONG, R_AHEAD = 0x6A09E667, 0x9E3779B9, 0x3C6EF372, 0xBB67AE85


def _to_codes(t, root, up=0.5):
    """Moments in 8 bits: each block of 256 values times 448 over its largest, in e4m3 (steps of 2^(e-3), 2^-9 at least), up
    where the part behind the step and `up` reach 1; a root above zero keeps at least the smallest code, so that no denominator
    vanishes. Returns the codes and the blocks' scales (code x scale = value)."""
    t = t.view(-1, BLOCK)
    top = t.abs().amax(1, keepdim=True).clamp_min(FLOOR)
    code = t * torch.div(torch.full_like(top, TOP), top)
    step = (code.view(torch.int32) & 0x7F800000).clamp_min_(121 << 23).sub_(3 << 23).view(torch.float32)
    code = torch.copysign(torch.floor(code.abs().div_(step).view(-1).add_(up)).view(-1, BLOCK).mul_(step), code)
    if root:
        code = torch.where(t > 0, code.clamp_min_(LEAST), code)
    return code.to(torch.float8_e4m3fn).view(-1), (top * (1.0 / TOP)).view(-1)


def _from_codes(code, scale, wide=torch.float32):
    return (code.to(wide).view(-1, BLOCK) * scale.to(wide).unsqueeze(1)).view(-1)


def _adamw_plain(s):
    """m <- b1 m + (1 - b1) g, v <- b2 v + (1 - b2) g^2, p <- p (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps),
    in this order of operations; the parameters' tensors lie in one flat buffer, so one pass of each operation serves all."""
    case, t = s["case"], s["case"]["step"] + 1
    s["case"] = dict(case, step=t)
    g = s["grad"].float()
    if case["bits"] == 32:
        m, v = s["exp_avg"], s["exp_avg_sq"]
    else:
        m = _from_codes(s["exp_avg"], s["exp_avg_scale"])
        v = _from_codes(s["exp_avg_rms"], s["exp_avg_rms_scale"]).square_()
    m.mul_(BETA1).add_(g * (1.0 - BETA1))
    v.mul_(BETA2).add_((g * g).mul_(1.0 - BETA2))
    root = v.sqrt()
    step = m / (root * (1.0 / math.sqrt(1.0 - BETA2 ** t)) + EPS)
    p = s["master"] if case["master"] else s["param"].float()
    p.mul_(1.0 - LR * DECAY).sub_(step.mul_(LR / (1.0 - BETA1 ** t)))
    s["param"].copy_(p)
    got = {"param": s["param"]}
    if case["master"]:
        got["master"] = p
    if case["bits"] == 8:
        s["exp_avg"], s["exp_avg_scale"] = _to_codes(m, False, _dither(s["place"], t, M_ALONG, M_AHEAD))
        s["exp_avg_rms"], s["exp_avg_rms_scale"] = _to_codes(root, True, _dither(s["place"], t, R_ALONG, R_AHEAD))
    got.update((n, s[n]) for n in STATE[case["bits"]])
    return got


def run(state):
    if state["case"]["op"] == "linear":
        if own:
            return _linear_own(state)
        with torch.no_grad():
            return {k: v.to(state["x"].dtype) for k, v in _linear_plain(state).items()}
    if own:
        state["opt"].step()
        return {"param": state["param"], **state["opt"].state_buffers()}
    with torch.no_grad():
        return _adamw_plain(state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "linear":
        m, k, n, b = case["m"], case["k"], case["n"], BYTES[case["dtype"]]
        ends = m * n * (1 + case["residual"]) + n * case["bias"]
        if not case["train"]:
            return {"bytes": b * (m * k + k * n + ends), "flops": 2 * m * k * n}
        return {"bytes": b * (m * k + k * n + ends + m * n + m * k + k * n + n * case["bias"]), "flops": 6 * m * k * n}
    n, b = sum(_sizes(case)), BYTES[case["dtype"]]
    moments = 16 if case["bits"] == 32 else 4 + 4 * 4 / BLOCK          # both read and written, the blocks' scales with them
    return {"bytes": int(n * (2 * b + b + moments + (8 - b if case["master"] else 0))), "flops": 16 * n}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def _codes64(t, root, place, turn, along, ahead):
    """As _to_codes, from values in 64 bits: e4m3 has 3 bits behind the leading one, and steps of 2^-9 below 2^-6."""
    up = ((place.long() * along + turn * ahead) % (1 << 32) // (1 << 16)).double() / 65536
    t = t.view(-1, BLOCK)
    top = t.abs().max(1, keepdim=True).values.clamp_min(FLOOR)
    c = t / top * TOP
    step = torch.ldexp(torch.ones_like(c), torch.frexp(c)[1].sub_(1).clamp_min_(-6) - 3)
    c = torch.sign(c) * torch.floor(torch.abs(c) / step + up.view(-1, BLOCK)) * step
    if root:
        c = torch.where(t > 0, torch.maximum(c, torch.full_like(c, LEAST)), c)
    return c.view(-1), (top / TOP).view(-1)


def exact(case, seed):
    """The same outputs from the definitions, in 64 bits. A quantised moment is given as its code's value, a scale as it is."""
    with torch.no_grad():
        if case["op"] == "linear":
            s = _linear_inputs(case, seed)
            a = torch.matmul(s["x"].double(), s["weight"].double())
            if s["bias"] is not None:
                a += s["bias"].double()
            normal = 0.5 * torch.special.erfc(-a / math.sqrt(2.0)) if case["act"] == "gelu" else None
            gate = 1.0 / (1.0 + torch.exp(-a)) if case["act"] == "silu" else None
            y = {"none": lambda: a, "relu": lambda: torch.maximum(a, torch.zeros_like(a)), "gelu": lambda: a * normal, "silu": lambda: a * gate}[case["act"]]()
            got = {"y": y + s["residual"].double() if s["residual"] is not None else y}
            if case["train"]:
                g = s["dy"].double()
                slope = {"none": lambda: 1.0, "relu": lambda: (a > 0).double(), "gelu": lambda: normal + a * torch.exp(-a * a / 2) / math.sqrt(2 * math.pi),
                         "silu": lambda: gate + a * gate * (1 - gate)}[case["act"]]()
                p = g * slope
                got["dx"] = torch.matmul(p, s["weight"].double().t())
                got["dw"] = torch.matmul(s["x"].double().t(), p)
                if s["bias"] is not None:
                    got["db"] = p.sum(0)
                if s["residual"] is not None:
                    got["dr"] = g
            return got
        s = _adamw_inputs(case, seed)
        t = case["step"] + 1
        g = s["grad"].double()
        if case["bits"] == 32:
            m, v = s["exp_avg"].double(), s["exp_avg_sq"].double()
        else:
            m = _from_codes(s["exp_avg"], s["exp_avg_scale"], torch.float64)
            v = _from_codes(s["exp_avg_rms"], s["exp_avg_rms_scale"], torch.float64) ** 2
        m = BETA1 * m + (1 - BETA1) * g
        v = BETA2 * v + (1 - BETA2) * g * g
        p = (s["master"] if case["master"] else s["param"]).double()
        p = p - LR * DECAY * p - LR * (m / (1 - BETA1 ** t)) / (torch.sqrt(v / (1 - BETA2 ** t)) + EPS)
        got = {"param": p}
        if case["master"]:
            got["master"] = p
        if case["bits"] == 32:
            got.update(exp_avg=m, exp_avg_sq=v)
        else:
            got["exp_avg"], got["exp_avg_scale"] = _codes64(m, False, s["place"], t, M_ALONG, M_AHEAD)
            got["exp_avg_rms"], got["exp_avg_rms_scale"] = _codes64(torch.sqrt(v), True, s["place"], t, R_ALONG, R_AHEAD)
        return got
