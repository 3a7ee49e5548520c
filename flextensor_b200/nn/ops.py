"""Compute definitions of the hot-path operators, PyTorch conventions.

Each function returns the output ``Tensor`` of a small op graph (see ``ir.py``), with the
same argument meaning, shape checks, loop-axis names and output-size formulas as the
reference's ``flextensor/nn/ops.py``:

  zero_pad2d             ops.py:83-117
  conv2d_nchw            ops.py:419-479   (pad -> conv [-> bias]: a 2- or 3-op graph)
  depthwise_conv2d_nchw  ops.py:622-678   (weight layout [C, factor, kh, kw])
  conv2d_nhwc            ops.py:482-560   (conv2d_nchwc with one channel block: channels-last tensors)
  conv1d                 ops.py:293-351   (the same kernels, on a one-row image)
  zero_pad3d             ops.py:157-189
  conv3d_ncdhw           ops.py:689-751   (the per-tap conv kernel with a depth-tap loop)
  gemm_conv2d_nchw       ops.py:982-1044  (im2col -> GEMM -> col2img: the conv2d result by another route)
  conv2d_1x1_packed      task.py:168-173  (out[b,k,i] = sum_rc A[b,rc,i] * B[k,rc])
  gemm                   ops.py:1074-1108 (four transpose variants)
  batch_gemm             ops.py:1111-1158
  gemm_int8              no ops.py symbol; contract of test/test_tvm/legacy/gemm_int8.py:15-21
  linear, route_experts, expert_plan, expert_linear, expert_combine
                         no counterpart: the feed-forward operators of language models (matrix product
                         with bias, activation, gate and residual; routing to experts and their products)

The reference is fp32 only; ``dtype`` follows the input tensors here so that the same
index expressions serve bf16 (fp32 accumulate) and int8 (int32 accumulate).
"""
from ..backend import MAX_EXPERTS, MAX_GROUPS, MAX_TOP_K
from ..ir import ComputeOp, Tensor, reduce_axis
from ..utils import assert_print


def _pair(value, what):
    if isinstance(value, int):
        return (value, value)
    value = tuple(int(v) for v in value)
    assert_print(len(value) == 2, "%s must be an int or a pair" % what)
    return value


def _acc_dtype(dtype):
    return {"float32": "float32", "bfloat16": "float32", "int8": "int32"}.get(dtype, dtype)


def zero_pad2d(inputs, padding=0):
    """Zero padding of [batch, channel, height, width]; padding int, (h, w) or (up, down, left, right)."""
    if isinstance(padding, int):
        padding = (padding,) * 4
    assert_print(isinstance(padding, tuple), "type(padding)={}".format(type(padding)))
    if len(padding) == 2:
        padding = (padding[0], padding[0], padding[1], padding[1])
    assert_print(len(padding) == 4)
    b, c, h, w = (int(s) for s in inputs.shape)
    shape = (b, c, h + padding[0] + padding[1], w + padding[2] + padding[3])
    op = ComputeOp("pad2d", "Padding", shape, inputs.dtype, [inputs], ("b", "c", "h", "w"),
                   attrs={"padding": tuple(padding)})
    return op.output(0)


def _bias_add(output, bias):
    op = ComputeOp("bias_add", "bias_add", tuple(int(s) for s in output.shape), output.dtype,
                   [output, bias], ("b", "c", "h", "w"), attrs={"axis": 1})
    return op.output(0)


def relu(inputs):
    """max(x, 0) elementwise; following a convolution (or its bias) it is folded into the conv kernel's
    epilogue, as the bias is - the conv + bias + ReLU chain of a network runs as one kernel."""
    names = {3: ("b", "c", "l"), 5: ("b", "c", "d", "h", "w")}.get(len(inputs.shape), ("b", "c", "h", "w")[:len(inputs.shape)])
    op = ComputeOp("relu", "relu", tuple(int(s) for s in inputs.shape), inputs.dtype, [inputs], names)
    return op.output(0)


def conv2d_nchw(inputs, weight, bias=None, stride=1, padding=0, dilation=1, groups=1):
    """inputs [N,C,H,W], weight [K, C/groups, kh, kw] -> [N, K, out_h, out_w]."""
    n, c, in_h, in_w = (int(s) for s in inputs.shape)
    k, cg, k_h, k_w = (int(s) for s in weight.shape)
    assert_print(cg * groups == c)
    kg = k // groups
    assert_print(kg * groups == k)
    stride, padding, dilation = _pair(stride, "stride"), _pair(padding, "padding"), _pair(dilation, "dilation")
    out_h = (in_h + 2 * padding[0] - dilation[0] * (k_h - 1) - 1) // stride[0] + 1
    out_w = (in_w + 2 * padding[1] - dilation[1] * (k_w - 1) - 1) // stride[1] + 1
    rc = reduce_axis((0, cg), name="rc")
    rh = reduce_axis((0, k_h), name="rh")
    rw = reduce_axis((0, k_w), name="rw")
    padded = zero_pad2d(inputs, padding=padding)
    op = ComputeOp("conv2d", "compute", (n, k, out_h, out_w), _acc_dtype(inputs.dtype), [padded, weight],
                   ("b", "c", "h", "w"), reduce_axes=[rc, rw, rh],
                   attrs={"stride": stride, "padding": padding, "dilation": dilation, "groups": groups})
    out = op.output(0)
    if bias is not None:
        out = _bias_add(out, bias)
    return out


def conv2d_nhwc(inputs, weight, bias=None, stride=1, padding=0, dilation=1, groups=1):
    """inputs [N,H,W,C], weight [K, C/groups, kh, kw] -> [N, out_h, out_w, K]: the conv2d of ``conv2d_nchw`` on
    channels-last tensors.  The reference rewrites conv2d tasks to the blocked NCHWc layout for its CPU target
    (flextensor/nn/ops.py:482-560 conv2d_nchwc: [N, C/v, H, W, v]); with one block holding all channels that is
    this layout, which is the one the tensor-core kernels read without a layout pass."""
    n, in_h, in_w, c = (int(s) for s in inputs.shape)
    k, cg, k_h, k_w = (int(s) for s in weight.shape)
    assert_print(cg * groups == c)
    kg = k // groups
    assert_print(kg * groups == k)
    stride, padding, dilation = _pair(stride, "stride"), _pair(padding, "padding"), _pair(dilation, "dilation")
    out_h = (in_h + 2 * padding[0] - dilation[0] * (k_h - 1) - 1) // stride[0] + 1
    out_w = (in_w + 2 * padding[1] - dilation[1] * (k_w - 1) - 1) // stride[1] + 1
    rc = reduce_axis((0, cg), name="rc")
    rh = reduce_axis((0, k_h), name="rh")
    rw = reduce_axis((0, k_w), name="rw")
    pad_op = ComputeOp("pad2d", "Padding", (n, in_h + 2 * padding[0], in_w + 2 * padding[1], c), inputs.dtype, [inputs],
                       ("b", "h", "w", "c"), attrs={"padding": (padding[0], padding[0], padding[1], padding[1]),
                                                    "layout": "nhwc"})
    op = ComputeOp("conv2d", "compute", (n, out_h, out_w, k), _acc_dtype(inputs.dtype), [pad_op.output(0), weight],
                   ("b", "h", "w", "c"), reduce_axes=[rc, rw, rh],
                   attrs={"stride": stride, "padding": padding, "dilation": dilation, "groups": groups, "form": "nhwc"})
    out = op.output(0)
    if bias is not None:
        bop = ComputeOp("bias_add", "bias_add", (n, out_h, out_w, k), out.dtype, [out, bias], ("b", "h", "w", "c"),
                        attrs={"axis": 3})
        out = bop.output(0)
    return out


def zero_pad1d(inputs, padding=0):
    """Zero padding of [batch, channel, length]; padding int or (left, right)."""
    if isinstance(padding, int):
        padding = (padding, padding)
    assert_print(isinstance(padding, tuple) and len(padding) == 2, "type(padding)={}".format(type(padding)))
    b, c, l = (int(s) for s in inputs.shape)
    op = ComputeOp("pad2d", "Padding", (b, c, l + padding[0] + padding[1]), inputs.dtype, [inputs], ("b", "c", "l"),
                   attrs={"padding": tuple(padding)})
    return op.output(0)


def conv1d(inputs, weight, bias=None, stride=1, padding=0, dilation=1, groups=1):
    """inputs [N,C,L], weight [K, C/groups, k] -> [N, K, out_len]: served by the conv2d kernels
    on a one-row image (flextensor/nn/ops.py:293-351)."""
    n, c, in_len = (int(s) for s in inputs.shape)
    k, cg, k_len = (int(s) for s in weight.shape)
    assert_print(cg * groups == c, "left=%d, right=%d" % (cg * groups, c))
    assert_print(k % groups == 0)
    stride = stride[0] if isinstance(stride, tuple) else int(stride)
    padding = padding[0] if isinstance(padding, tuple) else int(padding)
    dilation = int(dilation)
    out_len = (in_len + 2 * padding - dilation * (k_len - 1) - 1) // stride + 1
    rc = reduce_axis((0, cg), name="rc")
    rl = reduce_axis((0, k_len), name="rl")
    padded = zero_pad1d(inputs, padding=padding)
    op = ComputeOp("conv2d", "compute", (n, k, out_len), _acc_dtype(inputs.dtype), [padded, weight],
                   ("b", "c", "l"), reduce_axes=[rc, rl],
                   attrs={"stride": (1, stride), "padding": (0, padding), "dilation": (1, dilation), "groups": groups,
                          "form": "conv1d"})
    out = op.output(0)
    if bias is not None:
        bop = ComputeOp("bias_add", "bias_add", (n, k, out_len), out.dtype, [out, bias], ("b", "c", "l"),
                        attrs={"axis": 1})
        out = bop.output(0)
    return out


def _triple(value, what):
    if isinstance(value, int):
        return (value, value, value)
    value = tuple(int(v) for v in value)
    assert_print(len(value) == 3, "%s must be an int or a triple" % what)
    return value


def zero_pad3d(inputs, padding=0):
    """Zero padding of [batch, channel, depth, height, width]; padding int, (d, h, w) or
    (d_up, d_down, h_up, h_down, w_up, w_down)."""
    if isinstance(padding, int):
        padding = (padding,) * 6
    assert_print(isinstance(padding, tuple), "type(padding)={}".format(type(padding)))
    if len(padding) == 3:
        padding = (padding[0], padding[0], padding[1], padding[1], padding[2], padding[2])
    assert_print(len(padding) == 6)
    b, c, d, h, w = (int(s) for s in inputs.shape)
    shape = (b, c, d + padding[0] + padding[1], h + padding[2] + padding[3], w + padding[4] + padding[5])
    op = ComputeOp("pad2d", "Padding", shape, inputs.dtype, [inputs], ("b", "c", "d", "h", "w"),
                   attrs={"padding": tuple(padding)})
    return op.output(0)


def conv3d_ncdhw(inputs, weight, bias=None, stride=1, padding=0, dilation=1, groups=1):
    """inputs [N,C,D,H,W], weight [K, C/groups, kd, kh, kw] -> [N, K, out_d, out_h, out_w]
    (flextensor/nn/ops.py:689-751)."""
    n, c, in_d, in_h, in_w = (int(s) for s in inputs.shape)
    k, cg, k_d, k_h, k_w = (int(s) for s in weight.shape)
    assert_print(cg * groups == c)
    kg = k // groups
    assert_print(kg * groups == k)
    stride, padding, dilation = _triple(stride, "stride"), _triple(padding, "padding"), _triple(dilation, "dilation")
    out_d = (in_d + 2 * padding[0] - dilation[0] * (k_d - 1) - 1) // stride[0] + 1
    out_h = (in_h + 2 * padding[1] - dilation[1] * (k_h - 1) - 1) // stride[1] + 1
    out_w = (in_w + 2 * padding[2] - dilation[2] * (k_w - 1) - 1) // stride[2] + 1
    rc = reduce_axis((0, cg), name="rc")
    rd = reduce_axis((0, k_d), name="rd")
    rh = reduce_axis((0, k_h), name="rh")
    rw = reduce_axis((0, k_w), name="rw")
    padded = zero_pad3d(inputs, padding=padding)
    op = ComputeOp("conv2d", "compute", (n, k, out_d, out_h, out_w), _acc_dtype(inputs.dtype), [padded, weight],
                   ("b", "c", "d", "h", "w"), reduce_axes=[rc, rd, rw, rh],
                   attrs={"stride": stride, "padding": padding, "dilation": dilation, "groups": groups,
                          "form": "conv3d"})
    out = op.output(0)
    if bias is not None:
        bop = ComputeOp("bias_add", "bias_add", (n, k, out_d, out_h, out_w), out.dtype, [out, bias],
                        ("b", "c", "d", "h", "w"), attrs={"axis": 1})
        out = bop.output(0)
    return out


def gemm_conv2d_nchw(inputs, weight, bias=None, stride=1, padding=0, dilation=1, groups=1):
    """The reference builds this result as im2col -> GEMM -> col2img (flextensor/nn/ops.py:982-1044);
    the numbers are those of ``conv2d_nchw``, and here the same implicit-GEMM kernels compute them
    without materialising the column matrix."""
    return conv2d_nchw(inputs, weight, bias=bias, stride=stride, padding=padding, dilation=dilation, groups=groups)


def conv2d_1x1_packed(A, B):
    """out[b,k,i] = sum_rc A[b,rc,i] * B[k,rc]: a 1x1 convolution on pixels packed into one axis
    (flextensor/task.py:168-173), i.e. a batched GEMM with the same left operand for every item."""
    n, c, hw = (int(s) for s in A.shape)
    k, c2 = (int(s) for s in B.shape)
    assert_print(c2 == c)
    rc = reduce_axis((0, c), name="rc")
    op = ComputeOp("conv2d", "compute", (n, k, hw), _acc_dtype(A.dtype), [A, B], ("b", "k", "i"), reduce_axes=[rc],
                   attrs={"stride": (1, 1), "padding": (0, 0), "dilation": (1, 1), "groups": 1, "form": "packed_1x1"})
    return op.output(0)


def depthwise_conv2d_nchw(inputs, weight, bias=None, stride=1, padding=0, dilation=1):
    """inputs [N,C,H,W], weight [C, factor, kh, kw] -> [N, C*factor, out_h, out_w]."""
    n, c, in_h, in_w = (int(s) for s in inputs.shape)
    c2, factor, k_h, k_w = (int(s) for s in weight.shape)
    assert_print(c2 == c)
    stride, padding, dilation = _pair(stride, "stride"), _pair(padding, "padding"), _pair(dilation, "dilation")
    out_h = (in_h + 2 * padding[0] - dilation[0] * (k_h - 1) - 1) // stride[0] + 1
    out_w = (in_w + 2 * padding[1] - dilation[1] * (k_w - 1) - 1) // stride[1] + 1
    rh = reduce_axis((0, k_h), name="rh")
    rw = reduce_axis((0, k_w), name="rw")
    padded = zero_pad2d(inputs, padding=padding)
    op = ComputeOp("depthwise_conv2d", "compute", (n, c * factor, out_h, out_w), _acc_dtype(inputs.dtype),
                   [padded, weight], ("b", "c", "h", "w"), reduce_axes=[rw, rh],
                   attrs={"stride": stride, "padding": padding, "dilation": dilation, "factor": factor})
    out = op.output(0)
    if bias is not None:
        out = _bias_add(out, bias)
    return out


def _gemm_dims(a_shape, b_shape, transposeA, transposeB):
    """(M, N, K) of op(A).op(B) for 2-d shapes, with the reference's shape assertion."""
    if transposeA and transposeB:      # A[k,i], B[j,k]
        assert_print(a_shape[0] == b_shape[1])
        return a_shape[1], b_shape[0], b_shape[1]
    if transposeA:                     # A[k,i], B[k,j]
        assert_print(a_shape[0] == b_shape[0])
        return a_shape[1], b_shape[1], b_shape[0]
    if transposeB:                     # A[i,k], B[j,k]
        assert_print(a_shape[1] == b_shape[1])
        return a_shape[0], b_shape[0], b_shape[1]
    assert_print(a_shape[1] == b_shape[0])  # A[i,k], B[k,j]
    return a_shape[0], b_shape[1], b_shape[0]


def gemm(A, B, transposeA=False, transposeB=False):
    """C[i,j] = sum_k op(A)[i,k] * op(B)[k,j]."""
    m, n, k = _gemm_dims([int(s) for s in A.shape], [int(s) for s in B.shape], transposeA, transposeB)
    rk = reduce_axis((0, k), name="k")
    op = ComputeOp("gemm", "compute", (m, n), _acc_dtype(A.dtype), [A, B], ("i", "j"), reduce_axes=[rk],
                   attrs={"transposeA": bool(transposeA), "transposeB": bool(transposeB)})
    return op.output(0)


def batch_gemm(A, B, transposeA=False, transposeB=False, out_dtype=None):
    """C[b,i,j] = sum_k op(A[b])[i,k] * op(B[b])[k,j]; ``out_dtype`` defaults to the input dtype
    for bf16 (accumulation is always fp32) and to fp32 for fp32."""
    a_shape, b_shape = [int(s) for s in A.shape], [int(s) for s in B.shape]
    assert_print(a_shape[0] == b_shape[0])
    m, n, k = _gemm_dims(a_shape[1:], b_shape[1:], transposeA, transposeB)
    rk = reduce_axis((0, k), name="k")
    dtype = out_dtype or A.dtype
    op = ComputeOp("batch_gemm", "compute", (a_shape[0], m, n), dtype, [A, B], ("b", "i", "j"),
                   reduce_axes=[rk], attrs={"transposeA": bool(transposeA), "transposeB": bool(transposeB)})
    return op.output(0)


def gemm_int8(A, B, transposeA=False, transposeB=False):
    """int8 x int8 -> int32 GEMM; ``transposeB=True`` is the legacy script's B[n,k] layout."""
    assert_print(A.dtype == "int8" and B.dtype == "int8", "gemm_int8 takes int8 tensors")
    m, n, k = _gemm_dims([int(s) for s in A.shape], [int(s) for s in B.shape], transposeA, transposeB)
    rk = reduce_axis((0, k), name="k")
    op = ComputeOp("gemm_int8", "compute", (m, n), "int32", [A, B], ("i", "j"), reduce_axes=[rk],
                   attrs={"transposeA": bool(transposeA), "transposeB": bool(transposeB)})
    return op.output(0)


# ---------------------------------------------------------------- feed-forward operators of language models
_ACTIVATIONS = ("none", "relu", "gelu", "gelu_tanh", "silu")


def _operands(**named):
    """(names, tensors) of the operands that are given, in order."""
    given = [(name, t) for name, t in named.items() if t is not None]
    return tuple(name for name, _ in given), [t for _, t in given]


def _product_dims(x, weight, bias, residual, activation, gated, lead):
    """(rows, N, K) of a product with an epilogue; ``lead``: leading dimensions of weight and bias."""
    rows, k = (int(s) for s in x.shape)
    shape = [int(s) for s in weight.shape]
    assert_print(len(shape) == len(lead) + 2 and shape[:-2] == lead and shape[-1] == k,
                 "weight of shape %s for rows of %d" % (shape, k))
    assert_print(activation in _ACTIVATIONS, "activation must be one of %s" % (_ACTIVATIONS,))
    assert_print(x.dtype in ("bfloat16", "float16") and weight.dtype == x.dtype, "x and weight are bfloat16 or float16")
    wide = shape[-2]
    assert_print(not gated or wide % 2 == 0, "a gated weight has an even number of rows")
    n = wide // 2 if gated else wide
    if bias is not None:
        assert_print([int(s) for s in bias.shape] == lead + [wide] and bias.dtype == x.dtype, "bias of shape %s" % (bias.shape,))
    if residual is not None:
        assert_print([int(s) for s in residual.shape] == [rows, n] and residual.dtype == x.dtype, "residual of shape %s" % (residual.shape,))
    return rows, n, k


def linear(x, weight, bias=None, residual=None, activation="none", gated=False):
    """out[t,i] = act(sum_k x[t,k] * weight[i,k] + bias[i]) + residual[t,i]; ``gated``: weight [2N,K] holds the gate rows,
    then the others, out = act(gate) * other + residual.  bfloat16 or float16, one kernel."""
    t, n, k = _product_dims(x, weight, bias, residual, activation, gated, [])
    names, tensors = _operands(x=x, weight=weight, bias=bias, residual=residual)
    op = ComputeOp("linear", "linear", (t, n), x.dtype, tensors, ("t", "i"), reduce_axes=[reduce_axis((0, k), name="k")],
                   attrs={"operands": names, "activation": activation, "gated": bool(gated)})
    return op.output(0)


def route_experts(logits, top_k, bias=None, scoring="softmax", groups=1, top_groups=1, renormalize=True, scale=1.0):
    """(ids, weights), both [T, top_k]: the experts of every token and their weights (``backend.route_experts``)."""
    assert_print(logits.ndim == 2 and logits.dtype in ("float32", "bfloat16", "float16"),
                 "logits are [T, E] in float32, bfloat16 or float16")
    t, e = (int(s) for s in logits.shape)
    assert_print(1 <= e <= MAX_EXPERTS and top_k <= MAX_TOP_K and groups <= MAX_GROUPS,
                 "at most %d experts, top_k %d and %d groups" % (MAX_EXPERTS, MAX_TOP_K, MAX_GROUPS))
    if bias is not None:
        assert_print([int(s) for s in bias.shape] == [e] and bias.dtype == "float32", "bias is [E] in float32")
    assert_print(1 <= top_groups <= groups and e % groups == 0 and 1 <= top_k <= e // groups * top_groups,
                 "top_k %d of %d experts in %d groups, %d kept" % (top_k, e, groups, top_groups))
    assert_print(scoring in ("softmax", "sigmoid"), "scoring must be softmax or sigmoid")
    names, tensors = _operands(logits=logits, bias=bias)
    op = ComputeOp("route_experts", "route_experts", (t, top_k), "int32", tensors, ("t", "j"),
                   attrs={"operands": names, "scoring": scoring, "groups": int(groups), "top_groups": int(top_groups),
                          "renormalize": bool(renormalize), "scale": float(scale)},
                   more_outputs=[((t, top_k), "float32")])
    return op.output(0), op.output(1)


def expert_plan(ids, experts):
    """(offsets [experts+1], order [T*top_k], slots [T*top_k]): rows of ids [T, top_k] sorted by expert."""
    assert_print(ids.ndim == 2 and ids.dtype == "int32", "ids are [T, top_k] in int32")
    t, top_k = (int(s) for s in ids.shape)
    assert_print(1 <= experts <= MAX_EXPERTS and 1 <= top_k <= MAX_TOP_K,
                 "1 to %d experts and top_k of 1 to %d" % (MAX_EXPERTS, MAX_TOP_K))
    op = ComputeOp("expert_plan", "expert_plan", (experts + 1,), "int32", [ids], ("e",),
                   attrs={"tokens": t, "top_k": top_k, "experts": int(experts)},
                   more_outputs=[((t * top_k,), "int32"), ((t * top_k,), "int32")])
    return op.output(0), op.output(1), op.output(2)


def _plan_attrs(plan):
    assert_print(len(plan) == 3 and getattr(plan[0].op, "kind", None) == "expert_plan" and
                 all(t is plan[0].op.output(i) for i, t in enumerate(plan)), "plan is what expert_plan returned")
    return dict(plan[0].op.attrs)


def expert_linear(x, weight, plan, bias=None, activation="none", gated=False, gather=False):
    """out[p,i] for every sorted place p of expert e: the epilogue of ``linear`` over its row times weight[e] ([E,N,K], gated
    [E,2N,K]) plus bias[e].  ``gather``: x is [T,K], read by token; else [T*top_k,K], sorted."""
    sizes = _plan_attrs(plan)
    rows, n, k = _product_dims(x, weight, bias, None, activation, gated, [sizes["experts"]])
    assert_print(rows == (sizes["tokens"] if gather else sizes["tokens"] * sizes["top_k"]), "x has %d rows" % rows)
    names, tensors = _operands(x=x, weight=weight, bias=bias)
    op = ComputeOp("expert_linear", "expert_linear", (sizes["tokens"] * sizes["top_k"], n), x.dtype, tensors + list(plan),
                   ("p", "i"), reduce_axes=[reduce_axis((0, k), name="k")],
                   attrs={"operands": names + ("offsets", "order", "slots"), "activation": activation, "gated": bool(gated),
                          "gather": bool(gather), **sizes})
    return op.output(0)


def expert_combine(y, plan, weights=None, residual=None):
    """out[t,i] = residual[t,i] + sum_j weights[t,j] * y[place of (t, j), i]; dropped rows add nothing."""
    sizes = _plan_attrs(plan)
    assert_print(y.ndim == 2 and y.dtype in ("bfloat16", "float16"), "y is [T * top_k, N] in bfloat16 or float16")
    rows, n = (int(s) for s in y.shape)
    t, top_k = sizes["tokens"], sizes["top_k"]
    assert_print(rows == t * top_k, "y has %d rows" % rows)
    if weights is not None:
        assert_print([int(s) for s in weights.shape] == [t, top_k] and weights.dtype == "float32", "weights are [T, top_k] in float32")
    if residual is not None:
        assert_print([int(s) for s in residual.shape] == [t, n] and residual.dtype == y.dtype, "residual of shape %s" % (residual.shape,))
    names, tensors = _operands(y=y, weights=weights, residual=residual)
    op = ComputeOp("expert_combine", "expert_combine", (t, n), y.dtype, tensors + list(plan), ("t", "i"),
                   reduce_axes=[reduce_axis((0, top_k), name="j")],
                   attrs={"operands": names + ("offsets", "order", "slots"), **sizes})
    return op.output(0)
