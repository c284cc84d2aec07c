"""The operators on device memory (section 5 of ``include/fomoe_b200.h``) for torch tensors that live on the GPU.

Every call enqueues on torch's current stream of the handle's device, allocates its results (and the experts' workspace)
through torch on that stream, and neither copies to the host nor synchronises: calls can be captured into a CUDA graph.
Rows may be strided; the last axis of a tensor is contiguous.  FP8 tensors are ``torch.float8_e4m3fn`` (or ``uint8`` with
the same bytes).  The operators serve: autograd does not see them (results carry no gradient, and ``norm(inplace=True)``
writes x without its version counter)."""
import ctypes as C

F32, BF16, F8 = 0, 1, 2
_OVER = 1 << 31   # no C int (ctypes would keep the low 32 bits)


class RouteConfig(C.Structure):
    _fields_ = [("n_experts", C.c_int), ("top_k", C.c_int), ("score", C.c_int), ("n_group", C.c_int),
                ("topk_group", C.c_int), ("group_best", C.c_int), ("renorm", C.c_int), ("scale", C.c_float)]


class NormArgs(C.Structure):
    _fields_ = [("n_tokens", C.c_int), ("n", C.c_int), ("eps", C.c_float), ("offset", C.c_float), ("scale", C.c_float),
                ("x", C.c_void_p), ("x_type", C.c_int), ("x_stride", C.c_int64),
                ("block", C.c_void_p), ("block_type", C.c_int), ("block_stride", C.c_int64), ("post", C.c_void_p),
                ("gate", C.c_void_p), ("gate_stride", C.c_int64), ("gate_step", C.c_int),
                ("x_out", C.c_void_p), ("x_out_stride", C.c_int64), ("pre", C.c_void_p),
                ("h", C.c_void_p), ("h_type", C.c_int), ("h_stride", C.c_int64),
                ("h_scales", C.c_void_p), ("h_scales_stride", C.c_int64)]


class MatmulArgs(C.Structure):
    _fields_ = [("m", C.c_int), ("n", C.c_int), ("k", C.c_int),
                ("a", C.c_void_p), ("a_stride", C.c_int64), ("a_scales", C.c_void_p), ("a_scales_stride", C.c_int64),
                ("b", C.c_void_p), ("b_stride", C.c_int64), ("b_scales", C.c_void_p), ("b_scales_stride", C.c_int64),
                ("out", C.c_void_p), ("out_type", C.c_int), ("out_stride", C.c_int64)]


class ExpertsArgs(C.Structure):
    _fields_ = [("n_tokens", C.c_int), ("n_embd", C.c_int), ("n_inter", C.c_int),
                ("n_experts", C.c_int), ("top_k", C.c_int), ("has_shared", C.c_int),
                ("x", C.c_void_p), ("x_stride", C.c_int64), ("x_scales", C.c_void_p), ("x_scales_stride", C.c_int64),
                ("ids", C.c_void_p), ("weights", C.c_void_p), ("gate_up", C.c_void_p), ("gate_up_scales", C.c_void_p),
                ("down", C.c_void_p), ("down_scales", C.c_void_p), ("out", C.c_void_p), ("out_stride", C.c_int64)]


SIGS = {
    "fomoe_b200_ops_create": (C.c_void_p, [C.c_int]),
    "fomoe_b200_ops_destroy": (None, [C.c_void_p]),
    "fomoe_b200_ops_last_error": (C.c_char_p, [C.c_void_p]),
    "fomoe_b200_ops_status": (C.c_int, [C.c_void_p]),
    "fomoe_b200_ops_kernel_launches": (C.c_uint64, [C.c_void_p]),
    "fomoe_b200_ops_route": (C.c_int, [C.c_void_p, C.POINTER(RouteConfig), C.c_int, C.c_void_p, C.c_int, C.c_int64,
                                       C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p]),
    "fomoe_b200_ops_norm": (C.c_int, [C.c_void_p, C.POINTER(NormArgs), C.c_void_p]),
    "fomoe_b200_ops_f8_quantize": (C.c_int, [C.c_void_p, C.c_int, C.c_int, C.c_void_p, C.c_int, C.c_int64, C.c_void_p,
                                             C.c_int64, C.c_void_p, C.c_int64, C.c_void_p]),
    "fomoe_b200_ops_f8_matmul": (C.c_int, [C.c_void_p, C.POINTER(MatmulArgs), C.c_void_p]),
    "fomoe_b200_ops_f8_experts_workspace": (C.c_uint64, [C.POINTER(ExpertsArgs)]),
    "fomoe_b200_ops_f8_experts": (C.c_int, [C.c_void_p, C.POINTER(ExpertsArgs), C.c_void_p, C.c_uint64, C.c_void_p]),
}

SCORES = {"softmax": 0, "sigmoid": 1}


class DeviceOps:
    """Handle of the operators on one GPU.  Used from one thread at a time; any number of streams."""

    def __init__(self, device=0):
        import torch

        from . import lib
        self._l, self._t, self.device = lib(), torch, device
        self._h = self._l.fomoe_b200_ops_create(device)
        if not self._h:
            raise RuntimeError("fomoe_b200_ops_create failed (no such CUDA device, or not one this library is built for)")
        self._float = {torch.float32: F32, torch.bfloat16: BF16}
        self._out = {"f32": (torch.float32, F32), "bf16": (torch.bfloat16, BF16)}
        self._f8 = (torch.float8_e4m3fn, torch.uint8)
        self._f32, self._i32, self._u8 = (torch.float32,), (torch.int32,), (torch.uint8, torch.bool)
        # the current stream's handle without building a Stream object around it, where torch offers that
        self._raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)

    def close(self):
        """Release the handle.  Calls in flight and graphs that hold its calls may outlive it; their status is lost."""
        if getattr(self, "_h", None):
            self._l.fomoe_b200_ops_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()   # (asks nothing of the device: a wait would end a capture of another thread or stream)
        except Exception:
            pass

    def status(self):
        """0 nothing, 1 an expert id outside the table, 2 a bounded wait ran out (first, where both happened); reading clears it."""
        return int(self._l.fomoe_b200_ops_status(self._h))

    def kernel_launches(self):
        return int(self._l.fomoe_b200_ops_kernel_launches(self._h))

    def _ck(self, rc, what):
        if rc != 0:
            raise RuntimeError(f"{what}: {self._l.fomoe_b200_ops_last_error(self._h).decode()}")

    def _stream(self):
        if self._raw_stream is not None:
            return self._raw_stream(self.device)
        return self._t.cuda.current_stream(self.device).cuda_stream

    def _bad(self, t, name, types, shape, what):
        raise ValueError(f"{name}: {what} of {' or '.join(map(str, types))} on CUDA device {self.device}"
                         f"{'' if shape is None else f' of shape {tuple(shape)}'} is wanted, got {tuple(t.shape)} {t.dtype} on "
                         f"{t.device} with strides {t.stride()}")

    def _rows(self, t, name, types, shape=None):
        """Checks a 2-D tensor with contiguous rows, whose sizes are C ints; -> its row stride."""
        if t.numel() >= _OVER and max(t.shape) >= _OVER:
            raise ValueError(f"{name}: less than 2^31 rows and columns are taken, got {tuple(t.shape)}")
        if (t.dim() != 2 or t.dtype not in types or t.get_device() != self.device or (t.stride(1) != 1 and t.shape[1] > 1)
                or (shape is not None and t.shape != shape)):
            self._bad(t, name, types, shape, "a 2-D tensor with contiguous rows")
        return t.stride(0)

    def _flat(self, t, name, types, shape):
        """Checks a contiguous tensor; -> its address."""
        if t.shape != shape or t.dtype not in types or t.get_device() != self.device or not t.is_contiguous():
            self._bad(t, name, types, shape, "a contiguous tensor")
        return t.data_ptr()

    def route(self, logits, top_k, *, score="softmax", bias=None, n_group=1, topk_group=1, group_best=1, renorm=True,
              scale=1.0, valid=None):
        """logits [T, E] f32 or bf16 -> (ids int32 [T, top_k], weights f32 [T, top_k]); see fomoe_b200_ops_route."""
        t = self._t
        stride = self._rows(logits, "logits", self._float)
        T, E = logits.shape
        if score not in SCORES:
            raise ValueError(f"score: 'softmax' or 'sigmoid' is wanted, got {score!r}")
        b = None if bias is None else self._flat(bias, "bias", self._f32, (E,))
        v = None if valid is None else self._flat(valid, "valid", self._u8, (T,))
        if (top_k | n_group | topk_group | group_best) >> 31:
            raise ValueError("top_k, n_group, topk_group and group_best: 0 to 2^31 - 1 is wanted, got "
                             f"{(top_k, n_group, topk_group, group_best)}")
        k = top_k if top_k <= E else 0   # (more is refused by the call)
        ids, w = logits.new_empty((T, k), dtype=t.int32), logits.new_empty((T, k), dtype=t.float32)
        cfg = RouteConfig(E, top_k, SCORES[score], n_group, topk_group, group_best, 1 if renorm else 0, scale)
        self._ck(self._l.fomoe_b200_ops_route(self._h, cfg, T, logits.data_ptr(), self._float[logits.dtype], stride, b, v,
                                              ids.data_ptr(), w.data_ptr(), self._stream()), "route")
        return ids, w

    def norm(self, x, pre=None, *, block=None, post=None, gate=None, scale=1.0, eps=1e-6, offset=0.0, out="bf16",
             inplace=False):
        """The norms around a block (see fomoe_b200_ops_norm): x [T, n]; pre, post f32 [n]; block [T, n]; gate of block's
        type, [T, n], [1, n] or [T, 1].  out: 'f32', 'bf16' or 'f8'.  -> (x', h), or (x', h, scales) with 'f8'.  x' is x
        itself with inplace or without a block; without pre there is no h (None)."""
        t, fl = self._t, self._float
        xs = self._rows(x, "x", fl)
        T, n = x.shape
        x_out, blk, bt, bs, po, ga, gs, gp, xo, xos = x, None, 0, 0, None, None, 0, 0, None, 0
        if block is not None:
            bs = self._rows(block, "block", fl, (T, n))
            blk, bt = block.data_ptr(), fl[block.dtype]
            if post is not None:
                po = self._flat(post, "post", self._f32, (n,))
            if gate is not None:
                gs = self._rows(gate, "gate", (block.dtype,))
                gT, gn = gate.shape
                if gT not in (1, T) or gn not in (1, n):
                    raise ValueError(f"gate: [T, n], [1, n] or [T, 1] is wanted, got {(gT, gn)}")
                ga, gs, gp = gate.data_ptr(), gs if gT > 1 else 0, 1 if gn == n and n > 1 else 0
            if not inplace:
                x_out = t.empty_like(x)
            xo, xos = x_out.data_ptr(), x_out.stride(0)
        elif post is not None or gate is not None:
            raise ValueError("post and gate need a block")
        h = sc = pr = hp = sp = None
        ht = nb = hs = 0
        if pre is not None:
            pr = self._flat(pre, "pre", self._f32, (n,))
            if out == "f8":
                ht, nb = F8, (n + 127) // 128
                h, sc = t.empty_like(x, dtype=t.float8_e4m3fn), x.new_empty((T, nb), dtype=t.float32)
                sp = sc.data_ptr()
            elif out in self._out:
                dt, ht = self._out[out]
                h = t.empty_like(x, dtype=dt)
            else:
                raise ValueError(f"out: 'f32', 'bf16' or 'f8' is wanted, got {out!r}")
            hp, hs = h.data_ptr(), h.stride(0)
        a = NormArgs(T, n, eps, offset, scale, x.data_ptr(), fl[x.dtype], xs, blk, bt, bs, po, ga, gs, gp, xo, xos, pr, hp, ht,
                     hs, sp, nb)
        self._ck(self._l.fomoe_b200_ops_norm(self._h, a, self._stream()), "norm")
        return (x_out, h, sc) if out == "f8" else (x_out, h)

    def f8_quantize(self, x):
        """x [T, n] f32 or bf16 -> (e4m3 [T, n], scales f32 [T, ceil(n / 128)])."""
        t = self._t
        stride = self._rows(x, "x", self._float)
        T, n = x.shape
        nb = (n + 127) // 128
        q, sc = t.empty_like(x, dtype=t.float8_e4m3fn), x.new_empty((T, nb), dtype=t.float32)
        self._ck(self._l.fomoe_b200_ops_f8_quantize(self._h, T, n, x.data_ptr(), self._float[x.dtype], stride, q.data_ptr(), q.stride(0),
                                                    sc.data_ptr(), nb, self._stream()), "f8_quantize")
        return q, sc

    def f8_matmul(self, a, a_scales, b, b_scales, *, out="bf16"):
        """a [M, K] e4m3 with scales [M, ceil(K / 128)], b [N, K] with scales [ceil(N / 128), ceil(K / 128)] -> a b^T [M, N]."""
        if out not in self._out:
            raise ValueError(f"out: 'f32' or 'bf16' is wanted, got {out!r}")
        sa, sb = self._rows(a, "a", self._f8), self._rows(b, "b", self._f8)
        (M, K), (N, bk) = a.shape, b.shape
        if bk != K:
            raise ValueError(f"a has {K} columns, b has {bk}")
        nb = (K + 127) // 128
        ss = self._rows(a_scales, "a_scales", self._f32, (M, nb))
        sw = self._rows(b_scales, "b_scales", self._f32, ((N + 127) // 128, nb))
        dt, ty = self._out[out]
        c = a.new_empty((M, N), dtype=dt)
        args = MatmulArgs(M, N, K, a.data_ptr(), sa, a_scales.data_ptr(), ss, b.data_ptr(), sb, b_scales.data_ptr(), sw,
                          c.data_ptr(), ty, N)
        self._ck(self._l.fomoe_b200_ops_f8_matmul(self._h, args, self._stream()), "f8_matmul")
        return c

    def f8_experts(self, x, x_scales, ids, weights, gate_up, gate_up_scales, down, down_scales, *, shared=False,
                   workspace=None):
        """The experts of one layer (see fomoe_b200_ops_f8_experts): x [T, H] e4m3 with scales [T, H / 128], ids int32 and
        weights f32 [T, k], gate_up [R, 2 I, H], down [R, H, I] with their block scales; R records, the last one shared by
        all tokens if `shared`.  -> bf16 [T, H].  workspace: a uint8 tensor to use instead of one from torch's allocator
        (at least f8_experts_workspace bytes); calls that may overlap need their own."""
        t, s = self._t, 1 if shared else 0
        xs = self._rows(x, "x", self._f8)
        T, H = x.shape
        R, I2 = gate_up.shape[:2]
        I = I2 // 2
        k = ids.shape[1] if ids.dim() == 2 else 0
        if (R | I2 | k) >> 31:
            raise ValueError(f"records, rows of a record and slots: less than 2^31 are taken, got {(R, I2, k)}")
        if H % 128 or I2 % 256:
            raise ValueError(f"hidden size {H} and intermediate size {I2} / 2: multiples of 128 are wanted")
        hb, ib = H // 128, I // 128
        ss = self._rows(x_scales, "x_scales", self._f32, (T, hb))
        out = x.new_empty((T, H), dtype=t.bfloat16)
        args = ExpertsArgs(T, H, I, R - s, k, s, x.data_ptr(), xs, x_scales.data_ptr(), ss,
                           self._flat(ids, "ids", self._i32, (T, k)), self._flat(weights, "weights", self._f32, (T, k)),
                           self._flat(gate_up, "gate_up", self._f8, (R, I2, H)),
                           self._flat(gate_up_scales, "gate_up_scales", self._f32, (R, 2 * ib, hb)),
                           self._flat(down, "down", self._f8, (R, H, I)),
                           self._flat(down_scales, "down_scales", self._f32, (R, hb, ib)), out.data_ptr(), H)
        if workspace is None:
            size = self._l.fomoe_b200_ops_f8_experts_workspace(args)
            workspace = x.new_empty((size,), dtype=t.uint8)
        else:
            if workspace.get_device() != self.device or not workspace.is_contiguous():
                raise ValueError("workspace: a contiguous tensor on the handle's device is wanted")
            size = workspace.numel() * workspace.element_size()
        self._ck(self._l.fomoe_b200_ops_f8_experts(self._h, args, workspace.data_ptr(), size, self._stream()), "f8_experts")
        return out

    def f8_experts_workspace(self, n_tokens, n_embd, n_inter, n_experts, top_k, shared=False):
        """Bytes of workspace a call of f8_experts of these sizes needs (0: sizes that it refuses)."""
        if (n_tokens | n_embd | n_inter | n_experts | top_k) >> 31:
            return 0
        return int(self._l.fomoe_b200_ops_f8_experts_workspace(
            ExpertsArgs(n_tokens, n_embd, n_inter, n_experts, top_k, int(bool(shared)))))
