"""Key / value cache in 4 or 8 bits (csrc/me_kvq.hip): rows are quantised as they are written, attended to as they lie, and
can be read back.

A row (one token, one head) of head_dim values is held as 4-bit e2m1 or 8-bit e4m3 codes and one bfloat16 scale (amax / 6 or amax / 448,
cut to bfloat16): 34 or 66 bytes at head_dim 64 against 128 in bf16.  The codes lie in the order in which the matrix instructions take
them (include/midiemo.h describes it), 32 tokens to a block.  The decode step this serves: generate.py:92-122 of the
reference, made incremental; the attention is music_multi.py:211-235 for one query row."""
import torch

from . import ops

HEAD_DIMS = (32, 48, 64)
BLOCK = 32


def _need(ok, what):
    if not ok:
        raise RuntimeError("kv cache: " + what)


class QuantKVCache:
    """Cache of `batch` sequences, `heads` heads, at least `max_len` tokens (rounded up to blocks of 32).

    Positions (`pos` below) are a whole number, or an int32 device tensor of one value or one per sequence; those are read on the
    device (so a captured step can advance them), and what has no place is then left out instead of refused: rows past the cache's end,
    and a whole sequence whose position is negative or past the end.  Calls only enqueue work on the current stream of the
    cache's device.  None of them is differentiable: results carry no gradient."""

    def __init__(self, batch, heads, max_len, head_dim, bits=4, device="cuda"):
        _need(batch > 0 and heads > 0 and max_len > 0, "batch, heads and max_len must be positive")
        _need(head_dim in HEAD_DIMS and bits in (4, 8), "head_dim must be 32, 48 or 64 and bits 4 or 8 (got %r, %r)" % (head_dim, bits))
        blocks = -(-int(max_len) // BLOCK)
        z = lambda *s, dtype: torch.zeros(*s, dtype=dtype, device=device)
        size = BLOCK * head_dim * bits // 8
        self._set(z(batch, heads, blocks, size, dtype=torch.uint8), z(batch, heads, blocks * BLOCK, dtype=torch.bfloat16),
                  z(batch, heads, blocks, size, dtype=torch.uint8), z(batch, heads, blocks * BLOCK, dtype=torch.bfloat16), head_dim, bits)

    @classmethod
    def wrap(cls, k, k_scale, v, v_scale, head_dim, bits):
        """A cache over existing tensors: codes uint8 [B, H, blocks, 32 * head_dim * bits / 8], 16-byte aligned, and
        scales bfloat16 [B, H, blocks * 32]; none of them needs to be cleared before rows are written."""
        self = cls.__new__(cls)
        _need(head_dim in HEAD_DIMS and bits in (4, 8), "head_dim must be 32, 48 or 64 and bits 4 or 8 (got %r, %r)" % (head_dim, bits))
        _need(k.dim() == 4 and all(x > 0 for x in k.shape) and k.shape[3] == BLOCK * head_dim * bits // 8, "codes must be [B, H, blocks, %d], got %s" % (BLOCK * head_dim * bits // 8, tuple(k.shape)))
        for t, shape, dtype in ((k, k.shape, torch.uint8), (v, k.shape, torch.uint8), (k_scale, (*k.shape[:2], k.shape[2] * BLOCK), torch.bfloat16),
                                (v_scale, (*k.shape[:2], k.shape[2] * BLOCK), torch.bfloat16)):
            _need(t.shape == shape and t.dtype == dtype and t.is_contiguous() and t.device == k.device, "codes and scales must be contiguous tensors of matching shapes and types on one device")
        self._set(k, k_scale, v, v_scale, head_dim, bits)
        return self

    def _set(self, k, k_scale, v, v_scale, head_dim, bits):
        self.k, self.k_scale, self.v, self.v_scale = k, k_scale, v, v_scale
        self.batch, self.heads, self.head_dim, self.bits = k.shape[0], k.shape[1], head_dim, bits
        self.max_len = k.shape[2] * BLOCK
        self.device = k.device
        self.nbytes = 2 * (k.numel() + 2 * k_scale.numel())
        self._index = k.device.index
        # layouts (shapes, strides, types, devices: never addresses) that have passed the checks, with what the C call takes of them; a
        # decode loop makes the same calls again and again, and checks and arguments cost more host time than the launch
        self._seen = {}
        self.ref = ops.kvq_cache(k, k_scale, v, v_scale, head_dim, bits) if k.device.type == "cuda" else None

    # -------------------------------------------------------------- checks
    def _passed(self, key, check, *tensors):
        """check(*tensors) the first time a layout comes; what it returned"""
        value = self._seen.get(key)
        if value is None:
            for t in tensors:
                if t is not None and t.device != self.device:
                    _need(False, "a tensor is on %s, the cache on %s" % (t.device, self.device))
            value = check(*tensors)
            if len(self._seen) >= 256:
                self._seen.clear()
            self._seen[key] = value
        return value

    def _pos(self, pos, n, first=0):
        """(t, t_dev, ld_t) of a position for n rows"""
        if isinstance(pos, torch.Tensor):
            if not (pos.dtype is torch.int32 and pos.is_contiguous() and pos.numel() in (1, self.batch) and pos.device == self.device):
                _need(False, "a position tensor must be int32 with 1 or %d values on %s" % (self.batch, self.device))
            return 0, pos.data_ptr(), 1 if pos.numel() > 1 else 0
        if not (first <= pos and pos + n <= self.max_len):
            _need(False, "positions %d..%d do not fit %d tokens" % (pos, pos + n - 1, self.max_len))
        return int(pos), None, 0

    def _lens(self, lens):
        if lens is None:
            return None
        if not (lens.dtype is torch.int32 and lens.shape == (self.batch,) and lens.is_contiguous() and lens.device == self.device):
            _need(False, "lens must be int32 [%d] on %s" % (self.batch, self.device))
        return lens.data_ptr()

    def _check_rows(self, k, v):
        for x in (k, v):
            _need(x.dim() == 4 and x.shape == k.shape and x.shape[0] == self.batch and x.shape[2:] == (self.heads, self.head_dim) and x.dtype == k.dtype and
                  (x.stride(3) == 1 or x.numel() == 0), "rows must be [%d, n, %d, %d] with the last dimension contiguous, got %s" % (self.batch, self.heads, self.head_dim, tuple(x.shape)))
        _need(k.shape[1] <= self.max_len, "%d rows do not fit %d tokens" % (k.shape[1], self.max_len))
        return k.shape[1], ops.kvq_strides(k, v), ops._code(k.dtype)

    def _check_new(self, q, k, v):
        # a dimension of one entry has no stride of its own: torch leaves any number there, also in what it calls contiguous
        step = lambda x: tuple(d if n == 1 else s for s, n, d in zip(x.stride(), x.shape, (self.heads * self.head_dim, self.head_dim, 1)))
        for x in (k, v):
            _need(x.shape == (self.batch, self.heads, self.head_dim) and x.dtype == q.dtype and step(x) == step(k) and x.stride(2) == 1,
                  "new rows must be [%d, %d, %d] of q's type with equal strides and the last dimension contiguous, got %s" % (self.batch, self.heads, self.head_dim, tuple(x.shape)))
        return step(k)[:2]

    def _check_attend(self, q, rel, key_pad, out):
        _need(q.dim() == 3 and q.shape == (self.batch, self.heads, self.head_dim) and q.stride(2) == 1, "q must be [%d, %d, %d] with the last dimension contiguous, got %s" % (self.batch, self.heads, self.head_dim, tuple(q.shape)))
        if rel is not None:
            _need(rel.dim() == 2 and rel.shape[1] == self.head_dim and rel.shape[0] >= self.max_len and rel.is_contiguous() and rel.dtype == q.dtype,
                  "rel must be a contiguous [>= %d, %d] table of q's type" % (self.max_len, self.head_dim))
        if key_pad is not None:
            _need(key_pad.dtype == torch.uint8 and key_pad.dim() == 2 and key_pad.shape[0] == self.batch and key_pad.is_contiguous(),
                  "key_pad must be contiguous uint8 or bool [%d, n]" % self.batch)
        if out is not None:
            _need(out.shape == q.shape and out.dtype == q.dtype and out.stride(2) == 1 and all(s != 0 or x == 1 for s, x in zip(out.stride(), out.shape)), "out must match q")
        o = out.stride()[:2] if out is not None else (self.heads * self.head_dim, self.head_dim)
        return q.stride()[:2], o, rel.shape[0] if rel is not None else 0, key_pad.shape[1] if key_pad is not None else 0, ops._code(q.dtype)

    def _elsewhere(self):
        """the cache's device is not the current one"""
        if self.ref is None:
            _need(False, "it is on %s -- there is no CPU path" % self.device)
        return torch._C._cuda_getDevice() != self._index

    # -------------------------------------------------------------- calls
    def write(self, k, v, pos, lens=None):
        """Quantise k, v [B, n, H, head_dim] (float32, bfloat16 or float16; any strides, last dimension contiguous) into positions pos .. pos + n - 1;
        with lens (int32 [B]) only the first lens[b] rows of sequence b.  Everything else in the cache stays as it was."""
        self._rows("me_kvq_write", k, v, pos, lens)

    def read(self, pos, n, dtype=torch.float32, lens=None):
        """The rows at positions pos .. pos + n - 1 as (k, v) [B, n, H, head_dim] of `dtype`; rows from lens[b] on are zeros."""
        if not 0 <= n <= self.max_len:
            _need(False, "%r rows do not fit %d tokens" % (n, self.max_len))
        k = torch.empty(self.batch, n, self.heads, self.head_dim, dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        self._rows("me_kvq_read", k, v, pos, lens)
        return k, v

    def _rows(self, call, k, v, pos, lens):
        key = (k.shape, k.stride(), k.dtype, k.device, v.shape, v.stride(), v.dtype, v.device)
        n, strides, code = self._seen.get(key) or self._passed(key, self._check_rows, k, v)
        t, t_dev, ld_t = self._pos(pos, n)
        first = self._lens(lens)
        if n == 0:
            return
        if self._elsewhere():
            with torch.cuda.device(self._index):
                return self._rows(call, k, v, pos, lens)
        ops.check(getattr(ops.lib(), call)(self.ref, k.data_ptr(), v.data_ptr(), strides, n, t, t_dev, ld_t, first, code,
                                           torch._C._cuda_getCurrentRawStream(self._index)), call)

    def append_attend(self, q, k, v, pos, rel=None, key_pad=None, out=None, nsplit=0):
        """A decode step in one launch: write the rows k, v [B, H, head_dim] at pos, then attend to the keys 0 .. pos.  k and v are of q's type with
        equal strides, their rows 16-byte aligned."""
        key = (q.dtype, k.shape, k.stride(), k.dtype, k.device, v.shape, v.stride(), v.dtype, v.device)
        strides = self._seen.get(key) or self._passed(key, self._check_new, q, k, v)
        self._pos(pos, 1)
        return self.attend(q, pos, rel, key_pad, out, nsplit, (k, v, strides))

    def attend(self, q, pos, rel=None, key_pad=None, out=None, nsplit=0, _new=None):
        """softmax((q.k_j + q.rel[M-1-(pos-j)]) / sqrt(head_dim)) v over the cached keys j = 0 .. pos (pos = -1: none).

        q [B, H, head_dim]; rel [M, head_dim] of q's type with M >= max_len (the model's relative table) or None; key_pad uint8 / bool
        [B, n], 1 = masked key (a position tensor may pass n: keys from n on are not masked).  A row without a key gives zeros.  nsplit: key ranges that run side by side (0: chosen from the sizes)."""
        if key_pad is not None and key_pad.dtype is torch.bool:
            key_pad = key_pad.view(torch.uint8)
        key = (q.shape, q.stride(), q.dtype, q.device, rel is not None and (rel.shape, rel.stride(), rel.dtype, rel.device),
               key_pad is not None and (key_pad.shape, key_pad.stride(), key_pad.dtype, key_pad.device), out is not None and (out.shape, out.stride(), out.dtype, out.device))
        (qb, qh), (ob, oh), M, width, code = self._seen.get(key) or self._passed(key, self._check_attend, q, rel, key_pad, out)
        t, t_dev, ld_t = self._pos(pos, 1 if isinstance(pos, torch.Tensor) or pos >= 0 else 0, -1)
        tokens = self.max_len
        if t_dev is None:
            tokens = max(t + 1, 1)
            if key_pad is not None and width <= t:
                _need(False, "key_pad is narrower than the %d keys" % (t + 1))
        if not 0 <= nsplit <= 64:
            _need(False, "nsplit must be 0..64")
        if self._elsewhere():
            with torch.cuda.device(self._index):
                return self.attend(q, pos, rel, key_pad, out, nsplit, _new)
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        ns = nsplit or self._splits(tokens, rel is not None)
        size, part = 0, None
        if ns > 1:
            # the records of this call: from the caching allocator, so calls on two streams or in two captured graphs never share them
            size = self.batch * self.heads * ns * (self.head_dim + 4) * 4
            part = torch.empty(size, dtype=torch.uint8, device=self.device)
        tail = (rel.data_ptr() if M else None, M, key_pad.data_ptr() if key_pad is not None else None, width, out.data_ptr(), ob, oh,
                part.data_ptr() if size else None, size, ns, t, t_dev, ld_t, code, torch._C._cuda_getCurrentRawStream(self._index))
        if _new is None:
            ops.check(ops.lib().me_kvq_attn(self.ref, q.data_ptr(), qb, qh, *tail), "me_kvq_attn")
        else:
            k, v, (nb, nh) = _new
            ops.check(ops.lib().me_kvq_append_attn(self.ref, q.data_ptr(), qb, qh, k.data_ptr(), v.data_ptr(), nb, nh, *tail), "me_kvq_append_attn")
        return out

    def _splits(self, tokens, rel):
        key = (tokens, rel)
        value = self._seen.get(key)
        if value is None:
            if len(self._seen) >= 256:
                self._seen.clear()
            value = self._seen[key] = ops.kvq_splits(self.batch, self.heads, tokens, rel)
        return value
