"""ctypes binding of ``libtfpp_hip.so`` (C ABI declared in include/tfpp.h).

The binding is generated from the header at import time, so the Python side cannot drift from the declared
ABI; struct mirrors are verified against ``tfpp_struct_sizes``.  There is NO fallback: if the library is missing
or fails to load, every op raises (the product path never routes through PyTorch ATen kernels or the CPU oracle).
"""
import ctypes
import os
import re
import subprocess
import threading

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG_DIR)
HEADER = os.path.join(ROOT, 'include', 'tfpp.h')
CSRC = os.path.join(PKG_DIR, 'csrc')
LIB_PATH = os.path.join(PKG_DIR, 'libtfpp_hip.so')
SOURCES = ['gemm_kernels.hip', 'gemm_glds.hip', 'gemm_wgrad_glds.hip', 'attention_kernels.hip', 'conv3x3_halo.hip', 'wgrad3x3_halo.hip', 'pointwise_kernels.hip', 'norm_kernels.hip', 'bn_rows_kernels.hip', 'misc_kernels.hip', 'lidar_kernels.hip', 'swin_kernels.hip', 'bev_kernels.hip', 'head_kernels.hip', 'augment_kernels.hip', 'grad_clip.hip', 'block_norm.hip', 'diff_attention.hip']

F32, BF16 = 0, 1
ABI_VERSION = 10  # include/tfpp.h TFPP_ABI_VERSION
ACT_NONE, ACT_RELU, ACT_SIGMOID, ACT_GELU, ACT_TANH = 0, 1, 2, 3, 4
EINVAL = -1000

i32, i64, f32, vp = ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_void_p


class BnRows(ctypes.Structure):
  """tfpp_bn_rows: BatchNorm statistics still in the per-M-tile rows of the producing convolution (include/tfpp.h)"""
  _fields_ = [('partial', vp), ('nrows', i32), ('C', i32), ('count', i64), ('gamma', vp), ('beta', vp), ('running_mean', vp), ('running_var', vp),
              ('num_batches_tracked', vp), ('scale', vp), ('shift', vp), ('save_mean', vp), ('save_invstd', vp), ('momentum', f32), ('eps', f32)]


class ConvParams(ctypes.Structure):
  _fields_ = [('src', vp), ('w', vp), ('dst', vp), ('scale', vp), ('shift', vp), ('res', vp), ('B', i32), ('Hs', i32),
              ('Ws', i32), ('Cs', i32), ('Hd', i32), ('Wd', i32), ('Cd', i32), ('R', i32), ('S', i32), ('stride', i32),
              ('pad', i32), ('G', i32), ('ks_g', i32), ('n_g', i32), ('mode', i32), ('act', i32), ('dst_nchw', i32),
              ('alpha', f32), ('src_ld', i64), ('dst_ld', i64), ('res_ld', i64), ('dst_f32', i32), ('stats_partial', vp), ('stats_rows', i32), ('stats_store', i32), ('splitk_ws', vp),
              ('splitk_ws_floats', i64), ('splitk', i32), ('bns_y', vp), ('bns_x', vp), ('bns_mean', vp), ('bns_invstd', vp),
              ('bns_partial', vp), ('bns_ld', i64), ('bns_relu', i32), ('in_bn', BnRows), ('in_relu', i32), ('relu_mask', vp), ('relu_mask_ld', i64)]


class WgradParams(ctypes.Structure):
  _fields_ = [('dy', vp), ('x', vp), ('dw', vp), ('row_map', vp), ('col_map', vp), ('B', i32), ('Hs', i32), ('Ws', i32),
              ('Cs', i32), ('Hd', i32), ('Wd', i32), ('Cd', i32), ('R', i32), ('S', i32), ('stride', i32), ('pad', i32),
              ('G', i32), ('ks_g', i32), ('n_g', i32), ('c_real', i32), ('splits', i32), ('x_ld', i64), ('dy_ld', i64),
              ('dw_ld', i64), ('ws', vp), ('ws_floats', i64), ('x_scale', vp), ('x_shift', vp), ('x_relu', i32)]


class BgemmParams(ctypes.Structure):
  _fields_ = [('A', vp), ('B', vp), ('C', vp), ('bias', vp), ('M', i32), ('N', i32), ('K', i32), ('lda', i64),
              ('ldb', i64), ('ldc', i64), ('a_bs0', i64), ('a_bs1', i64), ('b_bs0', i64), ('b_bs1', i64), ('c_bs0', i64),
              ('c_bs1', i64), ('batch0', i32), ('batch1', i32), ('a_km', i32), ('b_km', i32), ('act', i32), ('c_f32', i32),
              ('alpha', f32), ('beta', f32)]


class AttnParams(ctypes.Structure):
  _fields_ = [('q', vp), ('k', vp), ('v', vp), ('o', vp), ('lse', vp), ('d_o', vp), ('dq', vp), ('dk', vp), ('dv', vp), ('delta', vp),
              ('debug_p', vp), ('B', i32), ('nh', i32), ('T', i32), ('d', i32), ('ld_q', i64), ('ld_kv', i64), ('ld_o', i64),
              ('scale', f32), ('p_drop', f32), ('seed', ctypes.c_uint64), ('seed_offset', vp), ('bias', vp), ('mask', vp), ('p_out', vp),
              ('n_mask', i32), ('ld_b', i64), ('ld_p', i64)]


class PackDesc(ctypes.Structure):
  _fields_ = [('src', vp), ('dst', vp), ('row_map', vp), ('col_map', vp), ('total', i64), ('in_ld', i64), ('out_ld', i64),
              ('blk_start', i64), ('kind', i32), ('dtype', i32), ('a', i32 * 8)]


class BlockNormParams(ctypes.Structure):
  _fields_ = [(n, vp) for n in ('x', 'a', 'gate', 'post_w', 'post_b', 'pre_w', 'pre_b', 'scale', 'y', 'h', 'stat', 'dy', 'dh', 'dx', 'da', 'dgate', 'dpost_w',
                                'dpost_b', 'dpre_w', 'dpre_b', 'dscale', 'partial')] + \
      [(n, i64) for n in ('ld_x', 'ld_a', 'ld_g', 'ld_dy', 'ld_dh')] + \
      [(n, i32) for n in ('B', 'T', 'C', 'layer', 'post', 'pre', 'gate_mode', 'gate_act', 'accumulate')] + [('alpha', f32), ('eps', f32)]


class DiffAttnParams(ctypes.Structure):
  _fields_ = [(n, vp) for n in ('q', 'k', 'v', 'lam', 'norm_w', 'out', 'o1', 'o2', 'lse', 'kv_len', 'q_start', 'key_mask', 'dout', 'd_o', 'slope', 'delta', 'partial', 'dlam',
                                'dnorm_w', 'dq_out', 'dk_out', 'dv_out')] + \
      [('ld_mask', i64), ('q_s', i64 * 4), ('k_s', i64 * 4), ('v_s', i64 * 3), ('o_s', i64 * 3), ('do_s', i64 * 3), ('dq_s', i64 * 4), ('dk_s', i64 * 4), ('dv_s', i64 * 3)] + \
      [(n, i32) for n in ('B', 'H', 'Hkv', 'Tq', 'Tk', 'd', 'dv', 'n_lam', 'norm', 'norm_w_bf16', 'causal', 'q_start_all', 'out_vec', 'do_vec', 'dq_vec', 'dk_vec', 'dv_vec', 'splits', 'dkv_splits')] + \
      [('scale', f32), ('out_scale', f32), ('eps', f32), ('dkv', vp)]


_CTYPE = {'int': i32, 'int32_t': i32, 'int64_t': i64, 'uint64_t': ctypes.c_uint64, 'uint32_t': ctypes.c_uint32, 'float': f32, 'double': ctypes.c_double}


def declared_functions(header=HEADER):
  """{name: [ctypes argtypes]} parsed from the ``int tfpp_*(...)`` declarations of include/tfpp.h."""
  with open(header, encoding='utf-8') as f:
    text = f.read()
  text = re.sub(r'/\*.*?\*/', '', text, flags=re.S)
  out = {}
  for m in re.finditer(r'\bint\s+(tfpp_\w+)\s*\(([^)]*)\)\s*;', text):
    name, args = m.group(1), m.group(2).strip()
    types = []
    if args and args != 'void':
      for a in args.split(','):
        a = a.strip()
        if '*' in a:
          types.append(vp)
        else:
          t = a.replace('const', '').split()[0]
          types.append(_CTYPE[t])
    out[name] = types
  return out


def source_hash():
  """64-bit hash over the kernel sources and the ABI header (file names + contents): compiled into the library by build() and
  compared by load(), so the binary under test is always the one these sources produce."""
  import hashlib
  h = hashlib.sha256()
  files = sorted(f for f in os.listdir(CSRC) if f.endswith(('.hip', '.h')))
  h.update(' '.join(HIPCC_FLAGS).encode() + b'\0')  # a library built with other flags is another library
  for path in [os.path.join(CSRC, f) for f in files] + [HEADER]:
    h.update(os.path.basename(path).encode() + b'\0')
    with open(path, 'rb') as f:
      h.update(f.read())
    h.update(b'\0')
  return int(h.hexdigest()[:16], 16)


# Compile flags of every kernel source.  -fno-slp-vectorize -fno-vectorize: no packed-FP32 VALU instructions (v_pk_fma_f32 / v_pk_add_f32 /
# v_pk_mul_f32).  Round 3 traced the "result depends on the co-runner" issue of round 2 to them: in layernorm_bwd_kernel the SLP vectorizer
# turned the two row sums into packed operations with op_sel lane swaps, and waves of that kernel that shared their CU with the persistent
# MFMA / LDS-transpose weight-gradient kernel returned a wrong sum c1 in ~2 % of the rows (tools/replay_bisect.py), the
# scalar code never does.  tests/test_kernel_resources.py fails the CPU suite if a packed FP32 instruction reappears in any kernel.
# -packed-fp32-ops takes the instructions away from the back end as well, which can still form them from scalar code.
HIPCC_FLAGS = ['--offload-arch=gfx950', '-O3', '-std=c++17', '-fno-slp-vectorize', '-fno-vectorize', '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops']
EXTRA_FLAGS = os.environ.get('TFPP_BUILD_FLAGS', '').split()  # experiments only (build(force=True)); the product build has none
HASH_PATH = LIB_PATH + '.srchash'  # written by build() next to the library (reading the embedded hash would dlopen the old binary)


def built_hash():
  """Source hash of the library on disk according to build()'s sidecar file (None: no library / no sidecar).  The authoritative
  check is load(), which reads the hash compiled into the binary."""
  if not (os.path.exists(LIB_PATH) and os.path.exists(HASH_PATH)):
    return None
  try:
    with open(HASH_PATH, encoding='utf-8') as f:
      return int(f.read().strip(), 16)
  except (OSError, ValueError):
    return None


def build(verbose=False, force=False):
  """Compile every HIP source for gfx950 into carla_garage_amd/libtfpp_hip.so (hipcc cross-compiles without a GPU)."""
  srcs = [os.path.join(CSRC, s) for s in SOURCES]
  want = source_hash()
  if not force and built_hash() == want:
    return LIB_PATH
  objs = []
  procs = []
  os.makedirs(os.path.join(PKG_DIR, 'build'), exist_ok=True)
  for s in srcs:
    o = os.path.join(PKG_DIR, 'build', os.path.basename(s) + '.o')
    objs.append(o)
    cmd = ['hipcc'] + HIPCC_FLAGS + ['-fPIC', f'-DTFPP_SOURCE_HASH=0x{want:016x}ULL'] + EXTRA_FLAGS + ['-c', s, '-o', o]
    procs.append((cmd, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
  for cmd, p in procs:
    outp = p.communicate()[0].decode()
    if p.returncode != 0:
      raise RuntimeError('hipcc failed: ' + ' '.join(cmd) + '\n' + outp)
    if verbose and outp:
      print(outp)
  cmd = ['hipcc', '--offload-arch=gfx950', '-shared', '-fPIC', '-o', LIB_PATH] + objs
  r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, check=False)
  if r.returncode != 0:
    raise RuntimeError('link failed: ' + r.stdout.decode())
  with open(HASH_PATH, 'w', encoding='utf-8') as f:
    f.write(f'{want:016x}\n')
  return LIB_PATH


class TfppError(RuntimeError):
  pass


class KernelProfiler:
  """Brackets every library call with HIP events on the launch stream (torch's current stream) and aggregates the
  elapsed time per kernel family; ``tag()`` lets ops.py attach a family name and algorithmic FLOPs to the next call."""

  def __init__(self):
    import torch
    self._torch = torch
    self.records = []
    self._pending = None

  def tag(self, family, flops=0.0, nbytes=0.0, group=None):
    """group: a set of LAYERS (whatever kernel runs them), e.g. 'fusion_linears' -- the north-star GEMMs are priced by layer, not by kernel name"""
    self._pending = (family, float(flops), float(nbytes), group)

  def run(self, name, fn, args):
    fam, flops, nbytes, group = self._pending if self._pending is not None else (name, 0.0, 0.0, None)
    self._pending = None
    e0 = self._torch.cuda.Event(enable_timing=True)
    e1 = self._torch.cuda.Event(enable_timing=True)
    e0.record()
    rc = fn(*args)
    e1.record()
    self.records.append((fam, flops, nbytes, e0, e1, group))
    return rc

  def summary(self, by_group=False):
    self._torch.cuda.synchronize()
    agg = {}
    for fam, flops, nbytes, e0, e1, group in self.records:
      keys = (group if isinstance(group, (tuple, list)) else (group,)) if by_group else (fam,)
      ms = e0.elapsed_time(e1)
      for key in keys:
        if key is None:
          continue
        a = agg.setdefault(key, dict(calls=0, ms=0.0, flops=0.0, bytes=0.0, kernels={}))
        a['calls'] += 1
        a['ms'] += ms
        a['flops'] += flops
        a['bytes'] += nbytes
        a['kernels'][fam] = a['kernels'].get(fam, 0) + 1
    return agg


class _Lib:
  """Lazy handle; ``lib.tfpp_xxx(...)`` raises TfppError on a non-zero return code."""

  def __init__(self):
    self._dll = None
    self._fns = {}
    self._loading = threading.Lock()
    self.profiler = None

  def raw(self, name):
    """The bare ctypes function (for entry points whose return value is data, not an error code)."""
    self.load()
    return self._fns[name]

  def load(self):
    if self._dll is None:
      with self._loading:  # (threads whose first calls come together: one loads, the others wait)
        if self._dll is None:
          self._load()
    return self

  def _load(self):
    if not os.path.exists(LIB_PATH):
      raise TfppError(f'{LIB_PATH} is missing: run `python -c "import __graft_entry__ as g; g.build()"` '
                      '(there is no PyTorch/CPU fallback for the HIP path)')
    # torch first: its wheel carries its own libamdhip64, and the library must bind to THAT copy of the HIP runtime (same SONAME: the loader
    # reuses what is already mapped).  Loaded before torch, libtfpp_hip.so pulls in /opt/rocm's copy, the process ends up with two runtimes and
    # every launch of this library fails with hipErrorNoDevice once torch has opened the device (seen with build() and smoke() in one process).
    import torch  # noqa: F401
    dll, fns = ctypes.CDLL(LIB_PATH), {}
    for name, argtypes in declared_functions().items():
      fn = getattr(dll, name)  # AttributeError if the library does not export a declared symbol
      fn.argtypes = argtypes
      fn.restype = ctypes.c_int
      fns[name] = fn
    sizes = (ctypes.c_int * 8)()
    n = dll.tfpp_struct_sizes(sizes, 8)
    mine = [ctypes.sizeof(ConvParams), ctypes.sizeof(WgradParams), ctypes.sizeof(BgemmParams), ctypes.sizeof(PackDesc),
            ctypes.sizeof(AttnParams)]
    mine.append(ctypes.sizeof(BnRows))
    mine.append(ctypes.sizeof(BlockNormParams))
    mine.append(ctypes.sizeof(DiffAttnParams))
    if n != len(mine) or list(sizes[:n]) != mine:
      raise TfppError(f'struct layout mismatch: library {list(sizes[:n])} vs ctypes {mine}')
    if dll.tfpp_version() != ABI_VERSION:
      raise TfppError(f'ABI version mismatch: library {dll.tfpp_version()}, binding {ABI_VERSION} (include/tfpp.h TFPP_ABI_VERSION: bumped with every signature change)')
    got = ctypes.c_uint64(0)
    fns['tfpp_source_hash'](ctypes.byref(got))
    if os.environ.get('TFPP_SKIP_HASH_CHECK', '0') != '1' and int(got.value) != source_hash():
      raise TfppError(f'{LIB_PATH} was built from other sources (hash {int(got.value):016x}, sources {source_hash():016x}): '
                      'rebuild with `python -c "import __graft_entry__ as g; g.build()"`')
    self._fns, self._dll = fns, dll  # (complete and checked: a load that raised has left nothing that a second call would take for a loaded library)

  def __getattr__(self, name):
    if name.startswith('_'):
      raise AttributeError(name)
    self.load()
    fn = self._fns[name]

    def call(*args):
      prof = self.__dict__.get('profiler')
      rc = fn(*args) if prof is None else prof.run(name, fn, args)
      if rc != 0:
        raise TfppError(f'{name} failed with code {rc}' + (' (invalid argument)' if rc == EINVAL else ' (hipError)'))

    call.__name__ = name
    self.__dict__[name] = call
    return call


lib = _Lib()
