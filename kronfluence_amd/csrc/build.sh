#!/usr/bin/env bash
# Builds libkronfluence_hip.so for gfx950 in-tree (the .so travels to the GPU box with the snapshot).
set -euo pipefail
here="$(cd "$(dirname "${BASH_SOURCE[0]}")" && pwd)"
out="${here}/../libkronfluence_hip.so"
HIPCC="${HIPCC:-/opt/rocm/bin/hipcc}"
# -packed-fp32-ops: no v_pk_{add,mul,fma}_f32 from ordinary float code (some of their forms have returned wrong results on this
# hardware now and then); hipcc's host pass does not know the feature and says so
flags=(--offload-arch=gfx950 -O3 -std=c++17 -fPIC -munsafe-fp-atomics -Wall -Wno-unused-function
       -Xclang -target-feature -Xclang -packed-fp32-ops)
mkdir -p "${here}/obj"
pids=()
units=(kf_kernels kf_eigh kf_score_v2 kf_attention kf_norm)
for src in "${units[@]}"; do
  stale=0
  [[ -f "${here}/obj/${src}.o" ]] || stale=1
  for dep in "${here}/${src}.hip" "${here}"/*.h "${here}/../../include/kronfluence_hip.h"; do
    [[ "${dep}" -nt "${here}/obj/${src}.o" ]] && stale=1
  done
  if [[ ${stale} -eq 1 ]]; then
    "${HIPCC}" "${flags[@]}" -c "${here}/${src}.hip" -o "${here}/obj/${src}.o" &
    pids+=($!)
  fi
done
for p in "${pids[@]:-}"; do [[ -n "${p}" ]] && wait "${p}"; done
objects=("${units[@]/#/${here}/obj/}")
objects=("${objects[@]/%/.o}")
"${HIPCC}" --offload-arch=gfx950 -shared -fPIC "${objects[@]}" -o "${out}"
echo "built ${out}"

# the autograd nodes over the C ABI (host code: no device code is in it)
ext="${here}/../_autograd.so"
stale=0
for dep in "${here}/kf_autograd.cpp" "${here}/../../include/kronfluence_hip.h" "${here}/build.sh"; do [[ "${dep}" -nt "${ext}" ]] && stale=1; done
if [[ ! -f "${ext}" || ${stale} -eq 1 ]]; then
  read -r torch_dir python_include cxx11 < <(python3 -c 'import os, sysconfig, torch
print(os.path.dirname(torch.__file__), sysconfig.get_paths()["include"], int(torch._C._GLIBCXX_USE_CXX11_ABI))')
  "${CXX:-g++}" -O2 -std=c++17 -fPIC -shared -Wall -D_GLIBCXX_USE_CXX11_ABI="${cxx11}" -D__HIP_PLATFORM_AMD__=1 -DUSE_ROCM=1 \
    -I"${torch_dir}/include" -I"${torch_dir}/include/torch/csrc/api/include" -I"${python_include}" -I"${ROCM_PATH:-/opt/rocm}/include" \
    "${here}/kf_autograd.cpp" -o "${ext}" -L"${torch_dir}/lib" -ltorch_python -ltorch_cpu -lc10 -lc10_hip \
    -L"${here}/.." -l:libkronfluence_hip.so -Wl,-rpath,'$ORIGIN'
fi
echo "built ${ext}"
