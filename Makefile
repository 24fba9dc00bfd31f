# Builds the gfx950 shared library (C ABI) in-tree.  `make` here, on CPU: hipcc cross-compiles.
HIPCC ?= /opt/rocm/bin/hipcc
HIPFLAGS = --offload-arch=gfx950 -O3 -fPIC -shared -std=c++17 -Xclang -target-feature -Xclang -packed-fp32-ops -Wno-unused-value
SRC = mineral_amd/csrc/ppo_capi.hip mineral_amd/csrc/replay.hip mineral_amd/csrc/linear_attention.hip mineral_amd/csrc/group_norm.hip mineral_amd/csrc/linear_act.hip
HDR = mineral_amd/csrc/gemm.hip.h mineral_amd/csrc/chain.hip.h mineral_amd/csrc/wgrad_group.hip.h mineral_amd/csrc/split_bf16.hip.h mineral_amd/csrc/ln_wgrad0.hip.h mineral_amd/csrc/ln_fwd0.hip.h mineral_amd/csrc/ppo_tail.hip.h mineral_amd/csrc/sac_capi.hip.inc mineral_amd/csrc/shac_capi.hip.inc include/mineral_ppo.h include/mineral_replay.h include/mineral_sac.h include/mineral_shac.h
MEMHDR = mineral_amd/csrc/memory_common.hip.h include/mineral_memory.h include/mineral_ppo.h
OBJDIR = mineral_amd/csrc/build
OBJ = $(patsubst mineral_amd/csrc/%.hip,$(OBJDIR)/%.o,$(SRC))
LIB = mineral_amd/libmineral_ppo.so

# torch.ops.mineral.* of the memory operators: host code over the C ABI, built against the installed torch
TORCH := $(shell python3 -c "import importlib.util as u; print(u.find_spec('torch').submodule_search_locations[0])")
TORCHLIB = mineral_amd/libmineral_torch.so

all: $(LIB) $(TORCHLIB)

$(TORCHLIB): mineral_amd/csrc/torch_ops.cpp include/mineral_memory.h include/mineral_ppo.h $(LIB)
	g++ -O2 -fPIC -shared -std=c++17 -D__HIP_PLATFORM_AMD__=1 -DUSE_ROCM=1 -isystem $(TORCH)/include -isystem $(TORCH)/include/torch/csrc/api/include -isystem /opt/rocm/include $< -o $@ \
	  -Lmineral_amd -l:libmineral_ppo.so -L$(TORCH)/lib -ltorch_cpu -ltorch_hip -lc10 -lc10_hip -Wl,-rpath,'$$ORIGIN'

$(LIB): $(OBJ)
	$(HIPCC) $(HIPFLAGS) $(OBJ) -o $@

$(OBJDIR)/ppo_capi.o $(OBJDIR)/replay.o: $(HDR)
$(OBJDIR)/linear_attention.o $(OBJDIR)/group_norm.o $(OBJDIR)/linear_act.o: $(MEMHDR)
$(OBJDIR)/%.o: mineral_amd/csrc/%.hip Makefile
	@mkdir -p $(OBJDIR)
	$(HIPCC) $(filter-out -shared,$(HIPFLAGS)) -c $< -o $@

# per-kernel register / LDS / spill table
resources: $(SRC) $(HDR) $(MEMHDR)
	$(HIPCC) $(HIPFLAGS) -Rpass-analysis=kernel-resource-usage $(SRC) -o /tmp/_mrl_res.so 2>&1 | python3 tools/resource_table.py

# instrumented diagnostic build (cycle stamps inside the GEMM main loop), see tools/ktrace_run.py
ktrace: $(SRC) $(HDR) $(MEMHDR)
	mkdir -p tools/bin && $(HIPCC) $(HIPFLAGS) -DMRL_KTRACE $(SRC) -o tools/bin/libmineral_ppo_ktrace.so

# the same with the main-loop ablation switches of tools/ktrace_ablate.sh compiled in
ktrace-ablate: $(SRC) $(HDR) $(MEMHDR)
	mkdir -p tools/bin && $(HIPCC) $(HIPFLAGS) -DMRL_KTRACE -DMRL_KTRACE_ABLATE $(SRC) -o tools/bin/libmineral_ppo_ktrace.so

# stand-alone measurement programs (run on the GPU box: tools/bin travels with the tree)
PROBES = mfma_peak_probe mfma_overlap_probe placement_probe bf16x3_split_probe mfma_shape_probe
probes:
	mkdir -p tools/bin && for p in $(PROBES); do $(HIPCC) --offload-arch=gfx950 -O3 -std=c++17 -Xclang -target-feature -Xclang -packed-fp32-ops tools/$$p.hip -o tools/bin/$$p || exit 1; done

clean:
	rm -f $(LIB) $(TORCHLIB) $(OBJ)
.PHONY: all resources ktrace ktrace-ablate probes clean
