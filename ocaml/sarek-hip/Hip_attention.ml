(* ctypes-foreign stubs for the operators on a paged cache (include/sarek_hip.h): rotary positions, the cache that tokens are
   appended to, attention over it.  Conventions and library as in Hip_bindings; lengths, starts and pages are device memory. *)
open Ctypes
open Hip_bindings

type rotary_plan
let rotary_plan : rotary_plan structure typ = structure "sarek_hip_rotary_plan"
let rp_turns = field rotary_plan "turns" (ptr uint64_t)
let rp_pairs = field rotary_plan "pairs" int
let rp_interleaved = field rotary_plan "interleaved" int
let rp_amplitude = field rotary_plan "amplitude" float
let () = seal rotary_plan

type kv_cache
let kv_cache : kv_cache structure typ = structure "sarek_hip_kv_cache"
let kc_keys = field kv_cache "keys" (ptr void)
let kc_values = field kv_cache "values" (ptr void)
let kc_page_stride = field kv_cache "page_stride" int64_t
let kc_slot_stride = field kv_cache "slot_stride" int64_t
let kc_head_stride = field kv_cache "head_stride" int64_t
let kc_n_pages = field kv_cache "n_pages" int64_t
let kc_page_size = field kv_cache "page_size" int
let kc_heads = field kv_cache "heads" int
let kc_head_dim = field kv_cache "head_dim" int
let kc_type = field kv_cache "type" int
let () = seal kv_cache

let rotary_turns =
  bind "sarek_hip_rotary_turns" (ptr double @-> ptr uint64_t @-> int @-> returning int)
let rotary =
  bind "sarek_hip_rotary"
    (ptr rotary_plan @-> ptr void @-> int64_t @-> int64_t @-> int @-> ptr void @-> int @-> int
   @-> ptr void @-> int64_t @-> int64_t @-> int64_t @-> int @-> int @-> ptr void @-> returning int)
let kv_append =
  bind "sarek_hip_kv_append"
    (ptr kv_cache @-> ptr void @-> int64_t @-> int64_t @-> ptr void @-> int64_t @-> int64_t
   @-> ptr void @-> int64_t @-> int64_t @-> ptr void @-> int64_t @-> int64_t @-> int
   @-> ptr rotary_plan @-> ptr int @-> int64_t @-> int @-> ptr int @-> ptr int @-> int @-> int64_t
   @-> int64_t @-> ptr void @-> returning int)
let attention_workspace_bytes =
  bind "sarek_hip_attention_workspace_bytes"
    (ptr kv_cache @-> int @-> int @-> int64_t @-> int @-> int64_t @-> returning int64_t)
let attention_paged =
  bind "sarek_hip_attention_paged"
    (ptr kv_cache @-> ptr void @-> int64_t @-> int64_t @-> int @-> ptr void @-> int64_t @-> int64_t
   @-> ptr float @-> ptr int @-> int64_t @-> int @-> ptr int @-> ptr int @-> int @-> int64_t @-> int
   @-> float @-> ptr void @-> int64_t @-> ptr void @-> returning int)
let attention_shared =
  bind "sarek_hip_attention_shared"
    (ptr kv_cache @-> ptr void @-> int64_t @-> int64_t @-> int @-> ptr void @-> int64_t @-> int64_t
   @-> ptr float @-> ptr int @-> int64_t @-> ptr int @-> int64_t @-> int @-> ptr int @-> ptr int
   @-> int @-> int64_t @-> int @-> float @-> ptr void @-> int64_t @-> ptr void @-> returning int)
