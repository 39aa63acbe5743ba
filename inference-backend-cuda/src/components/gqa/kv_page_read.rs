//! KV page read: the rows of chosen tokens gathered from the pages and converted to the model's type, the inverse of
//! `kv_page_write` (cache export, swap-out, a dense prefix for other kernels). Not compiled here; see Cargo.toml.
pub use super::kv_page_write::Config;
use super::kv_page_write::PageTableLayout;
use crate::error::expect_ok;
use crate::ffi;
use crate::metal::{Buffer, CommandRecorder, Device, Operator, ReplayU32};

#[derive(Clone, Copy, Debug, Eq, PartialEq)]
pub struct Shape {
    pub num_total_token_reads: u32,
    pub page_table_layout: PageTableLayout,
}

/// `flat_k` and `flat_v` are written; rows from the active count on stay as they are.
#[derive(Clone, Copy)]
pub struct Buffers<'a> {
    pub pages: &'a Buffer,
    pub flat_k: &'a Buffer,
    pub flat_v: &'a Buffer,
    pub req_slots: &'a Buffer,
    pub flat_token_indices: &'a Buffer,
    pub page_ids: &'a Buffer,
}

pub struct Compute {
    raw: *mut ffi::KhKvPageRead,
}

impl Compute {
    pub fn new(device: &Device, config: Config) -> Self {
        let mut raw = std::ptr::null_mut();
        expect_ok(unsafe { ffi::kh_kv_page_read_create(device.raw(), &config.to_ffi(), &mut raw) },
                  "kv_page_read::Compute::new");
        Self { raw }
    }

    pub fn invoke<'a>(&'a self, shape: Shape, buffers: Buffers<'a>, num_active_token_reads: ReplayU32,
                      page_table_index: ReplayU32) -> Invocation<'a> {
        Invocation { compute: self, shape, buffers, num_active_token_reads, page_table_index }
    }
}

impl Drop for Compute {
    fn drop(&mut self) {
        unsafe { ffi::kh_kv_page_read_destroy(self.raw) };
    }
}

pub struct Invocation<'a> {
    compute: &'a Compute,
    shape: Shape,
    buffers: Buffers<'a>,
    num_active_token_reads: ReplayU32,
    page_table_index: ReplayU32,
}

impl Operator for Invocation<'_> {
    fn record(self, recorder: &CommandRecorder<'_>) {
        let (ReplayU32::Value(reads), ReplayU32::Value(layer)) = (self.num_active_token_reads, self.page_table_index)
        else {
            panic!("kv page read takes its counts by value on the CUDA backend");
        };
        let shape = ffi::KhKvPageReadShape {
            num_total_token_reads: self.shape.num_total_token_reads,
            page_table_layout: self.shape.page_table_layout.to_ffi(),
        };
        let buffers = ffi::KhKvPageReadBuffers {
            pages: self.buffers.pages.raw(),
            flat_k: self.buffers.flat_k.raw(),
            flat_v: self.buffers.flat_v.raw(),
            req_slots: self.buffers.req_slots.raw(),
            flat_token_indices: self.buffers.flat_token_indices.raw(),
            page_ids: self.buffers.page_ids.raw(),
        };
        expect_ok(unsafe { ffi::kh_kv_page_read_invoke(self.compute.raw, recorder.stream().raw(), &shape, &buffers,
                                                       reads, layer) },
                  "kv page read");
    }
}
